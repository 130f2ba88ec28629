"""Operators of generation with an encrypted model: the ciphertext cache's pages, the value product over cached pages, and
rotary positions. Each case is one call of a decoding or prompt step; `op` says which, the rest its sizes:

  log_n    ring degree 2^log_n (2^(log_n - 1) slots)
  chain    Q primes of the chain: one of 60 bits and chain - 1 of `bits` bits
  special  special primes of 60 bits of the context that the framework's calls work in

  pages    page dst := old page src for `moves` pages in each of `planes` planes (K and V of the layers), all at once:
           `kind` copy (distinct pages), fork (one page into `moves` others), order (a permutation in place: compaction),
           lower (from a cache at a higher level, `from_limbs` primes a page)
  values   sum over `terms` cached pages of score x page, as a three-polynomial ciphertext, for `queries` queries that read the
           same pages; scores have `limbs` primes, pages `page_limbs`
  rotary   the factors of `tokens` positions on `axes` axes in the slot layout of the attention products
"""
import math
import os
import sys

import numpy as np
import torch

own = False

SCALE = 2.0 ** 40


# ---- the cases ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one page of the smallest ring copied before it is written to: launch and host time
        dict(name="pages_copy_n12_l3", op="pages", kind="copy", log_n=12, chain=4, bits=40, special=1, limbs=3, planes=1, pages=4, moves=1),
        # eight beams fork from one tail page, K and V of a layer, 16 limbs left of the benchmark's chain
        dict(name="pages_fork_n16_l16", op="pages", kind="fork", log_n=16, chain=24, bits=40, special=8, limbs=16, planes=2, pages=11, moves=8),
        # compaction after sequences have ended: most pages of a pool change places, K and V of two layers
        dict(name="pages_order_n14_l8", op="pages", kind="order", log_n=14, chain=8, bits=50, special=2, limbs=8, planes=4, pages=61, moves=47),
        # a prefix taken over into a cache five levels further down
        dict(name="pages_lower_n15_l9", op="pages", kind="lower", log_n=15, chain=14, bits=40, special=3, limbs=9, planes=2, pages=40, moves=24,
             from_limbs=14),
        # a short context in the smallest ring, three limbs left
        dict(name="values_n12_l3_t3", op="values", log_n=12, chain=4, bits=40, special=1, limbs=3, page_limbs=3, pages=5, terms=3, queries=1),
        # the benchmark's small ring, primes of 50 bits, pages two levels above the scores
        dict(name="values_n14_l6_t17", op="values", log_n=14, chain=8, bits=50, special=2, limbs=6, page_limbs=8, pages=20, terms=17, queries=1),
        # four query positions against one prefix
        dict(name="values_n15_l12_t24_q4", op="values", log_n=15, chain=12, bits=40, special=4, limbs=12, page_limbs=12, pages=24, terms=24, queries=4),
        # a context of 32 pages on the benchmark's chain
        dict(name="values_n16_l16_t32", op="values", log_n=16, chain=24, bits=40, special=8, limbs=16, page_limbs=16, pages=40, terms=32, queries=1),
        # the one position of a decoding step
        dict(name="rotary_token_n12", op="rotary", log_n=12, chain=4, bits=40, special=1, packing="pairs", heads=8, d_head=16, pairs=16, axes=1, tokens=1,
             reach=4096, dropped=False, pos="int64"),
        # frames of a video: time, height and width, some positions padding
        dict(name="rotary_video_n16", op="rotary", log_n=16, chain=24, bits=40, special=8, packing="pairs", heads=32, d_head=64, pairs=64, axes=3, tokens=1021,
             reach=512, dropped=True, pos="int32"),
        # a long context's far positions, interpolated, half of each head rotated, heads that leave slots over
        dict(name="rotary_far_n15", op="rotary", log_n=15, chain=14, bits=40, special=3, packing="interleaved", heads=9, d_head=80, pairs=20, axes=1, tokens=300,
             reach=1000000, dropped=False, pos="float64"),
        # a prompt of 4096 positions at the width of the benchmark's matrix (32 heads of 128), real slots
        dict(name="rotary_prompt_n16", op="rotary", log_n=16, chain=24, bits=40, special=8, packing="halves", heads=32, d_head=128, pairs=64, axes=1, tokens=4096,
             reach=8192, dropped=False, pos="int64"),
    ]


def _log_int(rng, lo, hi):
    """an integer of [lo, hi], spread evenly over the logarithm"""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["pages", "values", "rotary"])
    log_n = rng.randint(12, 16)
    chain = rng.randint(4, 24 if log_n >= 14 else 12)
    c = dict(op=op, log_n=log_n, chain=chain, bits=rng.choice([36, 40, 40, 45, 50, 55]), special=rng.randint(1, 4))
    page = 16 << log_n  # bytes of a page's limb
    if op == "pages":
        kind = rng.choice(["copy", "fork", "order", "lower"])
        limbs = rng.randint(1, chain)
        planes = rng.choice([1, 1, 2, 2, 4, 6])
        most = max(2, min(90, (800 << 20) // (2 * page * limbs * planes)))
        moves = _log_int(rng, 1 if kind != "order" else 2, most)
        pages = moves * (2 if kind == "copy" else 1) + rng.randint(1, 7)
        c.update(kind=kind, limbs=limbs, planes=planes, pages=pages, moves=moves)
        if kind == "lower":
            c["from_limbs"] = rng.randint(limbs, chain)
    elif op == "values":
        limbs = rng.randint(1, chain)
        queries = rng.choice([1, 1, 1, 2, 3, 4, 5])
        most = max(1, min(80, (1000 << 20) // (page * limbs * (queries + 1))))
        terms = _log_int(rng, 1, most)
        c.update(limbs=limbs, page_limbs=rng.choice([limbs, rng.randint(limbs, chain)]), pages=terms + rng.randint(0, 6), terms=terms, queries=queries)
    else:
        d_head = rng.choice([16, 32, 40, 64, 64, 80, 96, 128])
        packing = rng.choice(["pairs", "halves", "interleaved"])
        top = d_head if packing == "pairs" else d_head // 2
        heads = _log_int(rng, 1, (1 << (log_n - 1)) // d_head)
        per = (1 << (log_n - 1)) // (heads * d_head)
        most = max(1, (700 << 20) * per // ((16 << (log_n - 1)) * (1 if packing == "pairs" else 3)))
        c.update(packing=packing, heads=heads, d_head=d_head, pairs=rng.choice([top, max(1, top // 2), max(1, top // 4)]), axes=rng.choice([1, 2, 3, 4]),
                 tokens=_log_int(rng, 1, min(5000, most)), reach=rng.choice([512, 4096, 131072, 1000000]), dropped=rng.random() < 0.4,
                 pos=rng.choice(["int32", "int64", "float32", "float64"]))
    return c


# ---- primes: the largest ones = 1 (mod 2 N) of each size, handed out smallest first ------------------------------------
def _is_prime(n):
    d, r = n - 1, 0
    while d % 2 == 0:
        d, r = d // 2, r + 1
    for a in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37):
        x = pow(a, d, n)
        if x in (1, n - 1):
            continue
        for _ in range(r - 1):
            x = x * x % n
            if x == n - 1:
                break
        else:
            return False
    return True


_PRIMES = {}


def _primes(case):
    """Q primes, then the special primes"""
    key = case["log_n"], case["chain"], case["bits"], case["special"]
    if key not in _PRIMES:
        log_n, chain, bits, special = key
        sizes = [60] + [bits] * (chain - 1) + [60] * special
        found = {}
        for b in set(sizes):
            v, found[b] = (1 << b) + 1 - (2 << log_n), []
            while len(found[b]) < sizes.count(b):
                if _is_prime(v):
                    found[b].append(v)
                v -= 2 << log_n
        _PRIMES[key] = [found[b].pop() for b in sizes]
    return _PRIMES[key]


# ---- states ---------------------------------------------------------------------------------------------------------
_CONTEXTS = {}


def _context(case):
    """the framework and a context of the case's primes, made once for each parameter set as a server keeps it"""
    path = os.path.join(os.getcwd(), "phantom-fhe_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pyPhantom as ph
    key = case["log_n"], case["chain"], case["bits"], case["special"]
    if key not in _CONTEXTS:
        parms = ph.params(ph.scheme_type.ckks)
        parms.set_poly_modulus_degree(1 << case["log_n"])
        parms.set_coeff_modulus([ph.modulus(q) for q in _primes(case)])
        parms.set_special_modulus_size(case["special"])
        parms.set_galois_elts([(2 << case["log_n"]) - 1])
        _CONTEXTS[key] = ph.context(parms)
    return ph, _CONTEXTS[key]


def _residues(gen, q, *shape):
    """uniform residues [*shape][limbs][N] for the primes q [limbs][1]"""
    return torch.randint(0, 1 << 62, shape, dtype=torch.int64, device="cuda", generator=gen).remainder_(q)


def _moves(case, seed):
    """(dst, src) page numbers"""
    rng = np.random.default_rng(seed)
    order = [int(p) for p in rng.permutation(case["pages"])]
    m = case["moves"]
    if case["kind"] == "fork":
        return order[1:m + 1], [order[0]] * m
    if case["kind"] == "order":
        step = next(k for k in (5, 3, 2, 1) if math.gcd(k, m) == 1)
        return order[:m], [order[(i * step + 1) % m] for i in range(m)]
    if case["kind"] == "lower":
        return order[:m], [int(p) for p in rng.permutation(case["pages"])[:m]]
    return order[:m], order[m:2 * m]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    N, s = 1 << case["log_n"], {}
    q = torch.tensor(_primes(case), dtype=torch.int64, device="cuda")[:, None]
    if case["op"] == "pages":
        s["pool"] = _residues(gen, q[:case["limbs"]], case["planes"], case["pages"], 2, case["limbs"], N)
        if case["kind"] == "lower":
            s["source"] = _residues(gen, q[:case["from_limbs"]], case["planes"], case["pages"], 2, case["from_limbs"], N)
        s["dst"], s["src"] = _moves(case, seed)
    elif case["op"] == "values":
        rng = np.random.default_rng(seed)
        s["q"] = q[:case["limbs"]]
        s["scores"] = _residues(gen, s["q"], case["queries"], case["terms"], 2, case["limbs"], N)
        s["pool"] = _residues(gen, q[:case["page_limbs"]], 1, case["pages"], 2, case["page_limbs"], N)
        s["table"] = [int(p) for p in rng.permutation(case["pages"])[:case["terms"]]]
    else:
        whole = case["pos"].startswith("int")
        p = torch.randint(0, case["reach"], (case["tokens"], case["axes"]), device="cuda", generator=gen)
        if not whole:  # positions between the trained ones
            p = p.double() * 0.25
        s["positions"] = p.to(getattr(torch, case["pos"]))
        s["keep"] = torch.rand(case["tokens"], device="cuda", generator=gen) < 0.85 if case["dropped"] else None
        s["inv_freq"] = 10000.0 ** (-torch.arange(case["pairs"], dtype=torch.float64, device="cuda") / case["pairs"])
        s["axes"] = [j * case["axes"] // case["pairs"] for j in range(case["pairs"])]
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    if own:
        ph, ctx = _context(case)
        if case["op"] == "rotary":
            s["rotary"] = ph.rotary(ctx, s["inv_freq"], case["heads"], case["d_head"], axes=s["axes"], packing=case["packing"])
        else:
            s["cache"] = _cache(ph, ctx, case, s.pop("pool"))
            if "source" in s:
                s["from"] = _cache(ph, ctx, case, s.pop("source"))
        if case["op"] == "values":
            level = case["chain"] - case["limbs"] + 1
            s["queries"] = [[_ciphertext(ph, x, level) for x in row] for row in s["scores"]]
    elif case["op"] == "rotary":
        s["axes"] = torch.tensor(s["axes"], device="cuda")
    else:
        for k in ("dst", "src", "table"):
            if k in s:
                s[k] = torch.tensor(s[k], device="cuda")
    return s


def _cache(ph, ctx, case, pool):
    c = ph.ciphertext_cache(ctx, case["chain"] - pool.shape[3] + 1, pool.shape[1], planes=pool.shape[0], scale=SCALE)
    c.allocate(pool.shape[1])
    c.data.copy_(pool)
    return c


def _ciphertext(ph, data, level):
    ct = ph.ciphertext()
    ct._chain_index, ct._size, ct._limbs, ct._N, ct._scale, ct.data = level, data.shape[0], data.shape[1], data.shape[2], SCALE, data
    return ct


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        if case["op"] == "pages":
            state["cache"].copy(state["dst"], state["src"], source=state.get("from"))
            return state["cache"].data
        if case["op"] == "values":
            return [ct.data for ct in state["cache"].multiply_sum(state["queries"], state["table"])]
        return state["rotary"].factors(state["positions"], keep=state["keep"])
    return {"pages": _plain_pages, "values": _plain_values, "rotary": _plain_rotary}[case["op"]](state)


def _plain_pages(s):
    pool, l = s["pool"], s["case"]["limbs"]
    pool[:, s["dst"]] = s["source"][:, s["src"], :, :l] if "source" in s else pool[:, s["src"]]
    return pool


def _mul_small(x, y, q):
    """x y mod q for 0 <= x < q < 2^61 and 0 <= y < 2^31: the quotient in 64-bit floating point is off by one at most"""
    k = (x.double() * y / q.double()).long()
    r = x * y - k * q
    r = torch.where(r < 0, r + q, r)
    return torch.where(r >= q, r - q, r)


def _mul(x, y, q):
    """x y mod q, the second factor in two pieces of 31 bits"""
    high = _mul_small(_mul_small(x, y >> 31, q), 1 << 30, q)
    r = high + high - q
    r = torch.where(r < 0, r + q, r) + _mul_small(x, y & 0x7FFFFFFF, q) - q
    return torch.where(r < 0, r + q, r)


def _sum(x, q):
    """the sum over the terms mod q, in pieces of 30 bits"""
    high, low = (x >> 30).sum(1).remainder(q), (x & 0x3FFFFFFF).sum(1).remainder(q)
    r = _mul_small(high, 1 << 30, q) + low - q
    return torch.where(r < 0, r + q, r)


def _plain_values(s):
    q, a = s["q"], s["scores"]
    b = s["pool"][0][s["table"]][:, :, :s["case"]["limbs"]]
    a0, a1, b0, b1 = a[:, :, 0], a[:, :, 1], b[None, :, 0], b[None, :, 1]
    d1 = _sum(_mul(a0, b1, q), q) + _sum(_mul(a1, b0, q), q) - q
    out = torch.stack([_sum(_mul(a0, b0, q), q), torch.where(d1 < 0, d1 + q, d1), _sum(_mul(a1, b1, q), q)], 1)
    return list(out.unbind(0))


def _plain_rotary(s):
    c = s["case"]
    slots, width, T = 1 << (c["log_n"] - 1), c["heads"] * c["d_head"], c["tokens"]
    per = slots // width
    n = -(-T // per)
    angle = s["positions"].double()[:, s["axes"]] * s["inv_freq"]
    cos, sin = angle.cos(), angle.sin()
    ones = torch.ones(T, c["d_head"] - c["pairs"] * (1 if c["packing"] == "pairs" else 2), dtype=torch.float64, device="cuda")
    zero = torch.zeros_like(sin)
    if c["packing"] == "pairs":
        rows = [torch.complex(torch.cat([cos, ones], 1), torch.cat([sin, 0 * ones], 1))]
    elif c["packing"] == "halves":
        rows = [torch.cat([cos, cos, ones], 1), torch.cat([-sin, zero, 0 * ones], 1), torch.cat([zero, sin, 0 * ones], 1)]
    else:
        rows = [torch.cat([torch.stack(p, 2).flatten(1), rest], 1) for p, rest in (((cos, cos), ones), ((-sin, zero), 0 * ones), ((zero, sin), 0 * ones))]
    rows = torch.stack(rows).to(torch.complex128)
    if s["keep"] is not None:
        rows = rows * s["keep"][:, None]
    out = torch.zeros(len(rows), n * per, width, dtype=torch.complex128, device="cuda")
    out[:, :T] = rows.repeat(1, 1, c["heads"])
    return torch.nn.functional.pad(out.view(len(rows), n, per * width), (0, slots - per * width))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    N = 1 << case["log_n"]
    if case["op"] == "pages":
        sources = 1 if case["kind"] == "fork" else case["moves"]
        return {"bytes": (sources + case["moves"]) * case["planes"] * 16 * case["limbs"] * N, "flops": 0}
    if case["op"] == "values":
        g, t, l = case["queries"], case["terms"], case["limbs"]
        return {"bytes": 8 * l * N * (2 * t * (g + 1) + 3 * g), "flops": 8 * g * t * l * N}
    per = (N // 2) // (case["heads"] * case["d_head"])
    n = -(-case["tokens"] // per)
    size = {"int32": 4, "int64": 8, "float32": 4, "float64": 8}[case["pos"]]
    return {"bytes": 16 * n * (N // 2) * (1 if case["packing"] == "pairs" else 3) + size * case["tokens"] * case["axes"] + 8 * case["pairs"],
            "flops": 60 * case["tokens"] * case["pairs"]}


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "pages":
        new = s["pool"].clone()
        for d, p in zip(s["dst"], s["src"]):
            new[:, d] = s["source"][:, p, :, :case["limbs"]] if "source" in s else s["pool"][:, p]
        return new
    if case["op"] == "values":
        if case["queries"] * case["terms"] * case["limbs"] << case["log_n"] > 1 << 27:
            return None
        return [torch.stack([_definition(row, s, p) for p in range(3)]) for row in s["scores"]]
    slots, width, h = 1 << (case["log_n"] - 1), case["heads"] * case["d_head"], case["d_head"]
    per, r = slots // width, case["pairs"]
    n = -(-case["tokens"] // per)
    out = np.zeros((1 if case["packing"] == "pairs" else 3, n, slots), dtype=np.complex128)
    angle = s["positions"].double().cpu().numpy()[:, s["axes"]] * s["inv_freq"].cpu().numpy()
    cos, sin, keep = np.cos(angle), np.sin(angle), None if s["keep"] is None else s["keep"].cpu().numpy()
    for t in range(case["tokens"]):
        if keep is not None and not keep[t]:
            continue
        head = np.zeros((len(out), h), dtype=np.complex128)
        head[0] = 1.0
        if case["packing"] == "pairs":
            head[0, :r] = cos[t] + 1j * sin[t]
        else:
            first, second = (np.arange(r), np.arange(r) + r) if case["packing"] == "halves" else (2 * np.arange(r), 2 * np.arange(r) + 1)
            head[0, first], head[0, second], head[1, first], head[2, second] = cos[t], cos[t], -sin[t], sin[t]
        at = (t % per) * width
        out[:, t // per, at:at + width] = np.tile(head, (1, case["heads"]))
    return out


def _definition(row, s, p):
    """polynomial p of the sum of products, each product by doubling and adding over the bits of one factor"""
    q, acc = s["q"], torch.zeros_like(row[0, 0])
    for a, page in zip(row, s["table"]):
        b = s["pool"][0, page][:, :a.shape[1]]
        for x, y in ([(0, 0)], [(0, 1), (1, 0)], [(1, 1)])[p]:
            r = torch.zeros_like(acc)
            for bit in range(60, -1, -1):
                r = r + r
                r = torch.where(r >= q, r - q, r) + ((b[y] >> bit) & 1) * a[x]
                r = torch.where(r >= q, r - q, r)
            acc = acc + r
            acc = torch.where(acc >= q, acc - q, acc)
    return acc
