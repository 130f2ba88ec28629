"""The cache of ciphertexts in pages and what reads it: page moves and sums of products word for word against the same on the host
(integers of any size), the cache's bookkeeping, the attention products over cached pages, and a decoding step made of them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import pyPhantom as ph
from pyPhantom._native import LIB, check
from gpu_helpers import host, kernels_of, stream

N = 4096


def _is_prime(v):
    return all(pow(a, v - 1, v) == 1 for a in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37))


def _below(bits, count, N=N):
    """the `count` largest primes = 1 (mod 2 N) below 2^bits"""
    out, v = [], (1 << bits) + 1 - 2 * N
    while len(out) < count:
        if _is_prime(v):
            out.append(v)
        v -= 2 * N
    return out


def _ctx(primes, special=1, N=N):
    parms = ph.params(ph.scheme_type.ckks)
    parms.set_poly_modulus_degree(N)
    parms.set_coeff_modulus([ph.modulus(q) for q in primes])
    parms.set_special_modulus_size(special)
    return ph.context(parms)


# every arithmetic that a sum of products has: primes of 61 bits, 60, 55, 50, 45, 40 and 30
MIXED = _below(61, 1) + _below(60, 1) + _below(55, 1) + _below(50, 1) + _below(45, 1) + _below(41, 1) + _below(40, 1) + _below(30, 1)


@pytest.fixture(scope="module")
def mixed():
    return _ctx(MIXED + _below(60, 2)[1:])


def _residues(rng, ctx, *shape):
    """random residues, with the largest and the smallest among them; the last two axes are [limbs][N]"""
    q = ctx.primes[:shape[-1]].astype(np.uint64)[:, None]
    x = rng.integers(0, 1 << 62, (*shape, ctx.N), dtype=np.uint64) % q
    x[..., :7] = q - np.uint64(1)
    x[..., 7:9] = 0
    return x


def _fill(cache, rng):
    x = _residues(rng, cache.ctx, *cache.data.shape[:4])
    cache.data.copy_(torch.from_numpy(x.view(np.int64)))
    return x


def _ct(ctx, x, scale=2.0 ** 40):
    return ph.ciphertext.from_numpy(ctx, x, ctx.size_Q - x.shape[1] + 1, scale)


# ---- page moves ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("planes,pages,limbs", [(1, 1, 1), (1, 9, 3), (3, 17, 2), (5, 40, 8)])
def test_moves_are_made_all_at_once(mixed, planes, pages, limbs):
    rng = np.random.default_rng(planes * 100 + pages)
    cache = ph.ciphertext_cache(mixed, mixed.size_Q - limbs + 1, pages, planes)
    assert cache.allocate(pages) == list(range(pages)) and not host(cache.data).any()  # pages come zeroed
    was = _fill(cache, rng)
    for kind in ("shift", "reverse", "one", "random", "few", "none"):
        n = int(rng.integers(1, pages + 1))
        dst = [int(p) for p in rng.permutation(pages)[:n]]
        src = {"shift": dst[1:] + dst[:1], "reverse": dst[::-1], "one": [dst[0]] * n, "random": [int(p) for p in rng.integers(0, pages, n)],
               "few": [int(p) for p in rng.integers(0, min(2, pages), n)], "none": dst}[kind]
        cache.copy(dst, src)
        want = was.copy()
        want[:, dst] = was[:, src]
        was = want
        assert np.array_equal(host(cache.data), want), kind
    cache.copy([], [])


def test_a_move_of_more_pages_than_a_launch_takes(mixed):
    """1200 pages change places: one long cycle, a random permutation, one page into all, and the launches there are for them"""
    rng = np.random.default_rng(4)
    cache = ph.ciphertext_cache(mixed, mixed.size_Q, 1200)
    pages = cache.allocate(1200)
    was = _fill(cache, rng)
    for dst, src in ((pages, pages[1:] + pages[:1]), (pages, [int(p) for p in rng.permutation(1200)]), (pages[1:], [0] * 1199)):
        _, launched = kernels_of(mixed, lambda: cache.copy(dst, src))
        assert set(launched) == {"pages_move"} and 3 <= launched["pages_move"] <= 4
        want = was.copy()
        want[:, dst] = was[:, src]
        was = want
        assert np.array_equal(host(cache.data), want)


@pytest.mark.parametrize("limbs,of", [(1, 1), (1, 8), (3, 5), (8, 8)])
def test_pages_of_a_higher_level(mixed, limbs, of):
    rng = np.random.default_rng(limbs)
    low, high = (ph.ciphertext_cache(mixed, mixed.size_Q - l + 1, 12, 2) for l in (limbs, of))
    low.allocate(12), high.allocate(12)
    was, other = _fill(low, rng), _fill(high, rng)
    dst, src = [int(p) for p in rng.permutation(12)[:9]], [int(p) for p in rng.integers(0, 12, 9)]
    low.copy(dst, src, source=high)
    was[:, dst] = other[:, src, :, :limbs]
    assert np.array_equal(host(low.data), was) and np.array_equal(host(high.data), other)


def test_addresses_past_32_bits():
    """a pool of 4.5 GB: pages behind 2^32 bytes and 2^29 words, in the last plane"""
    ctx = _ctx(_below(40, 4, 1 << 16), N=1 << 16)
    cache = ph.ciphertext_cache(ctx, 1, 720, 2)
    cache.allocate(720)
    rng = np.random.default_rng(5)
    marks = [0, 1, 340, 341, 342, 718, 719]
    for plane in range(2):
        for p in marks:
            cache.data[plane, p].fill_(1000 * plane + p + 1)
    dst, src = [719, 0, 342, 1], [0, 719, 1, 341]
    cache.copy(dst, src)
    torch.cuda.synchronize()
    for plane in range(2):
        now = {p: p for p in marks}
        now.update(zip(dst, src))
        for p in marks:
            row = cache.data[plane, p]
            assert int(row.min()) == int(row.max()) == 1000 * plane + now[p] + 1
        assert not bool(cache.data[plane, 2:340].any()) and not bool(cache.data[plane, 343:718].any())
    # products read pages behind that line too
    x = _residues(rng, ctx, 2, 3)
    cache.data[1, 719].copy_(torch.from_numpy(x.view(np.int64)))
    a = _ct(ctx, _residues(rng, ctx, 2, 3))
    assert np.array_equal(cache.multiply_sum([a], [719], plane=1).numpy(), ph.multiply(ctx, a, _ct(ctx, x)).numpy())


# ---- sums of products -----------------------------------------------------------------------------------------------------------
def _sum_of_products(primes, a, b):
    """a [terms][2][l][N], b alike, in integers of any size"""
    q = np.array([int(p) for p in primes], dtype=object)[:, None]
    d = [0, 0, 0]
    for x, y in zip(a.astype(object), b.astype(object)):
        d = [d[0] + x[0] * y[0], d[1] + x[0] * y[1] + x[1] * y[0], d[2] + x[1] * y[1]]
    return np.stack([(v % q).astype(np.uint64) for v in d])


@pytest.mark.parametrize("terms", [1, 2, 3, 4, 5, 7, 8, 16, 31, 33])
def test_sum_of_products(mixed, terms):
    rng = np.random.default_rng(terms)
    a, b = _residues(rng, mixed, terms, 2, 8), _residues(rng, mixed, terms, 2, 8)
    got = ph.multiply_sum(mixed, [_ct(mixed, x) for x in a], [_ct(mixed, x, 2.0 ** 38) for x in b])
    assert got.size() == 3 and got.chain_index() == 1 and got.scale() == 2.0 ** 78
    assert np.array_equal(got.numpy(), _sum_of_products(MIXED, a, b))


@pytest.mark.parametrize("terms", [63, 64, 65, 129, 200])
def test_long_sums(terms):
    """where the sums in registers are brought back, and where a second launch adds to the first one's result; largest residues"""
    primes = _below(61, 1) + _below(60, 1) + _below(50, 1) + _below(41, 1)
    ctx = _ctx(primes + _below(60, 2)[1:])
    q = ctx.primes[:4].astype(np.uint64)[:, None]
    a = np.broadcast_to(q - np.uint64(1), (2, 4, N)).copy()  # every product is the largest there is
    a[:, :, ::2] = _residues(np.random.default_rng(terms), ctx, 2, 4)[:, :, ::2]
    got = ph.multiply_sum(ctx, [_ct(ctx, a)] * terms, [_ct(ctx, a)] * terms).numpy()
    one = _sum_of_products(primes, a[None], a[None])
    want = np.stack([(one[p].astype(object) * terms % q.astype(object)).astype(np.uint64) for p in range(3)])
    assert np.array_equal(got, want)


@pytest.mark.parametrize("queries", [1, 2, 3, 4, 5, 9])
@pytest.mark.parametrize("levels", [(3, 3), (3, 8), (5, 2)])
def test_queries_share_the_pages_and_levels_may_differ(mixed, queries, levels):
    la, lb = levels
    l, terms = min(levels), 6
    rng = np.random.default_rng(queries * 10 + la)
    cache = ph.ciphertext_cache(mixed, mixed.size_Q - lb + 1, 8, 2)
    cache.allocate(8)
    pool = _fill(cache, rng)
    a = _residues(rng, mixed, queries, terms, 2, la)
    table = [7, 2, 2, 0, 5, 1]  # a page may be named twice
    got = cache.multiply_sum([[_ct(mixed, x) for x in row] for row in a], table, plane=1)
    assert len(got) == queries and all(ct.chain_index() == mixed.size_Q - l + 1 for ct in got)
    for g in range(queries):
        want = _sum_of_products(MIXED[:l], a[g][:, :, :l], pool[1, table][:, :, :l])
        assert np.array_equal(got[g].numpy(), want)
    single = cache.multiply_sum([_ct(mixed, x) for x in a[0]], table, plane=1)
    assert np.array_equal(single.numpy(), got[0].numpy())


def test_one_term_is_the_tensor_product_in_every_ring():
    for log_n in (12, 13, 14, 15, 16, 17):
        ctx = _ctx(_below(60, 1, 1 << log_n) + _below(40, 2, 1 << log_n), N=1 << log_n)
        rng = np.random.default_rng(log_n)
        a, b = _ct(ctx, _residues(rng, ctx, 2, 2)), _ct(ctx, _residues(rng, ctx, 2, 2))
        assert np.array_equal(ph.multiply_sum(ctx, [a], [b]).numpy(), ph.multiply(ctx, a, b).numpy())
        cache = ph.ciphertext_cache(ctx, 1, 3, 2)
        cache.allocate(3)
        was = _fill(cache, rng)
        cache.copy([0, 1, 2], [2, 0, 1])
        assert np.array_equal(host(cache.data), was[:, [2, 0, 1]])


def test_views_that_are_not_contiguous(mixed):
    """a ciphertext whose polynomials lie apart (a slice of a higher level) counts as what it holds"""
    rng = np.random.default_rng(11)
    x = _residues(rng, mixed, 2, 8)
    high = _ct(mixed, x)
    view = high._like(high.data[:, :5], chain_index=4)
    assert not view.data.is_contiguous()
    got = ph.multiply_sum(mixed, [view, view], [view, view]).numpy()
    assert np.array_equal(got, _sum_of_products(MIXED[:5], np.stack([x[:, :5]] * 2), np.stack([x[:, :5]] * 2)))
    cache = ph.ciphertext_cache(mixed, 4, 2)
    (page, other) = cache.allocate(2)
    cache.store(page, view)
    cache.append(page, view)
    cache.append(other, high)  # dropped to the cache's level
    q = mixed.primes[:5].astype(np.uint64)[:, None]
    assert np.array_equal(cache.page(page).numpy(), (x[:, :5] + x[:, :5]) % q)
    assert np.array_equal(cache.page(other).numpy(), x[:, :5])


def test_words_that_are_not_there(mixed):
    """ciphertexts on the host, of another type, or with fewer words than their level has never reach a kernel"""
    rng = np.random.default_rng(18)
    good = _ct(mixed, _residues(rng, mixed, 2, 4))
    cache = ph.ciphertext_cache(mixed, good.chain_index(), 2)
    (page, _) = cache.allocate(2)
    bad = [good._like(good.data.cpu()), good.clone(), good.clone(), good.clone(), good._like(good.data[:, :3])]
    bad[1].data = good.data[:1]
    bad[2].data = good.data.double()
    bad[3].data = good.data[..., :N // 2]
    for ct in bad:
        for call in (lambda: ph.multiply_sum(mixed, [good, ct], [good, good]), lambda: ph.multiply_sum(mixed, [ct], [good]),
                     lambda: cache.multiply_sum([good, ct], [page, page]), lambda: ph.cached_qkt(mixed, None, None, ct, cache, [page], 2)):
            with pytest.raises(ValueError):
                call()
    for ct in bad[:2] + bad[3:4]:
        for call in (lambda: cache.store(page, ct), lambda: cache.append(page, ct)):
            with pytest.raises(ValueError):
                call()
    mask = ph.plaintext.from_numpy(mixed, _residues(rng, mixed, 4), good.chain_index())
    mask.data = mask.data[:3]
    with pytest.raises(ValueError, match="mismatch"):
        ph.cached_score_times_v(mixed, None, None, [good], cache, [page], mask, 2, 4, 2)


@pytest.mark.parametrize("terms", [1, 2, 3, 4])
@pytest.mark.parametrize("n", [1, 5, 33, 70])
def test_sums_of_ciphertexts_times_plaintexts(mixed, n, terms):
    """what rotary positions are applied with: n sums in one launch (of at most 32), against single products and additions"""
    rng = np.random.default_rng(n * 10 + terms)
    cts = [_ct(mixed, _residues(rng, mixed, 2, 8)) for _ in range(7)]
    pts = [ph.plaintext.from_numpy(mixed, _residues(rng, mixed, 8), 1) for _ in range(5)]
    pick = [[(int(rng.integers(7)), int(rng.integers(5))) for _ in range(terms)] for _ in range(n)]
    a = np.array([cts[i].data.data_ptr() for row in pick for i, _ in row], dtype=np.uint64)
    b = np.array([pts[j].data.data_ptr() for row in pick for _, j in row], dtype=np.uint64)
    out = mixed.empty(n, 2, 8)
    check(LIB.b2_multiply_plain_sum(mixed._h, 8, n, terms, a.ctypes.data, b.ctypes.data, out.data_ptr(), stream()))
    for k in {0, n // 2, n - 1}:
        want = ph.add_many(mixed, [ph.multiply_plain(mixed, cts[i], pts[j]) for i, j in pick[k]])
        assert torch.equal(out[k], want.data)
    for args, match in [((0, terms), "bad argument"), ((n, 0), "terms"), ((n, 5), "terms")]:
        with pytest.raises(ValueError, match=match):
            check(LIB.b2_multiply_plain_sum(mixed._h, 8, *args, a.ctypes.data, b.ctypes.data, out.data_ptr(), stream()))
    a[0] += np.uint64(8)
    with pytest.raises(ValueError, match="aligned"):
        check(LIB.b2_multiply_plain_sum(mixed._h, 8, n, terms, a.ctypes.data, b.ctypes.data, out.data_ptr(), stream()))


# ---- streams and graphs ---------------------------------------------------------------------------------------------------------
def test_captured_calls_replay(mixed):
    rng = np.random.default_rng(12)
    cache = ph.ciphertext_cache(mixed, 1, 6)
    cache.allocate(6)
    was = _fill(cache, rng)
    a = _residues(rng, mixed, 2, 2, 8)
    cts = [_ct(mixed, x) for x in a]
    table = [4, 1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.multiply_sum(cts, table)  # nothing of the first call is left to the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.copy([0, 1, 2, 3, 4, 5], [1, 2, 3, 4, 5, 0])
        out = cache.multiply_sum(cts, table)
    for _ in range(7):
        g.replay()
        was = was[:, [1, 2, 3, 4, 5, 0]]
        torch.cuda.synchronize()
        assert np.array_equal(host(cache.data), was)
        assert np.array_equal(out.numpy(), _sum_of_products(MIXED, a, was[0, table]))


def test_two_streams_at_once(mixed):
    """sums of two streams have nothing in common; a move on one stream does not touch the other cache"""
    rng = np.random.default_rng(13)
    caches, pools, streams, rows = [], [], [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(2):
        c = ph.ciphertext_cache(mixed, 1, 30)
        c.allocate(30)
        pools.append(_fill(c, rng))
        caches.append(c)
        rows.append([_ct(mixed, x) for x in _residues(rng, mixed, 20, 2, 8)])
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                outs[k].append(caches[k].multiply_sum(rows[k], list(range(20))))
                caches[k].copy(list(range(30)), list(range(1, 30)) + [0])
    torch.cuda.synchronize()
    for k in range(2):
        a = np.stack([c.numpy() for c in rows[k]])
        for i, out in enumerate(outs[k]):
            now = np.roll(pools[k], -i, axis=1)
            assert np.array_equal(out.numpy(), _sum_of_products(MIXED, a, now[0, :20]))


# ---- bookkeeping ----------------------------------------------------------------------------------------------------------------
def test_fork_share_and_free(mixed):
    rng = np.random.default_rng(14)
    cache = ph.ciphertext_cache(mixed, 6, 20, 2)
    table = cache.allocate(4)
    was = _fill(cache, rng)
    forks, launched = kernels_of(mixed, lambda: cache.fork(table, copies=3))
    assert launched == {"pages_move": 1}
    assert [f[:3] for f in forks] == [table[:3]] * 3 and len({f[3] for f in forks} | {table[3]}) == 4
    assert [cache.held(p) for p in table] == [4, 4, 4, 1] and cache.free_pages() == 20 - 7
    now = host(cache.data)
    assert all(np.array_equal(now[:, f[3]], was[:, table[3]]) for f in forks) and np.array_equal(now[:, :4], was[:, :4])
    with pytest.raises(ValueError, match="shared"):
        cache.append(table[0], cache.page(table[3]))
    cache.append(forks[0][3], cache.page(table[3]))
    cache.free(table)
    assert cache.free_pages() == 20 - 6
    with pytest.raises(ValueError, match="not allocated"):
        cache.free([table[3]])
    with pytest.raises(ValueError, match="more often"):
        cache.free(forks[0] + forks[0])
    for f in forks:
        cache.free(f)
    assert cache.free_pages() == 20
    assert cache.fork([], copies=2) == [[], []]
    whole = cache.fork(cache.allocate(3), tail=0)[0]
    assert whole == [0, 1, 2] and [cache.held(p) for p in whole] == [2, 2, 2]
    copied = cache.fork(whole, tail=9)[0]  # a tail longer than the table: everything is copied
    assert not set(copied) & set(whole)


def test_compact_and_resize(mixed):
    rng = np.random.default_rng(15)
    cache = ph.ciphertext_cache(mixed, 7, 24, 3)
    tables = [cache.allocate(5) for _ in range(4)]
    extra = cache.fork(tables[1], tail=1)[0]
    was = _fill(cache, rng)
    cache.free(tables[0])
    cache.free(tables[2])
    live = [tables[3], extra]  # tables[1] is held but not named: its pages keep their order behind the others
    contents = [was[:, t] for t in live]
    alone = was[:, tables[1][4]]
    new, launched = kernels_of(mixed, lambda: cache.compact(live))
    assert launched == {"pages_move": 1}
    assert new == [[0, 1, 2, 3, 4], [5, 6, 7, 8, 9]] and cache.free_pages() == 24 - 11
    now = host(cache.data)
    assert all(np.array_equal(now[:, t], c) for t, c in zip(new, contents)) and np.array_equal(now[:, 10], alone)
    assert [cache.held(p) for p in range(12)] == [1] * 5 + [2] * 4 + [1, 1, 0]
    with pytest.raises(ValueError, match="compact first"):
        cache.resize(10)
    cache.resize(11)
    assert cache.pages() == 11 and cache.free_pages() == 0 and np.array_equal(host(cache.data), now[:, :11])
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.allocate(1)
    cache.resize(13)
    assert cache.allocate(2) == [11, 12] and np.array_equal(host(cache.data)[:, :11], now[:, :11])
    for t in new:
        cache.free(t)
    assert cache.compact([]) == [] and cache.free_pages() == 13 - 7  # five pages of tables[1], two allocated last


def test_what_is_refused(mixed):
    cache = ph.ciphertext_cache(mixed, 3, 6, 2)
    t = cache.allocate(4)
    before = host(cache.data).copy()
    other = ph.ciphertext_cache(mixed, 5, 6, 2)
    other.allocate(6)
    one = ph.ciphertext_cache(mixed, 3, 6, 1)
    one.allocate(6)
    for call, match in [(lambda: cache.copy([0], [1, 2]), "as many"), (lambda: cache.copy([0, 0], [1, 2]), "named twice"),
                        (lambda: cache.copy([5], [0]), "not allocated"), (lambda: cache.copy([0], [6]), "out of range"),
                        (lambda: cache.copy([-1], [0]), "out of range"), (lambda: cache.copy([0], [0], source=other), "lower level"),
                        (lambda: cache.copy([0], [0], source=one), "other planes"), (lambda: cache.page(0, plane=2), "plane"),
                        (lambda: cache.fork(t, copies=0), "at least one"), (lambda: cache.fork(t, tail=-1), "at least one"),
                        (lambda: cache.allocate(-1), "negative"), (lambda: ph.ciphertext_cache(mixed, 1, 0), "at least one"),
                        (lambda: ph.ciphertext_cache(mixed, 0, 3), "chain index"), (lambda: ph.ciphertext_cache(mixed, 9, 3), "chain index"),
                        (lambda: cache.store(0, ph.mod_switch_to(mixed, cache.page(1), 4)), "higher level"),
                        (lambda: cache.append(0, cache.page(1)._like(cache.page(1).data, scale=2.0)), "scale"),
                        (lambda: cache.multiply_sum([], [0]), "empty"), (lambda: cache.multiply_sum([cache.page(0)], []), "as many"),
                        (lambda: cache.multiply_sum([cache.page(0)] * 2, [0]), "as many"), (lambda: cache.multiply_sum([cache.page(0)], [4]), "not allocated"),
                        (lambda: cache.multiply_sum([[cache.page(0)], []], [0]), "as many"),
                        (lambda: cache.multiply_sum([cache.page(0), other.page(0)], [0, 1]), "parameter mismatch"),
                        (lambda: ph.multiply_sum(mixed, [cache.page(0)], []), "empty"),
                        (lambda: ph.multiply_sum(mixed, [cache.page(0)], [ph.multiply(mixed, cache.page(0), cache.page(1))]), "2-polynomial")]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.allocate(3)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.fork(t, copies=3)
    assert cache.free_pages() == 2 and np.array_equal(host(cache.data), before)
    # the C entries' own checks
    d, s = np.array([0, 1], dtype=np.int64), np.array([1, 7], dtype=np.int64)
    args = lambda **k: [mixed._h, k.get("limbs", 6), k.get("planes", 2), k.get("pool", cache.data.data_ptr()), 6, k.get("src", 0), k.get("sl", 6), 6, 2,
                        k.get("dst", d.ctypes.data), k.get("s", s.ctypes.data), stream()]
    for kw, match in [({}, "source page out of range"), (dict(dst=s.ctypes.data, s=d.ctypes.data), "destination page out of range"), (dict(pool=0), "null"),
                      (dict(limbs=0), "size_Ql"), (dict(limbs=9), "size_Ql"), (dict(planes=0), "planes"), (dict(pool=cache.data.data_ptr() + 8), "aligned"),
                      (dict(src=cache.data.data_ptr() + 32, s=d.ctypes.data), "overlaps"), (dict(src=other.data.data_ptr(), sl=5, s=d.ctypes.data), "level")]:
        with pytest.raises(ValueError, match=match):
            check(LIB.b2_pages_move(*args(**kw)))
    for kw in (dict(src=cache.data.data_ptr(), sl=7, s=d.ctypes.data), dict(src=cache.data.data_ptr(), limbs=5, s=d.ctypes.data)):
        with pytest.raises(ValueError, match="another shape"):
            check(LIB.b2_pages_move(*args(**kw)))
    out = mixed.empty(3, 6)
    one_page = np.array([cache.data.data_ptr()], dtype=np.uint64)
    for at in (cache.data.data_ptr(), cache.data.data_ptr() + 8 * (2 * 6 * N - 4), cache.data.data_ptr() - 8 * (3 * 6 * N - 4)):
        with pytest.raises(ValueError, match="overlaps"):
            check(LIB.b2_multiply_sum(mixed._h, 6, 1, 1, one_page.ctypes.data, 6, one_page.ctypes.data, 6, at, stream()))
    a = np.array([cache.data.data_ptr(), cache.data.data_ptr() + 8], dtype=np.uint64)
    for n, la, lb, l, match in [(2, 6, 6, 6, "aligned"), (0, 6, 6, 6, "at least"), (1, 5, 6, 6, "below"), (1, 6, 9, 6, "below"), (1, 6, 6, 0, "size_Ql")]:
        with pytest.raises(ValueError, match=match):
            check(LIB.b2_multiply_sum(mixed._h, l, 1, n, a.ctypes.data, la, a.ctypes.data, lb, out.data_ptr(), stream()))
    assert np.array_equal(host(cache.data), before)


# ---- attention over cached pages ------------------------------------------------------------------------------------------------
SLOTS, SCALE = N // 2, 2.0 ** 40
HEADS, D_HEAD = 2, 4
D_TOTAL = HEADS * D_HEAD
PER = SLOTS // D_TOTAL


@pytest.fixture(scope="module")
def kit():
    parms = ph.params(ph.scheme_type.ckks)
    parms.set_poly_modulus_degree(N)
    parms.set_coeff_modulus(ph.create_coeff_modulus(N, [60] + [40] * 7 + [60] * 3))
    parms.set_special_modulus_size(3)
    ctx = ph.context(parms)
    sk = ph.secret_key(ctx, seed=31)
    enc = ph.ckks_encoder(ctx)
    return dict(ctx=ctx, sk=sk, enc=enc, rlk=sk.gen_relinkey(ctx), glk=sk.create_galois_keys(ctx))


def _enc(kit, v, chain=1):
    return kit["sk"].encrypt_symmetric(kit["ctx"], kit["enc"].encode_complex_vector(kit["ctx"], np.asarray(v, dtype=np.complex128), SCALE, chain))


def _dec(kit, ct):
    return np.asarray(kit["enc"].decode_complex_vector(kit["ctx"], kit["sk"].decrypt(kit["ctx"], ct)))


# Noise in a slot: an encryption's or key switch's error polynomial has coefficients of a few units, its slots at most about
# 8 sqrt(N) 3.2 = 1.6e3 units of 2^-40, 2e-9. A key switch divides by the special primes without rounding: each coefficient is off by
# 1/2 + (alpha - 1)/2 = 1.5 units on average (alpha = 3), which in the slots whose root is next to 1 adds up to 1.5 * 2 N / pi *
# |s| <= 1.5 * 2608 * 209 = 8.2e5 units, 7.4e-7 (|s| below 4 sqrt(2 N / 3) there), and j slots further to 1 / j of it. A score takes the
# relinearisation's, summed over d_head = 4 slots, and two rotations', the first doubled: 7 * 7.4e-7 = 5.2e-6. score x V: a score's
# noise, four more key switches', summed over the slots near 1 only (sum 1/j < 9): below 9 * (5.2e-6 + 4 * 7.4e-7) = 7.4e-5.
SCORE_TOL, VALUE_TOL = 6e-6, 1e-4


@pytest.mark.parametrize("pages", [1, 3, 19])
def test_attention_products_over_pages(kit, pages):
    ctx, rlk, glk = kit["ctx"], kit["rlk"], kit["glk"]
    rng = np.random.default_rng(pages)
    q = rng.uniform(-1, 1, (HEADS, D_HEAD))
    K, V = rng.uniform(-1, 1, (2, pages, PER, HEADS, D_HEAD))
    cache = ph.ciphertext_cache(ctx, 1, pages + 4, 2, scale=SCALE)
    cache.allocate(4)
    table = cache.allocate(pages)[::-1]
    for i, p in enumerate(table):
        cache.store(p, _enc(kit, K[i].ravel()))
        cache.store(p, _enc(kit, V[i].ravel()), plane=1)
    cq = _enc(kit, np.tile(q.ravel(), PER))
    scores = ph.cached_qkt(ctx, rlk, glk, cq, cache, table, D_HEAD)
    assert len(scores) == pages and all(s.chain_index() == 2 and s.scale() == SCALE for s in scores)
    want_s = np.einsum("hi,cthi->cth", q, K)
    for i in {0, pages // 2, pages - 1}:
        assert np.max(np.abs(_dec(kit, scores[i]).real.reshape(PER, HEADS, D_HEAD)[:, :, 0] - want_s[i])) < SCORE_TOL
    mask = np.zeros((PER, HEADS, D_HEAD))
    mask[:, :, 0] = 1.0
    mask_pt = kit["enc"].encode_double_vector(ctx, mask.ravel(), float(ctx.primes[ctx.limbs_at(2) - 1]), 2)
    out, launched = kernels_of(ctx, lambda: ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table, mask_pt, D_HEAD, D_TOTAL, PER, plane=1))
    assert launched["multiply_sum"] == 1 and out.chain_index() == 4 and out.scale() == SCALE
    got, want = _dec(kit, out).real, np.einsum("cth,cthi->hi", want_s, V).ravel()
    assert np.max(np.abs(got[:D_TOTAL] - want)) < VALUE_TOL * pages and np.max(np.abs(got[-D_TOTAL:] - want)) < VALUE_TOL * pages
    assert ph.cached_qkt(ctx, rlk, glk, cq, cache, [], D_HEAD) == [] and cache.ciphertexts([]) == []
    if pages == 3:  # the list forms take the pages as they are, and agree
        lists = ph.compute_qkt(ctx, rlk, glk, cq, cache.ciphertexts(table), D_HEAD)
        assert np.max(np.abs(_dec(kit, lists[1]) - _dec(kit, scores[1]))) < SCORE_TOL
        low = ph.mod_switch_to(ctx, cq, 3)  # a query below the pages' level
        deep = ph.cached_qkt(ctx, rlk, glk, low, cache, table, D_HEAD)
        assert deep[0].chain_index() == 4 and np.max(np.abs(_dec(kit, deep[0]) - _dec(kit, scores[0]))) < SCORE_TOL
    for call, match in [(lambda: ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table[1:], mask_pt, D_HEAD, D_TOTAL, PER), "size mismatch"),
                        (lambda: ph.cached_score_times_v(ctx, rlk, glk, [], cache, [], mask_pt, D_HEAD, D_TOTAL, PER), "empty"),
                        (lambda: ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table, mask_pt, 3, D_TOTAL, PER), "d_head"),
                        (lambda: ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table, mask_pt, D_HEAD, D_TOTAL, 5), "positions_per_ct"),
                        (lambda: ph.cached_qkt(ctx, rlk, glk, cq, cache, table, 6), "power of 2"),
                        (lambda: ph.cached_qkt(ctx, rlk, glk, cq, cache, [pages + 9], D_HEAD), "out of range")]:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("log_n,chain,special,bconv", [(12, 4, 1, None), (13, 5, 1, None), (13, 5, 3, "int"), (14, 4, 2, None), (15, 6, 2, "fp"), (16, 5, 2, None), (17, 4, 1, None)])
def test_attention_products_in_every_ring(log_n, chain, special, bconv, monkeypatch):
    """down to the last level the products have room for, in every ring, with and without the batched key switch, against numbers and
    against the lists' forms; a page named twice counts twice"""
    n, slots = 1 << log_n, 1 << (log_n - 1)
    if bconv:
        monkeypatch.setenv("B2_BCONV", bconv)
    heads, d_head = 4, 8
    d_total, per = 32, slots // 32
    steps = {1, 2, 4, -1, -2, -4} | {32 << k for k in range(log_n - 6)}
    parms = ph.params(ph.scheme_type.ckks)
    parms.set_poly_modulus_degree(n)
    parms.set_coeff_modulus(ph.create_coeff_modulus(n, [60] + [40] * (chain - 1) + [60] * special))
    parms.set_special_modulus_size(special)
    parms.set_galois_elts(sorted(ph.get_elts_from_steps(sorted(steps), n)))
    ctx = ph.context(parms)
    sk, enc = ph.secret_key(ctx, seed=log_n), ph.ckks_encoder(ctx)
    rlk, glk = sk.gen_relinkey(ctx), sk.create_galois_keys(ctx)
    rng = np.random.default_rng(log_n)
    top = ctx.size_Q - 3  # four limbs left: q * k, the mask and score x V take three
    encrypt = lambda v: sk.encrypt_symmetric(ctx, enc.encode_double_vector(ctx, v, SCALE, top))
    decrypt = lambda ct: np.asarray(enc.decode_complex_vector(ctx, sk.decrypt(ctx, ct))).real
    q = rng.uniform(-1, 1, (heads, d_head))
    K, V = rng.uniform(-1, 1, (2, 3, per, heads, d_head))
    cache = ph.ciphertext_cache(ctx, top, 3, 2, scale=SCALE)
    for p in cache.allocate(3):
        cache.store(p, encrypt(K[p].ravel()))
        cache.store(p, encrypt(V[p].ravel()), plane=1)
    cq, table = encrypt(np.tile(q.ravel(), per)), [2, 0, 2, 1]
    scores = ph.cached_qkt(ctx, rlk, glk, cq, cache, table, d_head)
    lists = ph.compute_qkt(ctx, rlk, glk, cq, cache.ciphertexts(table), d_head)
    mask = np.zeros((per, heads, d_head))
    mask[:, :, 0] = 1.0
    mask_pt = enc.encode_double_vector(ctx, mask.ravel(), float(ctx.primes[ctx.limbs_at(top + 1) - 1]), top + 1)
    out = ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table, mask_pt, d_head, d_total, per, plane=1)
    plain = ph.score_times_v(ctx, rlk, glk, lists, cache.ciphertexts(table, plane=1), mask_pt, d_head, d_total, per)
    assert out.chain_index() == plain.chain_index() == ctx.size_Q and out.data.shape == plain.data.shape == (2, 1, n)
    # ModDown's floor as above, 2 N / pi * |s| * (1 + (alpha - 1) / 2) units of 2^-40 in the slots next to 1, |s| < 4 sqrt(2 N / 3): a
    # score takes it (2 d_head - 1) times over, a value d_head + 3 times more, over the slots near 1 (sum 1/j < 12); and the rescales
    # of the lists' forms floor, which adds half a unit to each of theirs
    unit = 2 * n / np.pi * 4 * np.sqrt(2 * n / 3) * (1.5 + (special - 1) / 2) * 2.0 ** -40
    score_tol, value_tol = (2 * d_head - 1) * unit, 12 * (3 * d_head + 2) * unit
    want = np.einsum("hi,cthi->cth", q, K[table])
    for i in range(4):
        for ct in (scores[i], lists[i]):
            assert np.max(np.abs(decrypt(ct).reshape(per, heads, d_head)[:, :, 0] - want[i])) < score_tol
    total = np.einsum("cth,cthi->hi", want, V[table]).ravel()
    for ct in (out, plain):
        got = decrypt(ct)
        assert np.max(np.abs(got[:d_total] - total)) < value_tol and np.max(np.abs(got[-d_total:] - total)) < value_tol


def test_a_captured_decoding_step(kit):
    """rotation of the query, its products with the cached keys and values, and a fork of the pages in one graph: replayed, it gives
    what the calls give, for whatever the query and the pages then hold"""
    ctx, enc, rlk, glk = kit["ctx"], kit["enc"], kit["rlk"], kit["glk"]
    rng = np.random.default_rng(19)
    rot = ph.rotary(ctx, [1.0, 0.01], HEADS, D_HEAD, packing="halves")
    cache = ph.ciphertext_cache(ctx, 2, 6, 2, scale=SCALE)
    table = cache.allocate(2)
    fresh = lambda: _enc(kit, rng.uniform(-1, 1, SLOTS), 1)
    low = lambda: _enc(kit, rng.uniform(-1, 1, SLOTS), 2)
    mask = np.zeros((PER, HEADS, D_HEAD))
    mask[:, :, 0] = 1.0
    mask_pt = enc.encode_double_vector(ctx, mask.ravel(), float(ctx.primes[ctx.limbs_at(3) - 1]), 3)
    for p in table:
        cache.store(p, low()), cache.store(p, low(), plane=1)
    q, pos = fresh(), torch.full((PER,), 3, device="cuda")
    copy = cache.allocate(2)

    def step():
        (r,) = rot.forward(enc, [q], pos, galois_key=glk)
        cache.copy(copy, table)
        scores = ph.cached_qkt(ctx, rlk, glk, r, cache, copy, D_HEAD)
        return ph.cached_score_times_v(ctx, rlk, glk, scores, cache, copy, mask_pt, D_HEAD, D_TOTAL, PER, plane=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        q.data.copy_(fresh().data)
        pos.fill_(100 * k)
        cache.store(table[k % 2], low(), plane=k % 2)
        g.replay()
        torch.cuda.synchronize()
        got = out.data.clone()
        cache.data[:, copy] = 0
        assert torch.equal(step().data, got) and bool(got.any())


@pytest.mark.parametrize("packing", ["halves", "interleaved"])
def test_generation_step(kit, packing):
    """keys and values of a few positions rotated and put into pages one after another, the sequence forked, one more position in
    each fork, attention of a rotated query over each, the forks given back, the pool compacted, and attention once more"""
    ctx, enc, rlk, glk = kit["ctx"], kit["enc"], kit["rlk"], kit["glk"]
    rng = np.random.default_rng(17)
    inv_freq = 10000.0 ** (-np.arange(2) / 2)
    rot = ph.rotary(ctx, inv_freq, HEADS, D_HEAD, packing=packing)
    assert rot.positions_per_ct == PER
    cache = ph.ciphertext_cache(ctx, 2, 9, 2, scale=SCALE)
    cache.allocate(2)
    table = cache.allocate(2)  # the first page full up to its last position, the second empty
    first = PER - 2

    def turned(x, p):
        t = p * inv_freq
        c, s = np.cos(t), np.sin(t)
        lo, hi = (x[:, :2], x[:, 2:]) if packing == "halves" else (x[:, ::2], x[:, 1::2])
        a, b = lo * c - hi * s, lo * s + hi * c
        return np.concatenate([a, b], 1) if packing == "halves" else np.stack([a, b], 2).reshape(HEADS, D_HEAD)

    def put(table, p, k, v):
        page, at = table[p // PER], p % PER
        keep = torch.zeros(PER, dtype=torch.bool, device="cuda")
        keep[at] = True
        pos = torch.full((PER,), p, dtype=torch.int64, device="cuda")
        (ck,) = rot.forward(enc, [_enc(kit, np.tile(k.ravel(), PER))], pos, keep=keep, galois_key=glk)
        cache.append(page, ck)
        cv = np.zeros((PER, D_TOTAL))
        cv[at] = v.ravel()
        cache.append(page, _enc(kit, cv.ravel(), 2), plane=1)

    def attend(table, p, q, known):
        (cq,) = rot.forward(enc, [_enc(kit, np.tile(q.ravel(), PER))], torch.full((PER,), p, device="cuda"), galois_key=glk)
        scores = ph.cached_qkt(ctx, rlk, glk, cq, cache, table, D_HEAD)
        mask = np.zeros((PER, HEADS, D_HEAD))
        mask[:, :, 0] = 1.0
        mask_pt = enc.encode_double_vector(ctx, mask.ravel(), float(ctx.primes[ctx.limbs_at(3) - 1]), 3)
        out = ph.cached_score_times_v(ctx, rlk, glk, scores, cache, table, mask_pt, D_HEAD, D_TOTAL, PER, plane=1)
        want = sum(np.einsum("hi,hi->h", turned(q, p), turned(k, j))[:, None] * v for j, (k, v) in known.items())
        assert np.max(np.abs(_dec(kit, out)[:D_TOTAL].real - want.ravel())) < VALUE_TOL

    draw = lambda: rng.uniform(-1, 1, (HEADS, D_HEAD))
    known = {}
    for p in range(first, first + 3):  # crosses from one page into the next
        known[p] = draw(), draw()
        put(table, p, *known[p])
    forks, seen = cache.fork(table, copies=2), []
    for f in forks:
        seen.append({**known, first + 3: (draw(), draw())})
        put(f, first + 3, *seen[-1][first + 3])
    q = draw()
    for f, s in zip(forks, seen):
        attend(f, first + 4, q, s)
    attend(table, first + 3, q, known)
    cache.free(forks[0])
    cache.free([0, 1])
    table, fork = cache.compact([table, forks[1]])
    assert table == [0, 1] and fork == [0, 2] and cache.free_pages() == 6
    cache.resize(3)
    attend(fork, first + 4, q, seen[1])
    attend(table, first + 3, q, known)
