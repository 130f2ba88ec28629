"""Generation with an encrypted model: calls that the operators' documentation allows and their first tests do not make."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import pyPhantom as ph
from pyPhantom._native import LIB, check
from gpu_helpers import stream
from test_gpu_cache import MIXED, _below, _ct, _ctx, _residues


@pytest.fixture(scope="module")
def kit():
    parms = ph.params(ph.scheme_type.ckks)
    parms.set_poly_modulus_degree(8192)
    parms.set_coeff_modulus(ph.create_coeff_modulus(8192, [60, 40, 40, 40] + [60] * 2))
    parms.set_special_modulus_size(2)
    ctx = ph.context(parms)
    sk = ph.secret_key(ctx, seed=5)
    return dict(ctx=ctx, sk=sk, enc=ph.ckks_encoder(ctx), glk=sk.create_galois_keys(ctx))


def _encrypt(kit, rng, chain):
    ctx = kit["ctx"]
    return kit["sk"].encrypt_symmetric(ctx, kit["enc"].encode_double_vector(ctx, rng.uniform(-1, 1, ctx.N // 2), 2.0 ** 40, chain))


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
def test_rotated_views(kit, packing):
    """the first limbs of a higher level, as a view whose polynomials lie apart, rotate to the words that a dense copy rotates to"""
    ctx, enc = kit["ctx"], kit["enc"]
    rng = np.random.default_rng(1)
    high = [_encrypt(kit, rng, 1) for _ in range(3)]
    views = [x._like(x.data[:, :3], chain_index=2) for x in high]
    assert not any(v.data.is_contiguous() for v in views)
    dense = [v._like(v.data.contiguous()) for v in views]
    rot = ph.rotary(ctx, [1.0, 0.1], 8, 16, packing=packing)
    pos = torch.arange(3 * rot.positions_per_ct, device="cuda")
    got = rot.forward(enc, views, pos, galois_key=kit["glk"])
    want = rot.forward(enc, dense, pos, galois_key=kit["glk"])
    for g, w in zip(got, want):
        assert torch.equal(g.data, w.data) and bool(g.data.any())


def test_plain_sums_onto_their_operands(kit):
    """the result of a batch may not lie on what a later launch of it still reads"""
    ctx, l = kit["ctx"], 2
    one = 8 * ctx.N
    pool = torch.zeros(8, l, ctx.N, dtype=torch.int64, device="cuda")
    at = pool.data_ptr()

    def call(out, cts, pts):
        a, b = (np.array(v, dtype=np.uint64) for v in (cts, pts))
        check(LIB.b2_multiply_plain_sum(ctx._h, l, len(a), 1, a.ctypes.data, b.ctypes.data, out, stream()))

    poly = lambda k: at + k * l * one  # a ciphertext takes two, a plaintext one, the two results four
    for out, cts, pts in [(0, [4, 3], [6, 7]), (2, [0, 1], [6, 7]), (0, [4, 4], [6, 3]), (4, [0, 2], [4, 3]), (0, [2, 4], [6, 7])]:
        with pytest.raises(ValueError, match="overlaps"):
            call(poly(out), [poly(k) for k in cts], [poly(k) for k in pts])
    with pytest.raises(ValueError, match="overlaps"):  # by a little
        call(poly(0), [poly(4), poly(4) - 32], [poly(6), poly(7)])
    call(poly(0), [poly(4)] * 2, [poly(6), poly(7)])
    call(poly(4), [poly(2)] * 2, [poly(0), poly(3)])
    assert not bool(pool.any())


def test_positions_that_torch_negates_on_the_fly(kit):
    """the imaginary part of a conjugate is a view with a bit instead of a sign"""
    rot = ph.rotary(kit["ctx"], [1.0, 0.1], 8, 16)
    z = torch.complex(torch.zeros(5, dtype=torch.float64, device="cuda"), torch.arange(5, dtype=torch.float64, device="cuda"))
    p = z.conj().imag
    assert p.is_neg()
    assert torch.equal(rot.factors(p), rot.factors(p.clone())) and not torch.equal(rot.factors(p), rot.factors(z.imag))


# ---- what the host looks at, and what it cannot while a graph is captured ---------------------------------------------------------
@pytest.mark.parametrize("packing", ["pairs", "interleaved"])
def test_factors_and_plaintexts_that_are_refused(kit, packing):
    ctx, enc, rng = kit["ctx"], kit["enc"], np.random.default_rng(2)
    rot = ph.rotary(ctx, [1.0, 0.1], 8, 16, packing=packing)
    x, pos = _encrypt(kit, rng, 2), torch.arange(rot.positions_per_ct, dtype=torch.float64, device="cuda")
    good = rot.factors(pos)
    for value in (1e9, float("nan"), complex(0, float("inf"))):
        bad = good.clone()
        bad[-1, 0, 5] = value
        with pytest.raises(ValueError, match="too large"):
            rot.encode(enc, bad, 2)
    plain = [[enc.encode_complex_vector(ctx, v.cpu().numpy(), 2.0 ** 40, 2) for v in vec] for vec in good]
    with pytest.raises(ValueError, match="scale mismatch"):
        rot.apply([x], plain, kit["glk"])
    at_prime = [[enc.encode_complex_vector(ctx, v.cpu().numpy(), float(ctx.primes[2]), 2) for v in vec] for vec in good]
    (y,) = rot.apply([x], at_prime, kit["glk"])
    (z,) = rot.forward(enc, [x], pos, galois_key=kit["glk"])
    assert y.scale() == z.scale() == 2.0 ** 40 and torch.equal(y.data, z.data)  # the same coefficients, one vector after another
    keep = torch.ones(len(pos), dtype=torch.bool, device="cuda")
    pos[3], keep[3] = float("nan"), False
    rot.forward(enc, [x], pos, keep=keep, galois_key=kit["glk"])
    with pytest.raises(ValueError, match="finite"):
        rot.forward(enc, [x], pos, galois_key=kit["glk"])


def test_captured_rotations(kit):
    """factors, encode and apply, and forward with positions in floating point, in one graph: nothing waits for the device"""
    ctx, enc, rng = kit["ctx"], kit["enc"], np.random.default_rng(3)
    rot = ph.rotary(ctx, [1.0, 0.1], 8, 16, packing="halves")
    x, pos = _encrypt(kit, rng, 2), torch.arange(rot.positions_per_ct, dtype=torch.float64, device="cuda")

    def call():
        (y,) = rot.apply([x], rot.encode(enc, rot.factors(pos), 2), kit["glk"])
        (z,) = rot.forward(enc, [x], pos, galois_key=kit["glk"])
        return y.data, z.data

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, z = call()
    for _ in range(2):
        pos.add_(0.5)
        g.replay()
        assert torch.equal(y, z) and all(torch.equal(a, y) for a in call())


def test_resized_on_another_stream(kit):
    """the pages that stay keep their words where the pool was made on one stream and is resized, and given back, on another"""
    ctx = kit["ctx"]
    cache = ph.ciphertext_cache(ctx, 1, 40, 2)
    table = cache.allocate(20)
    mark = torch.arange(1, 21, device="cuda")[:, None, None, None]
    cache.data[:, :20] = mark
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for pages in (30, 25, 50, 20):
            cache.resize(pages)
    torch.full((2, 40, 2, 4, ctx.N), 77, dtype=torch.int64, device="cuda")  # what would take the memory given back
    torch.cuda.current_stream().wait_stream(side)
    assert cache.pages() == len(table) == 20 and bool((cache.data == mark).all())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.copy([0], [1])
        with pytest.raises(RuntimeError, match="captured"):
            cache.resize(30)
    g.replay()
    assert cache.pages() == 20 and bool((cache.data[:, 0] == 2).all())


# ---- several queries in every arithmetic ------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def pool():
    """three scores and three pages of the eight primes of every arithmetic (61 to 30 bits), the first of each the largest residues
    throughout, and the nine products of a score and a page in integers of any size"""
    ctx = _ctx(MIXED + _below(60, 2)[1:])
    rng = np.random.default_rng(21)
    q = np.array(MIXED, dtype=object)[:, None]
    sides = []
    for _ in range(2):
        x = _residues(rng, ctx, 3, 2, 8)
        x[0] = ctx.primes[:8].astype(np.uint64)[:, None] - np.uint64(1)
        sides.append(x)
    a, b = (x.astype(object) for x in sides)
    products = [[[u[0] * v[0] % q, (u[0] * v[1] + u[1] * v[0]) % q, u[1] * v[1] % q] for v in b] for u in a]
    return ctx, q, [_ct(ctx, x) for x in sides[0]], sides[1], products


@pytest.mark.parametrize("queries", [1, 2, 3, 4, 5, 7])
@pytest.mark.parametrize("terms", [1, 7, 8, 9, 15, 30, 60, 61, 64, 65, 129])
def test_long_sums_of_several_queries(pool, queries, terms):
    """past what the sums in registers take before they are brought back (7 products below 2^50, 60 below 2^41, 8 and 31 above) and
    into a second and third launch, which add to the first one's results. The first query's operands are the largest residues in
    every term, the others' are drawn for every term of every query: an operand read in another's place shows"""
    ctx, q, scores, pages, products = pool
    rng = np.random.default_rng(100 * queries + terms)
    cache = ph.ciphertext_cache(ctx, 1, 5)
    cache.allocate(5)
    held = [0, 1, 2, 0, 1]
    for p, k in enumerate(held):
        cache.data[0, p].copy_(torch.from_numpy(pages[k].view(np.int64)))
    for largest in (True, False):
        pick = rng.integers(0, 3, (queries, terms))
        table = [0] * terms if largest else [int(p) for p in rng.integers(0, 5, terms)]
        if largest:
            pick[0] = 0
        got = cache.multiply_sum([[scores[k] for k in row] for row in pick], table)
        assert len(got) == queries
        for g in range(queries):
            count = np.zeros((3, 3), dtype=int)
            np.add.at(count, (pick[g], [held[p] for p in table]), 1)
            for p in range(3):
                want = sum(int(count[i, j]) * products[i][j][p] for i in range(3) for j in range(3) if count[i, j]) % q
                assert np.array_equal(got[g].numpy()[p], want.astype(np.uint64)), (largest, g, p)
