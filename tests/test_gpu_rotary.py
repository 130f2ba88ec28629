"""Rotary factors against the formula in 64 bits, in every slot, and rotated ciphertexts against rotated vectors."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import pyPhantom as ph
from pyPhantom._native import LIB, check
from gpu_helpers import stream

# A sine or cosine is within 2 units in the last place on the device and 1 on the host, for the same (rounded) angle; the factor's
# product with the scaling rounds once more, on either side. Units in the last place of values up to 1 are at most 2^-53.
TOL = 4 * 2.0 ** -53


def _ctx(log_n, special=1, chain=(60, 40, 40, 40)):
    parms = ph.params(ph.scheme_type.ckks)
    parms.set_poly_modulus_degree(1 << log_n)
    parms.set_coeff_modulus(ph.create_coeff_modulus(1 << log_n, list(chain) + [60] * special))
    parms.set_special_modulus_size(special)
    return ph.context(parms)


@pytest.fixture(scope="module")
def ctx():
    return _ctx(12)


def _formula(slots, positions, inv_freq, heads, d_head, axes, packing, scaling=1.0, keep=None, conjugate=False):
    """positions [tokens][axes] as numpy; every slot by itself"""
    r, T, width = len(inv_freq), len(positions), heads * d_head
    per = slots // width
    n = -(-T // per)
    out = np.zeros((1 if packing == "pairs" else 3, n, slots), dtype=np.complex128)
    for t in range(T):
        if keep is not None and not keep[t]:
            continue
        theta = [float(np.float64(positions[t][axes[j]]) * np.float64(inv_freq[j])) for j in range(r)]
        c = [scaling * math.cos(v) for v in theta]
        s = [(-scaling if conjugate else scaling) * math.sin(v) for v in theta]
        head = np.zeros((len(out), d_head), dtype=np.complex128)
        head[0] = 1.0
        for j in range(r):
            if packing == "pairs":
                head[0, j] = complex(c[j], s[j])
            else:
                x, y = (j, j + r) if packing == "halves" else (2 * j, 2 * j + 1)
                head[:, x], head[:, y] = (c[j], -s[j], 0), (c[j], 0, s[j])
        at = t % per * width
        out[:, t // per, at:at + width] = np.tile(head, (1, heads))
    return out


def _check(got, want, scaling=1.0):
    got = got.cpu().numpy()
    assert got.shape == want.shape
    assert np.max(np.abs(np.stack([got.real - want.real, got.imag - want.imag])), initial=0.0) <= TOL * abs(scaling)
    assert np.array_equal(got == 0, want == 0)  # slots of no position, and the zeros of A and B


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
@pytest.mark.parametrize("heads,d_head,pairs", [(1, 2, 1), (4, 8, 4), (3, 10, 5), (2, 64, 9), (8, 16, 8), (5, 200, 100), (1, 300, 150), (1, 2048, 1024), (7, 256, 3)])
def test_layouts(ctx, packing, heads, d_head, pairs):
    """heads shorter and longer than a CTA, widths that leave slots over, pairs that leave elements over; the last ciphertext part full"""
    rng = np.random.default_rng(heads * d_head)
    per = 2048 // (heads * d_head)
    f = 10000.0 ** (-np.arange(pairs) / pairs)
    rot = ph.rotary(ctx, f, heads, d_head, packing=packing)
    assert rot.positions_per_ct == per
    for tokens in sorted({1, per, per + 1, 2 * per + max(1, per // 3)}):
        if tokens > 200:
            continue
        p = rng.integers(0, 5000, (tokens, 1))
        got = rot.factors(torch.from_numpy(p).cuda())
        _check(got, _formula(2048, p, f, heads, d_head, [0] * pairs, packing))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("axes", [1, 2, 3])
def test_axes_types_and_strides(ctx, dtype, axes):
    rng = np.random.default_rng(axes)
    pairs, tokens = 6, 21
    which = [int(a) for a in rng.integers(0, axes, pairs)]
    which[0] = axes - 1
    f = 1.0 / (1.0 + np.arange(pairs)) ** 2
    p = rng.integers(-300, 30000, (tokens, axes)).astype(np.float64) / (1 if not dtype.is_floating_point else 8)
    rot = ph.rotary(ctx, f, 4, 12, axes=which, packing="halves")
    plain = torch.from_numpy(p).to(dtype).cuda()
    want = _formula(2048, plain.cpu().numpy(), f, 4, 12, which, "halves")
    wide = torch.full((tokens * 3, axes * 2 + 1), 9, dtype=dtype, device="cuda")
    wide[1::3, 1::2] = plain
    across = plain.t().contiguous().t()
    for x in (plain, wide[1::3, 1::2], across):
        _check(rot.factors(x), want)
    if axes == 1:
        _check(rot.factors(plain[:, 0]), want)
        _check(rot.factors(plain[:1].expand(tokens, 1)), _formula(2048, plain[:1].expand(tokens, 1).cpu().numpy(), f, 4, 12, which, "halves"))


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
def test_dropped_positions(ctx, packing):
    """none kept, all kept, some kept; what stands in a dropped position's place does not matter"""
    rng = np.random.default_rng(3)
    f = np.array([1.0, 0.01])
    rot = ph.rotary(ctx, f, 16, 8, packing=packing)
    p = rng.uniform(0, 100, (37, 1))
    for keep in (np.zeros(37, dtype=bool), np.ones(37, dtype=bool), rng.random(37) < 0.5):
        x = p.copy()
        x[~keep] = rng.choice([np.inf, -np.inf, np.nan, 1e300], ((~keep).sum(), 1))
        wide = torch.zeros(37, 2, dtype=torch.bool, device="cuda")
        wide[:, 1] = torch.from_numpy(keep)
        want = _formula(2048, x, f, 16, 8, [0, 0], packing, keep=keep)
        _check(rot.factors(torch.from_numpy(x).cuda(), keep=wide[:, 1]), want)
        assert not keep.any() or want.any()


@pytest.mark.parametrize("packing", ["pairs", "interleaved"])
def test_inverse_and_scaling(ctx, packing):
    f = np.array([1.0, 0.25, 1e-4])
    p = np.arange(9).reshape(9, 1)
    for scaling in (1.0, 1.3, -0.5):
        rot = ph.rotary(ctx, f, 2, 9, packing=packing, scaling=scaling)
        for conj in (False, True):
            _check(rot.factors(torch.from_numpy(p).cuda(), conjugate=conj), _formula(2048, p, f, 2, 9, [0] * 3, packing, scaling, conjugate=conj), max(1.0, abs(scaling)))


def test_far_positions(ctx):
    """angles far beyond where a short reduction of the argument holds"""
    f = np.array([1.0, 0.7310585786300049, 1e-3, 12345.678])
    p = np.array([[0], [1], [-1], [105615], [105616], [1 << 20], [1 << 31], [(1 << 53) - 1], [-(1 << 60)]])
    rot = ph.rotary(ctx, f, 1, 4)
    _check(rot.factors(torch.from_numpy(p).cuda()), _formula(2048, p, f, 1, 4, [0] * 4, "pairs"))


def test_no_positions_and_largest_ring():
    c = _ctx(17, chain=(60, 40))
    rot = ph.rotary(c, [1.0, 0.5], 4, 4, packing="halves")
    assert rot.factors(torch.zeros(0, 1, dtype=torch.int64, device="cuda")).shape == (3, 0, 1 << 16)
    enc = ph.ckks_encoder(c)
    assert rot.encode(enc, rot.factors(torch.zeros(0, dtype=torch.int64, device="cuda")), 1) == [[], [], []]
    p = np.arange(4099).reshape(-1, 1)  # two ciphertexts, the second nearly empty
    got = rot.factors(torch.from_numpy(p).cuda()).cpu().numpy()
    want = _formula(1 << 16, p, [1.0, 0.5], 4, 4, [0, 0], "halves")
    assert np.max(np.abs(got - want)) <= 2 * TOL and np.array_equal(got == 0, want == 0)


def test_captured_and_on_other_streams(ctx):
    f = np.array([1.0, 0.5, 0.25, 0.125])
    rot = ph.rotary(ctx, f, 4, 8, packing="halves")
    p = torch.arange(64, device="cuda").reshape(64, 1)
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot.factors(p, keep)
    torch.cuda.current_stream().wait_stream(side)
    want = _formula(2048, p.cpu().numpy(), f, 4, 8, [0] * 4, "halves")
    _check(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rot.factors(p, keep)
    for k in range(3):
        p.add_(1000 + k)
        keep[k] = False
        g.replay()
        _check(out, _formula(2048, p.cpu().numpy(), f, 4, 8, [0] * 4, "halves", keep=keep.cpu().numpy()))


def test_what_is_refused(ctx):
    good = dict(inv_freq=[1.0, 0.5], heads=4, d_head=8)
    for bad, match in [(dict(packing="thirds"), "packing"), (dict(heads=0), "heads"), (dict(d_head=0), "heads"), (dict(heads=257), "heads"),
                       (dict(inv_freq=[]), "pairs"), (dict(inv_freq=[1.0] * 9), "pairs"), (dict(inv_freq=[1.0] * 5, packing="halves"), "pairs"),
                       (dict(axes=[0]), "axis"), (dict(axes=[0, -1]), "axis")]:
        with pytest.raises(ValueError, match=match):
            ph.rotary(ctx, **{**good, **bad})
    rot = ph.rotary(ctx, **good, axes=[0, 2])
    p = torch.zeros(5, 3, dtype=torch.int64, device="cuda")
    for args, match in [((p[:, :2],), "axes"), ((p.to(torch.int16),), "int32"), ((p[None],), "positions"), ((p.cpu(),), "device"),
                        ((p, torch.ones(4, dtype=torch.bool, device="cuda")), "truth value"), ((p, torch.ones(5, device="cuda")), "truth value"),
                        ((p, torch.ones(5, dtype=torch.bool)), "device")]:
        with pytest.raises(ValueError, match=match):
            rot.factors(*args)
    enc = ph.ckks_encoder(ctx)
    fac = rot.factors(p)
    for args, match in [((enc, fac[0], 1), "factors"), ((enc, fac.real, 1), "factors"), ((enc, fac, 0), "chain index"), ((enc, fac, 4), "end of modulus"),
                        ((enc, fac, 9), "chain index")]:
        with pytest.raises(ValueError, match=match):
            rot.encode(*args)
    with pytest.raises(ValueError, match="as many"):
        rot.apply([], rot.encode(enc, fac, 1))
    other = _ctx(13)
    with pytest.raises(ValueError, match="another context"):
        rot.encode(ph.ckks_encoder(other), fac, 1)
    with pytest.raises(ValueError, match="scale out of bounds"):
        ph.rotary(ctx, [1.0], 4, 8, scaling=1e9).encode(enc, fac, 1)
    out = torch.empty(4096, dtype=torch.complex128, device="cuda")

    def c_entry(packing=0, tokens=1, heads=4, d_head=8, pairs=2, pos=p.data_ptr(), kind=1, out=out.data_ptr()):
        check(LIB.b2_rotary_factors(ctx._h, packing, tokens, heads, d_head, pairs, pos, kind, 3, 1, rot.inv_freq.data_ptr(), rot.axes.data_ptr(), 0, 0, 1.0, 0,
                                    out, stream()))

    for kw, match in [(dict(packing=3), "packing"), (dict(kind=4), "type"), (dict(heads=1 << 40, d_head=1 << 40), "slots"), (dict(heads=257), "slots"),
                      (dict(pairs=0), "pairs"), (dict(pairs=9), "pairs"), (dict(pairs=5, packing=2), "pairs"), (dict(pos=0), "null"), (dict(out=out.data_ptr() + 8), "aligned"), (dict(pos=p.data_ptr() + 4), "aligned"),
                      (dict(tokens=1 << 40), "2\\^30")]:
        with pytest.raises(ValueError, match=match):
            c_entry(**kw)
    c_entry(tokens=0, pos=0, out=0)


@pytest.fixture(scope="module")
def kit():
    c = _ctx(13, special=2, chain=(60, 40, 40, 40))
    sk = ph.secret_key(c, seed=5)
    return dict(ctx=c, sk=sk, enc=ph.ckks_encoder(c), glk=sk.create_galois_keys(c))


# An encryption's error is at most about 8 sqrt(N) 3.2 = 2.3e3 units of 2^-40 in a slot, a key switch's and a rescale's about as much
# (half a unit a coefficient times the ternary secret); factors are rounded at 2^40, half a unit a coefficient: sqrt(N) units. Five
# such terms with factors up to 1: 1.2e4 units, 1.1e-8.
# A key switch divides by the special primes as the reference does, without rounding: each coefficient is off by 1/2 + (alpha - 1)/2
# = 1 unit on average for alpha = 2 special primes. An offset m in every coefficient is m sum_k zeta^k in a slot, m 2 N / pi = 5.2e3
# units where the slot's root zeta is next to 1, and in the second polynomial that times |s(zeta)|, below 4 sqrt(2 N / 3) = 296 for a
# ternary secret of N = 8192: 1.5e6 units, 1.4e-6. A slot takes one of the two rotations (A and B do not overlap).
CT_TOL = {"pairs": 1e-7, "halves": 1.5e-6, "interleaved": 1.5e-6}


@pytest.mark.parametrize("vectors", [1, 3, 17])
def test_batch_of_encodings_is_the_single_ones(kit, vectors):
    ctx, enc = kit["ctx"], kit["enc"]
    n = ctx.N // 2
    z = torch.randn(vectors, n, dtype=torch.complex128, device="cuda", generator=torch.Generator("cuda").manual_seed(vectors))
    one, many = (torch.empty(vectors, ctx.N, dtype=torch.int64, device="cuda") for _ in range(2))
    for k in range(vectors):
        check(LIB.b2_encode_coeffs(ctx._h, z[k].clone().data_ptr(), enc._d_rot.data_ptr(), enc._d_ksi.data_ptr(), 2.0 ** 30 / n, one[k].data_ptr(), stream()))
    check(LIB.b2_encode_coeffs_batch(ctx._h, vectors, z.data_ptr(), enc._d_rot.data_ptr(), enc._d_ksi.data_ptr(), 2.0 ** 30 / n, many.data_ptr(), stream()))
    assert torch.equal(one, many) and bool(one.any())
    with pytest.raises(ValueError, match="bad argument"):
        check(LIB.b2_encode_coeffs_batch(ctx._h, 0, z.data_ptr(), enc._d_rot.data_ptr(), enc._d_ksi.data_ptr(), 1.0, many.data_ptr(), stream()))


def test_more_ciphertexts_than_go_together(kit):
    """the ciphertexts of a long prompt, 16 at a time, are each what they are alone"""
    ctx, enc, sk = kit["ctx"], kit["enc"], kit["sk"]
    rot = ph.rotary(ctx, [1.0, 0.1], 64, 16, packing="interleaved")
    n = 19
    x = sk.encrypt_symmetric(ctx, enc.encode_double_vector(ctx, np.random.default_rng(1).uniform(-1, 1, ctx.N // 2), 2.0 ** 40, 3))
    pos = torch.arange(n * rot.positions_per_ct - 1, device="cuda")
    out = rot.forward(enc, [x] * n, pos, galois_key=kit["glk"])
    assert len(out) == n
    for i in (0, 15, 16, n - 1):
        per = rot.positions_per_ct
        (alone,) = rot.forward(enc, [x], pos[i * per:(i + 1) * per], galois_key=kit["glk"])
        assert torch.equal(alone.data, out[i].data)
    assert rot.forward(enc, [], pos[:0], galois_key=kit["glk"]) == []


@pytest.mark.parametrize("packing,d_head,pairs", [("pairs", 8, 8), ("pairs", 12, 5), ("halves", 16, 8), ("halves", 20, 8), ("interleaved", 16, 8), ("interleaved", 10, 4)])
def test_rotated_ciphertexts(kit, packing, d_head, pairs):
    ctx, enc, sk = kit["ctx"], kit["enc"], kit["sk"]
    rng = np.random.default_rng(d_head)
    heads, slots = 8, ctx.N // 2
    f = 10000.0 ** (-np.arange(pairs) / pairs)
    axes = [j % 2 for j in range(pairs)]
    rot = ph.rotary(ctx, f, heads, d_head, axes=axes, packing=packing)
    per, width = rot.positions_per_ct, heads * d_head
    tokens = 2 * per - 3  # three places of the second ciphertext are dropped: they hold no position
    p = rng.integers(0, 4000, (tokens, 2))
    x = rng.uniform(-1, 1, (2 * per, heads, d_head)) + (1j * rng.uniform(-1, 1, (2 * per, heads, d_head)) if packing == "pairs" else 0)
    vec = np.zeros((2, slots), dtype=np.complex128)
    vec[:, :per * width] = x.reshape(2, -1)
    cts = [sk.encrypt_symmetric(ctx, enc.encode_complex_vector(ctx, v, 2.0 ** 40, 2)) for v in vec]
    glk = None if packing == "pairs" else kit["glk"]
    tol = CT_TOL[packing]
    theta = p[:, axes] * f
    z = np.exp(1j * theta)[:, None, :]
    want = np.zeros_like(x)
    want[:tokens] = x[:tokens]
    if packing == "pairs":
        want[:tokens, :, :pairs] = x[:tokens, :, :pairs] * z
    else:
        lo, hi = (slice(0, pairs), slice(pairs, 2 * pairs)) if packing == "halves" else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
        y = (x[:tokens, :, lo] + 1j * x[:tokens, :, hi]) * z
        want[:tokens, :, lo], want[:tokens, :, hi] = y.real, y.imag
    pos = torch.from_numpy(p).cuda()
    if packing != "pairs":
        with pytest.raises(ValueError, match="Galois key"):
            rot.forward(enc, cts, pos)
    with pytest.raises(ValueError, match="positions for"):
        rot.forward(enc, cts[:1], pos, galois_key=glk)
    with pytest.raises(ValueError, match="mismatch"):  # factors of another level
        rot.apply(cts, rot.encode(enc, rot.factors(pos), 1), glk)
    with pytest.raises(ValueError, match="mismatch"):  # ciphertexts of two levels
        rot.forward(enc, [cts[0], ph.mod_switch_to_next(ctx, cts[1])], pos, galois_key=glk)
    out = rot.forward(enc, cts, pos, galois_key=glk)
    for i, ct in enumerate(out):
        assert ct.chain_index() == 3 and ct.scale() == 2.0 ** 40
        got = enc.decode_complex_vector(ctx, sk.decrypt(ctx, ct))
        assert np.max(np.abs(got[:per * width] - want.reshape(2, -1)[i])) < tol and np.max(np.abs(got[per * width:]), initial=0.0) < tol
    back = rot.forward(enc, out, pos, conjugate=True, galois_key=glk)  # the inverse brings them back
    want = x.copy()
    want[tokens:] = 0
    got = np.stack([enc.decode_complex_vector(ctx, sk.decrypt(ctx, ct)) for ct in back])[:, :per * width]
    assert np.max(np.abs(got - want.reshape(2, -1))) < 2 * tol
