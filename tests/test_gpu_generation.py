"""Generation with an encrypted model: calls that the operators' documentation allows and their first tests do not make."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import pyPhantom as ph
from pyPhantom._native import LIB, check
from gpu_helpers import stream


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
