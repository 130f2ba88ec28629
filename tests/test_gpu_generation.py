"""Generation with an encrypted model: calls that the operators' documentation allows and their first tests do not make."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import pyPhantom as ph


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
