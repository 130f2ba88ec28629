"""What rotary gives its kernels, and what it refuses, without a GPU: the native calls are replaced by ones that read the addresses
that they are given the way the kernels do."""
import ctypes
import importlib
import math
import types

import numpy as np
import pytest
import torch

import pyPhantom as ph
from pyPhantom import _native, rotary as rotary_class
from pyPhantom import cache as cache_module

rotary_module = importlib.import_module("pyPhantom.rotary")
N, PRIME = 16, 1099511480321


def _words(address, count):
    return np.ctypeslib.as_array((ctypes.c_int64 * count).from_address(address)).copy()


class _Native:
    """the entries that rotated ciphertexts take; every ciphertext and plaintext that the products read is kept in `read`"""

    def __init__(self):
        self.read, self.calls = [], []

    def b2_multiply_plain_sum(self, h, l, n, terms, cts, pts, out, stream):
        self.calls.append("sum")
        cts, pts = ((ctypes.c_uint64 * (n * terms)).from_address(a) for a in (cts, pts))
        self.read.append([(_words(c, 2 * l * N), _words(p, l * N)) for c, p in zip(cts, pts)])
        return 0

    def b2_rescale_rounded_batch(self, *args):
        return 0

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append(name)
            return 0

        return entry


def _context(size_Q=4, bits=40):
    ctx = types.SimpleNamespace(N=N, size_Q=size_Q, device=-1, _h=None, primes=np.full(size_Q + 1, PRIME, dtype=np.uint64),
                                chain_bits=[bits * k for k in range(size_Q + 2)])
    ctx.limbs_at = lambda k: size_Q - (k - 1)
    ctx.empty = lambda *shape: torch.zeros((*shape, N), dtype=torch.int64)
    return ctx


@pytest.fixture
def native(monkeypatch):
    lib = _Native()
    for module in (rotary_module, cache_module):
        monkeypatch.setattr(module, "LIB", lib)
        monkeypatch.setattr(module, "_stream", lambda: 0)
    monkeypatch.setattr(_native, "_current_device", lambda: -1)

    def hoist(ctx, ct, glk, steps):  # reads two dense polynomials behind the address, as the kernel does
        x = torch.from_numpy(_words(ct.data.data_ptr(), 2 * ct._limbs * N)).reshape(2, ct._limbs, N)
        return [ct._like(x + 1000 * s) for s in steps]

    monkeypatch.setattr(rotary_module, "hoist_rotations", hoist)
    return lib


def _rotary(ctx, packing, scaling=1.0):
    rot = object.__new__(rotary_class)  # without the tables, which lie on a device
    rot.ctx, rot.packing, rot.scaling, rot._vecs, rot.step = ctx, packing, scaling, 1 if packing == "pairs" else 3, 1
    return rot


def _ciphertext(data, chain):
    ct = ph.ciphertext()
    ct._chain_index, ct._size, ct._limbs, ct._N, ct._scale, ct.data = chain, data.shape[0], data.shape[1], N, 2.0 ** 40, data
    return ct


def _plaintext(data, chain, scale=float(PRIME)):
    pt = ph.plaintext()
    pt._chain_index, pt._N, pt._limbs, pt._scale, pt.data = chain, N, data.shape[0], scale, data
    return pt


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
@pytest.mark.parametrize("n", [1, 3, 17])
def test_words_that_the_products_read(native, packing, n):
    """ciphertexts whose polynomials lie apart (the first limbs of a higher level) count as what they hold, rotated or not"""
    ctx, l = _context(), 3
    rot = _rotary(ctx, packing)
    high = torch.arange(n * 2 * 4 * N).reshape(n, 2, 4, N)
    xs = [_ciphertext(x[:, :l] if i % 2 == 0 else x[:, :l].clone(), 2) for i, x in enumerate(high)]
    pts = [[_plaintext(torch.full((l, N), 100 * v + i), 2) for i in range(n)] for v in range(rot._vecs)]
    out = rot.apply(xs, pts, galois_key="key")
    assert len(out) == n and all(ct.chain_index() == 3 and ct.scale() == 2.0 ** 40 for ct in out)
    read = [pair for call in native.read for pair in call]
    assert len(read) == n * rot._vecs
    for i in range(n):
        for v, offset in zip(range(rot._vecs), (0, 1000, -1000)):
            ct, pt = read[i * rot._vecs + v]
            assert np.array_equal(ct, high[i, :, :l].reshape(-1).numpy() + offset)
            assert np.array_equal(pt, np.full(l * N, 100 * v + i))


def _no_call(native, call, match):
    with pytest.raises(ValueError, match=match):
        call()
    assert native.calls == [] and native.read == []


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.int32, torch.float64, torch.uint8])
def test_plaintext_words_of_another_type(native, packing, dtype):
    """words shorter than the kernel's would be read past their end"""
    ctx, l = _context(), 3
    rot = _rotary(ctx, packing)
    xs = [_ciphertext(torch.zeros(2, l, N, dtype=torch.int64), 2) for _ in range(2)]
    pts = [[_plaintext(torch.zeros(l, N, dtype=torch.int64), 2) for _ in range(2)] for _ in range(rot._vecs)]
    pts[-1][1].data = torch.zeros(l, N, dtype=dtype)
    _no_call(native, lambda: rot.apply(xs, pts, "key"), "mismatch")


@pytest.mark.parametrize("dtype", [torch.int32, torch.float64, torch.uint8])
def test_mask_words_of_another_type(native, dtype):
    ctx = _context()
    cache = ph.ciphertext_cache(ctx, 1, 2)
    cache._held, cache._free = [1, 1], []
    score = _ciphertext(torch.zeros(2, 4, N, dtype=torch.int64), 1)
    mask = _plaintext(torch.zeros(4, N, dtype=dtype), 1)
    _no_call(native, lambda: ph.cached_score_times_v(ctx, None, None, [score], cache, [0], mask, 2, 4, 2), "mismatch")


@pytest.mark.parametrize("packing", ["pairs", "halves", "interleaved"])
@pytest.mark.parametrize("scale", [2.0 ** 40, 2.0 ** 30, PRIME * 1.001, float("nan")])
def test_plaintexts_at_another_scale(native, packing, scale):
    """the rescale removes the prime: a result at the ciphertext's scale comes from plaintexts at the prime's"""
    ctx, l = _context(), 3
    rot = _rotary(ctx, packing)
    xs = [_ciphertext(torch.zeros(2, l, N, dtype=torch.int64), 2) for _ in range(2)]
    pts = [[_plaintext(torch.zeros(l, N, dtype=torch.int64), 2) for _ in range(2)] for _ in range(rot._vecs)]
    pts[-1][0].set_scale(scale)
    _no_call(native, lambda: rot.apply(xs, pts, "key"), "scale mismatch")


def _pages(ctx, scale, chain=1):
    cache = ph.ciphertext_cache(ctx, chain, 2, scale=scale)
    cache._held, cache._free = [1, 1], []
    return cache


@pytest.mark.parametrize("scale", [2.0 ** 38, 2.0 ** 39, 2.0 ** 41, 2.0 ** 50])
def test_pages_and_masks_at_a_scale_that_the_rescale_does_not_remove(native, scale):
    """the products over pages keep the nominal scale, which holds where the other factor's scale is about the removed prime"""
    ctx = _context()
    ct = _ciphertext(torch.zeros(2, 4, N, dtype=torch.int64), 1)
    mask = lambda s: _plaintext(torch.zeros(4, N, dtype=torch.int64), 1, s)
    _no_call(native, lambda: ph.cached_qkt(ctx, None, None, ct, _pages(ctx, scale), [0], 2), "scale mismatch")
    _no_call(native, lambda: ph.cached_score_times_v(ctx, None, None, [ct], _pages(ctx, scale), [0], mask(float(PRIME)), 2, 4, 2), "scale mismatch")
    _no_call(native, lambda: ph.cached_score_times_v(ctx, None, None, [ct], _pages(ctx, 2.0 ** 40), [0], mask(scale), 2, 4, 2), "scale mismatch")


def test_the_prime_that_each_product_over_pages_removes(native):
    """primes of several sizes: the score's, the mask's and the pages' scales go with the primes of their own levels"""
    ctx = _context()
    ctx.primes = np.array([1 << 60, 1 << 50, 1 << 45, 1 << 40, 1 << 30], dtype=np.uint64)
    ct = _ciphertext(torch.zeros(2, 4, N, dtype=torch.int64), 1)
    mask = _plaintext(torch.zeros(4, N, dtype=torch.int64), 1, 2.0 ** 40)
    for chain, scale in ((1, 2.0 ** 45), (3, 2.0 ** 50)):  # pages at the masked scores' level or above, or one below
        for wrong in (2.0 ** 40, 2.0 ** 60):
            _no_call(native, lambda: ph.cached_score_times_v(ctx, None, None, [ct], _pages(ctx, wrong, chain), [0], mask, 2, 4, 2), "scale mismatch")
        with pytest.raises(AttributeError):  # past the checks: no key was given
            ph.cached_score_times_v(ctx, None, None, [ct], _pages(ctx, scale, chain), [0], mask, 2, 4, 2)
        native.calls.clear()
    with pytest.raises(AttributeError):
        ph.cached_qkt(ctx, None, None, ct, _pages(ctx, 2.0 ** 40), [0], 2)


def _encoder(ctx):
    ctx.device = "cpu"  # tensors are made on it
    return types.SimpleNamespace(ctx=ctx, slots=ctx.N // 2, _d_rot=torch.zeros(1), _d_ksi=torch.zeros(1))


@pytest.mark.parametrize("value,at", [(1e9, (0, 0, 0)), (-1e9j, (2, 1, 7)), (math.inf, (0, 1, 3)), (complex(0, -math.inf), (1, 0, 0)), (math.nan, (0, 0, 7)),
                                      (complex(1, math.nan), (2, 0, 2))])
def test_factors_that_no_plaintext_holds(native, monkeypatch, value, at):
    """coefficients past 62 bits, and what is no number, are refused as the encoder refuses them: a coefficient is at most the scale
    times the largest part times sqrt(2)"""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_native, "_current_device", lambda: "cpu")
    ctx = _context()
    rot, factors = _rotary(ctx, "halves"), torch.ones(3, 2, N // 2, dtype=torch.complex128)
    assert [len(v) for v in rot.encode(_encoder(ctx), factors, 2)] == [2, 2, 2]
    native.calls.clear()
    factors[at] = value
    _no_call(native, lambda: rot.encode(_encoder(ctx), factors, 2), "encoded values are too large")


def test_factors_as_large_as_a_plaintext_holds(native, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_native, "_current_device", lambda: "cpu")
    ctx = _context(bits=42)  # two limbs hold 84 bits: the 62 of a coefficient come first
    rot, factors = _rotary(ctx, "pairs"), torch.zeros(1, 1, N // 2, dtype=torch.complex128)
    most = 2.0 ** 61 / (1.4143 * PRIME)
    factors[0, 0, 3] = complex(0.5, -0.999 * most)
    rot.encode(_encoder(ctx), factors, 3)
    factors[0, 0, 3] = complex(0.5, -1.001 * most)
    native.calls.clear()
    _no_call(native, lambda: rot.encode(_encoder(ctx), factors, 3), "encoded values are too large")
    ctx = _context(bits=21)  # two limbs hold 42 bits
    factors[0, 0, 3] = 1.0
    _no_call(native, lambda: _rotary(ctx, "pairs").encode(_encoder(ctx), factors, 3), "encoded values are too large")


@pytest.mark.parametrize("bad", [dict(inv_freq=[1.0, math.nan]), dict(inv_freq=[math.inf, 1.0]), dict(inv_freq=[1.0, -1e300]), dict(scaling=math.nan),
                                 dict(scaling=math.inf)])
def test_angles_that_are_no_numbers(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: None)
    good = dict(inv_freq=[1.0, -0.5], heads=2, d_head=4, packing="pairs")
    ctx = types.SimpleNamespace(N=N, device="cpu")
    rotary_class(ctx, **good)
    rotary_class(ctx, **{**good, "scaling": -2.0, "inv_freq": [1e280, 0.0]})
    with pytest.raises(ValueError, match="finite"):
        rotary_class(ctx, **{**good, **bad})


class _Rotary(rotary_class):
    """on the host: factors of nothing, and what forward would do with them is counted"""

    def factors(self, positions, keep=None, conjugate=False):
        return torch.ones(1, 1, N // 2, dtype=torch.complex128)

    def _encode(self, *args):
        return [["plaintext"]]

    def apply(self, xs, plaintexts, galois_key=None):
        return list(xs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_kept_positions_that_are_no_numbers(monkeypatch, dtype, bad):
    """they would spoil every slot of their ciphertext; in a dropped position's place, or on an axis that no pair follows, they do not count"""
    capturing = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    monkeypatch.setattr(_native, "_current_device", lambda: "cpu")
    rot = _Rotary(types.SimpleNamespace(N=N, device="cpu"), [1.0, 0.5], 2, 4, axes=[0, 2])
    x = types.SimpleNamespace(_chain_index=1)
    p = torch.ones(3, 3, dtype=dtype)
    assert rot.forward(None, [x], p) == [x]
    p[:, 1] = bad
    assert rot.forward(None, [x], p) == [x]
    keep = torch.tensor([True, False, True])
    p[1, 2] = bad
    assert rot.forward(None, [x], p, keep=keep) == [x]
    for k in (None, ~keep):
        with pytest.raises(ValueError, match="finite"):
            rot.forward(None, [x], p, keep=k)
    capturing.append(1)  # the host cannot look
    assert rot.forward(None, [x], p) == [x]
    one = _Rotary(types.SimpleNamespace(N=N, device="cpu"), [0.0, 2.0], 2, 4)
    capturing.clear()
    with pytest.raises(ValueError, match="finite"):
        one.forward(None, [x], p[:, 2])
    assert one.forward(None, [x], p[:1, 2]) == [x] and one.forward(None, [x], p[:, 2].nan_to_num(0, 0, 0).long()) == [x]


def test_angles_past_the_doubles(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_native, "_current_device", lambda: "cpu")
    rot = _Rotary(types.SimpleNamespace(N=N, device="cpu"), [1e-200, -1e250, 1e-3], 2, 4, axes=[0, 0, 1])
    x = types.SimpleNamespace(_chain_index=1)
    assert rot.forward(None, [x], torch.tensor([[1e50, 1e300]], dtype=torch.float64)) == [x]
    with pytest.raises(ValueError, match="finite"):
        rot.forward(None, [x], torch.tensor([[1e60, 0.0]], dtype=torch.float64))
