"""The cache's bookkeeping without a GPU: which pages are taken, shared, given back and renumbered, with the moves made on host
tensors, and the calls that are refused before anything reaches the device."""
import random
import types

import numpy as np
import pytest
import torch

import pyPhantom as ph
from pyPhantom import cache as cache_module
from pyPhantom._native import LIB, check

N = 16


def _fake_context(size_Q=4):
    ctx = types.SimpleNamespace(N=N, size_Q=size_Q, device=-1, _h=None, primes=np.full(size_Q + 1, 97, dtype=np.uint64))
    ctx.limbs_at = lambda k: size_Q - (k - 1)
    ctx.empty = lambda *shape: torch.full((*shape, N), -7, dtype=torch.int64)
    return ctx


@pytest.fixture
def new(monkeypatch):
    def move(self, dst, src, source=None):
        assert len(set(dst)) == len(dst) == len(src)
        was = (self if source is None else source).data.clone()
        for d, s in zip(dst, src):
            self.data[:, d] = 0 if s < 0 else was[:, s, :, :self._limbs]

    monkeypatch.setattr(ph.ciphertext_cache, "_move", move)
    return lambda pages, planes=2, chain=1, ctx=None: ph.ciphertext_cache(ctx or _fake_context(), chain, pages, planes)


def _marks(cache, table):
    return [int(cache.data[0, p, 0, 0, 0]) for p in table]


def _scaled(cache):
    other = ph.ciphertext_cache(cache.ctx, 1, 2, 2, scale=2.0 ** 39)
    other.allocate(2)
    return other


def _mark(cache, page, value):
    cache.data[:, page] = value


def test_random_life_of_sequences(new):
    """sequences grow, fork, end and are compacted in any order: each reads what was written to it, whoever shared a page with it"""
    rng = random.Random(1)
    for _ in range(20):
        cache = new(rng.randint(8, 40))
        live, stamp = [], 0
        for _ in range(120):
            act = rng.randrange(5)
            if act == 0 and cache.free_pages() >= 3:
                t = cache.allocate(rng.randint(0, 3))
                assert _marks(cache, t) == [0] * len(t)
                live.append((t, [0] * len(t)))
            elif act == 1 and live:
                t, want = live[rng.randrange(len(live))]
                if t and cache.held(t[-1]) == 1:
                    stamp += 1
                    _mark(cache, t[-1], stamp)
                    want[-1] = stamp
            elif act == 2 and live and cache.free_pages() >= 4:
                t, want = rng.choice(live)
                copies = rng.randint(1, 2)
                forks = cache.fork(t, copies=copies, tail=rng.randint(0, 2))
                live += [(f, list(want)) for f in forks]
            elif act == 3 and live:
                t, _ = live.pop(rng.randrange(len(live)))
                cache.free(t)
            elif act == 4 and live:
                new_tables = cache.compact([t for t, _ in live])
                live = [(t, want) for t, (_, want) in zip(new_tables, live)]
                used = cache.pages() - cache.free_pages()
                assert {p for t, _ in live for p in t} == set(range(used))
                assert all(b == a + 1 for a, b in zip(live[0][0], live[0][0][1:]))
            for t, want in live:
                assert _marks(cache, t) == want
            for p in range(cache.pages()):
                assert cache.held(p) == sum(t.count(p) for t, _ in live)
        for t, _ in live:
            cache.free(t)
        assert cache.free_pages() == cache.pages()


def test_page_numbers_of_any_kind(new):
    cache = new(6)
    cache.allocate(6)
    for p in range(6):
        _mark(cache, p, p + 1)
    cache.copy(torch.tensor([0, 1]), np.array([2, 3]))
    cache.copy(range(4, 6), (0, 1))
    assert _marks(cache, range(6)) == [3, 4, 3, 4, 3, 4]
    cache.free(np.array([5]))
    assert cache.free_pages() == 1 and cache.allocate(1) == [5]
    pages = list(torch.tensor([4, 4]))  # two objects, one page
    with pytest.raises(ValueError, match="more often"):
        cache.free(pages)
    assert cache.fork(pages, tail=0) == [[4, 4]] and cache.held(4) == 3
    assert cache.compact([pages, [np.int64(1)]]) == [[0, 0], [1]]
    with pytest.raises(TypeError):
        cache.free([0.0])


@pytest.mark.parametrize("call,match", [
    (lambda c, o: c.copy([0], [0, 1]), "as many"), (lambda c, o: c.copy([4], [0]), "not allocated"), (lambda c, o: c.copy([0], [4]), "not allocated"),
    (lambda c, o: c.copy([9], [0]), "out of range"), (lambda c, o: c.copy([-1], [0]), "out of range"), (lambda c, o: c.copy([0], [-1]), "out of range"),
    (lambda c, o: c.copy([1], [0]), "shared"), (lambda c, o: c.copy([0], [0], source=o), "another context"), (lambda c, o: c.free([4]), "not allocated"),
    (lambda c, o: c.free([0, 0]), "more often"), (lambda c, o: c.free([6]), "out of range"), (lambda c, o: c.fork([4]), "not allocated"),
    (lambda c, o: c.fork([0], copies=0), "at least one"), (lambda c, o: c.fork([0], tail=-2), "at least one"), (lambda c, o: c.allocate(-1), "negative"),
    (lambda c, o: c.compact([[0], [5]]), "not allocated"), (lambda c, o: c.resize(2), "compact first"), (lambda c, o: c.resize(0), "compact first"),
    (lambda c, o: c.page(0, 2), "plane"), (lambda c, o: c.page(0, -1), "plane"), (lambda c, o: c.ciphertexts([0], 7), "plane"), (lambda c, o: c.held(6), "out of range"),
    (lambda c, o: c.multiply_sum([], [0]), "empty"), (lambda c, o: c.multiply_sum([c.page(0)], [0, 2]), "as many"), (lambda c, o: c.multiply_sum([[]], []), "as many"),
    (lambda c, o: c.multiply_sum([c.page(0)], [5]), "not allocated"), (lambda c, o: c.append(1, c.page(0)), "shared"), (lambda c, o: c.store(1, c.page(0)), "shared"),
    (lambda c, o: c.store(0, o.page(0)), "higher level"), (lambda c, o: c.append(0, c.page(2)._like(c.page(2).data, scale=3.0)), "scale"),
    (lambda c, o: c.append(0, c.page(2)._like(c.page(2).data[:1])), "two-polynomial"),
    (lambda c, o: c.append(0, c.page(2)._like(c.page(2).data.double())), "two-polynomial"),
    (lambda c, o: c.append(0, c.page(2)._like(c.page(2).data[:, :2])), "higher level"),  # two limbs that pass for four
    (lambda c, o: c.store(0, c.page(2)._like(c.page(2).data[:, :2])), "higher level"),
    (lambda c, o: c.copy([0], [0], source=_scaled(c)), "scale"),
    (lambda c, o: c.multiply_sum([c.page(0)._like(c.page(0).data[:, :2], chain_index=1)], [0]), "parameter mismatch"),
])
def test_refused_calls_change_nothing(new, call, match):
    cache, other = new(6), new(3, chain=3)
    table = cache.allocate(4)  # 0 .. 3, page 1 held twice
    cache.fork([1], tail=0)
    other.allocate(3)
    for p in table:
        _mark(cache, p, 50 + p)
    before = cache.data.clone()
    with pytest.raises(ValueError, match=match):
        call(cache, other)
    assert torch.equal(cache.data, before) and cache.free_pages() == 2 and [cache.held(p) for p in range(6)] == [1, 2, 1, 1, 0, 0]


def test_running_out_of_pages(new):
    cache = new(5)
    table = cache.allocate(3)
    for call in (lambda: cache.allocate(3), lambda: cache.fork(table, copies=3), lambda: cache.fork(table, copies=1, tail=3)):
        with pytest.raises(RuntimeError, match="out of pages"):
            call()
    assert cache.free_pages() == 2 and cache.allocate(0) == []


def test_a_failed_move_takes_no_pages(new, monkeypatch):
    cache = new(6)
    table = cache.allocate(2)

    def broken(self, dst, src, source=None):
        raise RuntimeError("CUDA error")

    monkeypatch.setattr(ph.ciphertext_cache, "_move", broken)
    for call in (lambda: cache.allocate(2), lambda: cache.fork(table), lambda: cache.compact([[1], [0]])):
        with pytest.raises(RuntimeError, match="CUDA error"):
            call()
        assert cache.free_pages() == 4 and [cache.held(p) for p in range(6)] == [1, 1, 0, 0, 0, 0]


def test_shapes_that_are_refused():
    ctx = _fake_context()
    for pages, planes, chain, match in [(0, 1, 1, "at least one"), (1, 0, 1, "at least one"), (1, 1, 0, "chain index"), (1, 1, 5, "chain index")]:
        with pytest.raises(ValueError, match=match):
            ph.ciphertext_cache(ctx, chain, pages, planes)
    good = dict(inv_freq=[1.0, 0.5], heads=2, d_head=4)
    for bad, match in [(dict(packing="other"), "packing"), (dict(heads=0), "heads"), (dict(heads=3), "heads"), (dict(d_head=-4), "heads"), (dict(inv_freq=[]), "pairs"),
                       (dict(inv_freq=[1.0] * 5), "pairs"), (dict(inv_freq=[1.0] * 3, packing="halves"), "pairs"), (dict(axes=[0, -1]), "axis"), (dict(axes=[0]), "axis")]:
        with pytest.raises(ValueError, match=match):
            ph.rotary(types.SimpleNamespace(N=N, device="cpu"), **{**good, **bad})


def test_entries_refuse_a_missing_context():
    for call in (lambda: LIB.b2_pages_move(None, 1, 1, 0, 1, 0, 1, 1, 0, 0, 0, 0), lambda: LIB.b2_multiply_sum(None, 1, 1, 1, 0, 1, 0, 1, 0, 0),
                 lambda: LIB.b2_multiply_plain_sum(None, 1, 1, 1, 0, 0, 0, 0), lambda: LIB.b2_encode_coeffs_batch(None, 1, 0, 0, 0, 1.0, 0, 0),
                 lambda: LIB.b2_rotary_factors(None, 0, 1, 1, 1, 1, 0, 0, 1, 1, 0, 0, 0, 0, 1.0, 0, 0, 0)):
        with pytest.raises(ValueError, match="null context"):
            check(call())


def test_another_current_device(monkeypatch):
    """calls are made with the context's device current, and the caller's is current again afterwards"""
    seen = []

    class Guard:
        def __init__(self, device):
            seen.append(("to", device))

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *a):
            seen.append("out")

    from pyPhantom import _native
    monkeypatch.setattr(_native, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    with _native.on_device(types.SimpleNamespace(device=0)):
        pass
    assert seen == []
    with _native.on_device(types.SimpleNamespace(device=3)):
        seen.append("call")
    assert seen == [("to", 3), "in", "call", "out"]
    assert cache_module.on_device is _native.on_device
