"""What a cache does to the memory that it gives back, without a GPU: on which stream, and not while a graph is captured. And which
scales it takes."""
import types

import pytest
import torch

import pyPhantom as ph
from pyPhantom import _native, cache as cache_module

N = 16


class _Pool(torch.Tensor):
    """a tensor that remembers the streams that it was handed to"""

    def record_stream(self, stream):
        self.streams = getattr(self, "streams", []) + [stream]


@pytest.fixture
def cache(monkeypatch):
    calls = []
    entry = types.SimpleNamespace(b2_pages_move=lambda *args: calls.append(args) or 0)
    monkeypatch.setattr(cache_module, "LIB", entry)
    monkeypatch.setattr(cache_module, "_stream", lambda: 7)
    monkeypatch.setattr(_native, "_current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "the stream that resize works on")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ctx = types.SimpleNamespace(N=N, size_Q=4, device=-1, _h=None)
    ctx.limbs_at = lambda k: 5 - k
    ctx.empty = lambda *shape: torch.zeros((*shape, N), dtype=torch.int64).as_subclass(_Pool)
    c = ph.ciphertext_cache(ctx, 1, 6, 2)
    c.allocate(3)
    calls.clear()
    c.calls = calls
    return c


def test_resize_holds_the_old_memory_until_it_is_read(cache):
    """the pool may have been made on another stream than the one that copies from it: its memory must not go back before the copy"""
    old = cache.data
    cache.resize(4)
    assert len(cache.calls) == 1 and cache.pages() == 4 and cache.data is not old
    assert old.streams == ["the stream that resize works on"]


def test_resize_is_not_captured(cache, monkeypatch):
    """a graph would read the memory given back here at every replay"""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    old = cache.data
    with pytest.raises(RuntimeError, match="captured"):
        cache.resize(4)
    assert cache.data is old and cache.pages() == 6 and cache.free_pages() == 3 and cache.calls == []


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 0.0, -2.0 ** 40])
def test_scales_that_are_no_scales(cache, scale):
    """NaN compares as unequal to nothing: neither a cache nor what goes into one may have it"""
    with pytest.raises(ValueError, match="scale out of bounds"):
        ph.ciphertext_cache(cache.ctx, 1, 2, scale=scale)
    ct = cache.page(1).clone()
    ct.set_scale(scale)
    other = ph.ciphertext_cache(cache.ctx, 1, 6, 2)
    other.allocate(6)
    other._scale = scale
    cache.calls.clear()
    for call in (lambda: cache.store(0, ct), lambda: cache.append(0, ct), lambda: cache.copy([0], [0], source=other)):
        with pytest.raises(ValueError, match="scale mismatch"):
            call()
    assert cache.calls == [] and not bool(cache.data.any())
