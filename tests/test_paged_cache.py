"""PagedCache without a device: what its calls hand to the page copies, on which stream, in which order among threads, and what
is left when a copy cannot be made."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import satori_amd as S
from satori_amd.cache import CacheLayout, PagedCache


class Copies:
    """Stands in for satori_hip_cache_copy_pages: keeps what it is called with, and fails while `failing`."""

    def __init__(self, monkeypatch):
        self.calls, self.failing = [], False
        monkeypatch.setattr(S._ffi.lib(), "satori_hip_cache_copy_pages", self)

    def __call__(self, context, pool, page_bytes, page_count, sources, destinations, count, stream):
        if self.failing:
            return 8
        lists = [ctypes.cast(p, ctypes.POINTER(ctypes.c_int))[:count] for p in (sources, destinations)]
        self.calls.append((*lists, stream))
        return 0


def host_only_cache(pages):
    """A PagedCache whose pool nobody reads (its copies go to Copies)."""
    return PagedCache(SimpleNamespace(handle=None), CacheLayout(1, 1, 32), pages, pool=16)


def test_page_moves_take_a_stream(monkeypatch):
    copies = Copies(monkeypatch)
    c = host_only_cache(16)
    s = c.open()
    c.extend([s], [40])
    f = c.fork(s)[0]
    c.extend([f], [1], 77)
    twin = c.copy(s, stream=78)
    c.free([s])
    c.compact(79)
    c.copy_pages([0], [9], 80)
    c.extend([f], [1])
    assert [call[2] for call in copies.calls] == [77, 78, 79, 80]
    other = c.fork(twin)[0]
    c.extend([other], [1])
    assert copies.calls[-1][2] is None  # the context stream
