"""PagedCache without a device: what its calls hand to the page copies, on which stream, in which order among threads, and what
is left when a copy cannot be made."""
from __future__ import annotations

import ctypes
import threading
import time
from types import SimpleNamespace

import numpy as np
import pytest

import satori_amd as S
from satori_amd.cache import CacheLayout, CachePlan, PagedCache


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


def _slow(call):
    """A call that lets other threads in before it begins."""
    def slow(*arguments):
        time.sleep(1e-3)
        return call(*arguments)
    return slow


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


def test_a_copy_that_fails_is_made_up_for(monkeypatch):
    copies = Copies(monkeypatch)
    c = host_only_cache(16)
    s = c.open()
    c.extend([s], [40])
    f = c.fork(s)[0]
    copies.failing = True
    before = c.free_pages
    for _ in range(2):  # (the second finds what is due, and makes nothing of its own)
        with pytest.raises(S.InvalidOperationException):
            c.extend([f], [1])
        assert c.tokens(f) == 41
        with pytest.raises(S.InvalidOperationException):
            c.copy(s)
        assert c.free_pages == before - 1, "a copy that failed leaves nothing"
        c.truncate(f, 40)
    c.free([s])
    with pytest.raises(S.InvalidOperationException):
        c.compact()
    plan = object.__new__(CachePlan)
    plan.cache, plan._handle = c, None
    with pytest.raises(S.InvalidOperationException):
        plan.set([f], [1])
    copies.failing = False
    c.extend([f], [1], 5)
    assert c.pages(f) == [0, 1]
    assert copies.calls == [([1], [2], 5), ([2], [1], 5)], "in their order, before what comes next"
    c.extend([f], [1])
    assert len(copies.calls) == 2


def test_a_failed_copy_leaves_the_sequences_as_they_were(monkeypatch):
    copies = Copies(monkeypatch)
    c = host_only_cache(16)
    s = c.open()
    c.extend([s], [40])
    copies.failing = True
    with pytest.raises(S.InvalidOperationException):
        c.copy(s)
    assert c.free_pages == 14 and c.open() == 1, "no sequence is left behind"
    copies.failing = False
    assert c.copy(s) == 2 and copies.calls == [([0, 1], [2, 3], None)]


def test_threads_that_extend_while_others_copy_read_and_compact(monkeypatch):
    # What takes a size first and then a call, with room for it, meets no error of another thread's making; and page copies are
    # enqueued in the order in which the table changed: played back on a model of the pool, every sequence holds its own tokens.
    monkeypatch.setattr(S._ffi.lib(), "satori_hip_pages_copy", _slow(S._ffi.lib().satori_hip_pages_copy))
    monkeypatch.setattr(S._ffi.lib(), "satori_hip_pages_compact", _slow(S._ffi.lib().satori_hip_pages_compact))
    pool = np.full(4000, -1)

    class Played(Copies):
        def __call__(self, context, address, page_bytes, page_count, sources, destinations, count, stream):
            time.sleep(1e-4)  # (as a launch may take)
            super().__call__(context, address, page_bytes, page_count, sources, destinations, count, stream)
            moved_from, moved_to, _ = self.calls.pop()
            pool[moved_to] = pool[moved_from]
            return 0

    Played(monkeypatch)
    c = host_only_cache(4000)
    long_one = c.open()
    c.extend([long_one], [32 * 1100])  # (longer than the buffer that lists are read into)
    parent = c.open()
    c.extend([parent], [40])
    shared = c.pages(parent)[1]
    pool[shared] = 7
    errors = []

    def guarded(body):
        def run():
            try:
                for _ in range(60):
                    body()
            except Exception as e:  # noqa: BLE001
                errors.append(e)
        return run

    def forks():
        f = c.fork(parent, 3)
        c.extend(f, [1] * 3)
        c.free(f)

    def grow():
        c.extend([long_one], [32])

    def copy():
        c.free([c.copy(long_one)])

    def read():
        assert len(c.pages(long_one)) >= 1100

    threads = [threading.Thread(target=guarded(body)) for body in (forks, grow, copy, read, c.compact, forks)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert pool[c.pages(parent)[1]] == 7
