"""Pages that sequences share (satori_hip_pages_*, host only): random calls against a model in which every sequence has a
list of its own tokens and the pool an entry per position, so that what a sequence reads through its table is what was
written for it whatever is forked, copied, shortened, freed or compacted; and the refusals, after which nothing changed."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import satori_amd as S
from satori_amd.cache import CacheLayout, ElementType, PageTable


class Model:
    """Sequences as token lists, a pool of page contents and the page table under test."""

    def __init__(self, pages, page_tokens):
        self.table = PageTable(pages, page_tokens)
        self.pool = np.full((pages, page_tokens), -1, np.int64)
        self.sequences = {}
        self.next = 0

    def move(self, moves):
        sources, destinations = moves
        assert not set(sources.tolist()) & set(destinations.tolist()), "moves that race"
        assert len(set(destinations.tolist())) == destinations.size
        self.pool[destinations] = self.pool[sources]

    def extend(self, ids, counts):
        self.move(self.table.extend(ids, counts))
        for s, n in zip(ids, counts):
            pages = self.table.pages(s)
            for _ in range(n):
                p = len(self.sequences[s])
                self.pool[pages[p // self.table.page_tokens], p % self.table.page_tokens] = self.next
                self.sequences[s].append(self.next)
                self.next += 1

    def check(self):
        held = np.zeros(self.table.page_count, int)
        for s, tokens in self.sequences.items():
            pages = self.table.pages(s)
            assert self.table.tokens(s) == len(tokens)
            assert len(pages) == -(-len(tokens) // self.table.page_tokens)
            got = self.pool[pages].reshape(-1)[:len(tokens)] if pages else np.zeros(0, int)
            assert got.tolist() == tokens, f"sequence {s}"
            held[pages] += 1
        assert self.table.free_pages == int((held == 0).sum())
        return held


@pytest.mark.parametrize("page_tokens", [32, 64, 256])
def test_random_calls_keep_every_sequence(page_tokens):
    g = np.random.Generator(np.random.PCG64(page_tokens))
    m = Model(40, page_tokens)
    refused = 0
    for step in range(600):
        live = list(m.sequences)
        what = int(g.integers(10))
        before = {s: m.table.pages(s) for s in live}
        try:
            if not live or what == 0:
                s = m.table.open()
                assert s == min(set(range(len(live) + 1)) - set(live)), "the lowest free number"
                m.sequences[s] = []
            elif what <= 4:
                chosen = [s for s in live if g.random() < 0.5]
                m.extend(chosen, [int(g.integers(0, 4 if g.random() < 0.7 else 5 * page_tokens)) for _ in chosen])
            elif what <= 6:
                parent = int(g.choice(live))
                for f in m.table.fork(parent, int(g.integers(0, 3))):
                    m.sequences[f] = list(m.sequences[parent])
                    assert m.table.pages(f) == m.table.pages(parent)
            elif what == 7:
                s = int(g.choice(live))
                n = int(g.integers(0, len(m.sequences[s]) + 1))
                m.table.truncate(s, n)
                del m.sequences[s][n:]
            elif what == 8:
                parent = int(g.choice(live))
                s, moves = m.table.copy(parent)
                m.move(moves)
                m.sequences[s] = list(m.sequences[parent])
                assert not set(m.table.pages(s)) & set(m.table.pages(parent))
            else:
                gone = [int(s) for s in g.choice(live, size=min(len(live), 2), replace=False)]
                m.table.free(gone)
                for s in gone:
                    del m.sequences[s]
                m.move(m.table.compact())
                held = m.check()
                assert np.all(held[:(held > 0).sum()] > 0), "pages in use come first"
        except S.OutOfMemoryException:
            refused += 1
            assert {s: m.table.pages(s) for s in live} == before, "a refused call changes nothing"
        m.check()
    assert refused > 5


def test_the_last_holder_of_a_shared_page_keeps_it():
    t = PageTable(8, 32)
    a = t.open()
    t.extend([a], [40])
    b, c = t.fork(a, 2)
    sources, destinations = t.extend([a, b, c], [1, 1, 1])
    assert sources.tolist() == [1, 1] and destinations.tolist() == [2, 3]
    assert [t.pages(s) for s in (a, b, c)] == [[0, 2], [0, 3], [0, 1]]
    # A fork on a page's border shares no page that is written to.
    t.truncate(a, 32)
    d = t.fork(a)[0]
    sources, _ = t.extend([a, d], [1, 1])
    assert sources.size == 0 and t.pages(a)[0] == t.pages(d)[0] == 0 and t.pages(a)[1] != t.pages(d)[1]


def test_no_tokens_and_no_sequences():
    t = PageTable(2, 32)
    a = t.open()
    assert t.extend([a], [0])[0].size == 0 and t.extend([], [])[0].size == 0
    assert t.pages(a) == [] and t.tokens(a) == 0
    assert t.fork(a, 0) == [] and t.fork(a) == [1]
    copied, (sources, _) = t.copy(a)
    assert copied == 2 and sources.size == 0
    assert t.compact()[0].size == 0
    t.free([])
    t.truncate(a, 0)
    assert t.free_pages == 2


def test_refusals():
    for arguments in ((0, 32), (-1, 32), (4, 16), (4, 0), (4, 48), (4, 512)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            PageTable(*arguments)
    with pytest.raises(S.OverflowException):
        PageTable(2 ** 30, 32)
    t = PageTable(4, 32)
    a = t.open()
    t.extend([a], [70])
    for call in (lambda: t.extend([a, a], [1, 1]), lambda: t.extend([7], [1]), lambda: t.extend([-1], [1]),
                 lambda: t.free([a, a]), lambda: t.free([a, 3]), lambda: t.fork(9), lambda: t.copy(2),
                 lambda: t.truncate(5, 0), lambda: t.pages(1), lambda: t.extend([a], [])):
        with pytest.raises(S.ArgumentException):
            call()
    for call in (lambda: t.extend([a], [-1]), lambda: t.truncate(a, 71), lambda: t.truncate(a, -1),
                 lambda: t.fork(a, -1)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            call()
    for call in (lambda: t.extend([a], [59]), lambda: t.copy(a), lambda: t.extend([a], [2 ** 31 - 71])):
        with pytest.raises(S.OutOfMemoryException):
            call()
    with pytest.raises(S.OverflowException):
        t.extend([a], [2 ** 31 - 70])
    assert t.pages(a) == [0, 1, 2] and t.tokens(a) == 70 and t.free_pages == 1
    # Arrays that could be too short are refused before anything changes.
    lib, n = S._ffi.lib(), ctypes.c_int()
    ids, counts, room = (np.array(v, np.int32) for v in ([a], [1], [0, 0]))
    p = lambda x: ctypes.c_void_p(x.ctypes.data)  # noqa: E731
    assert lib.satori_hip_pages_extend(t.handle, p(ids), p(counts), 1, p(room), p(room), 0, ctypes.byref(n)) == 1
    assert lib.satori_hip_pages_sequence(t.handle, a, None, p(room), 2, None) == 1
    assert lib.satori_hip_pages_extend(t.handle, None, p(counts), 1, p(room), p(room), 1, ctypes.byref(n)) == 10
    assert lib.satori_hip_pages_open(None, ctypes.byref(n)) == 10
    assert t.tokens(a) == 70
    t.dispose()
    t.dispose()
    with pytest.raises(S.ObjectDisposedException):
        t.open()


def test_page_bytes():
    for head_dim, width in ((1, 32), (32, 32), (33, 64), (80, 96), (100, 128), (129, 192), (256, 256)):
        layout = CacheLayout(layers=3, kv_heads=2, head_dim=head_dim, page_tokens=64, type=ElementType.F32)
        assert layout.page_bytes == 3 * 2 * 2 * 64 * width * 4
    assert CacheLayout(28, 2, 128).page_bytes == 28 * 2 * 2 * 32 * 128 * 2
    with pytest.raises(S.NotSupportedException):
        CacheLayout(1, 1, 257).page_bytes
    for layout in (CacheLayout(0, 1, 64), CacheLayout(1, 1, 64, 48), CacheLayout(1, 1, 64, 32, 7)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            layout.page_bytes
    for layout in (CacheLayout(1, 0, 64), CacheLayout(1, 1, 0), CacheLayout(1, -2, 64)):
        with pytest.raises(S.ArgumentException):
            layout.page_bytes
    with pytest.raises(S.OverflowException):
        CacheLayout(1, 2 ** 30, 256).page_bytes


def test_threads_read_lists_at_once():
    # Reads share one buffer: each thread gets its own sequence's list, while another thread forks and frees.
    import threading

    t = PageTable(4000)
    sequences = [t.open() for _ in range(4)]
    t.extend(sequences, [1, 32 * 40, 32 * 700, 32 * 1500])  # (the last is longer than the buffer)
    expected = [t.pages(s) for s in sequences]
    assert [len(e) for e in expected] == [1, 40, 700, 1500]
    wrong, done = [], threading.Event()

    def read(i):
        for _ in range(300):
            if t.pages(sequences[i]) != expected[i]:
                wrong.append(i)

    def churn():
        while not done.is_set():
            forks = t.fork(sequences[1], 3)
            t.extend(forks, [1] * 3)
            t.free(forks)

    threads = [threading.Thread(target=read, args=(i % 4,)) for i in range(8)] + [threading.Thread(target=churn)]
    for thread in threads:
        thread.start()
    for thread in threads[:-1]:
        thread.join()
    done.set()
    threads[-1].join()
    assert not wrong
    t.dispose()
    with pytest.raises(S.ObjectDisposedException):
        t.pages(sequences[0])
