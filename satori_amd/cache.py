"""Several sequences over one key/value cache: pages that sequences share (satori_hip_pages_*), the plan of a batch over
them and its cache write and attention (satori_hip_cache_*).

The reference keeps one sequence per DenseSession (src/Satori.Core/Model/DenseSession.cs:20); this is the form for hosts
that answer several requests at once. A step of a batch: extend the sequences by their new positions, set the plan, then per
layer append (bias, rotation, cache write) and attend; projections run over the batch's rows as positions.
"""
from __future__ import annotations

import ctypes
import enum
import threading
from array import array
from collections import deque
from collections.abc import Sequence
from dataclasses import dataclass

import numpy as np

from . import ArgumentException, HipContext, _check, _ffi


class ElementType(enum.IntEnum):
    F32 = 0
    F16 = 1


def _ints(values) -> np.ndarray:
    if isinstance(values, np.ndarray) and values.dtype == np.int32 and values.flags.c_contiguous:
        return values.reshape(-1)
    return np.array(_array(values), np.int32)  # (integers of 32 bits or an error: a cast of numpy's would wrap)


def _array(values) -> array:
    """Plain ints for a call: a tenth of the time that numpy takes to make and to locate a short array."""
    return array("i", values.tolist() if isinstance(values, np.ndarray) else values)


def _address(values: array) -> int:
    return values.buffer_info()[0]


def _at(values: np.ndarray) -> ctypes.c_void_p:
    return ctypes.c_void_p(values.ctypes.data)


def _pointer(address: int) -> ctypes.c_void_p:
    return ctypes.c_void_p(address or None)


class _Moves:
    """Page moves of one call: `count` of them, in the caller's arrays of `room` each."""

    def __init__(self, room: int):
        self.room, self.buffer = room, array("i", bytes(8 * room + 4))
        self.sources = _address(self.buffer)
        self.destinations, self.counted = self.sources + 4 * room, self.sources + 8 * room

    @property
    def count(self) -> int:
        return self.buffer[2 * self.room]

    def arrays(self) -> tuple[np.ndarray, np.ndarray]:
        values, n = np.frombuffer(self.buffer, np.int32), self.count
        return values[:n], values[self.room:self.room + n]


class PageTable:
    """Page lists and reference counts of a cache of `page_count` pages (satori_hip_pages): host only. Calls that need
    page bytes to follow return them as moves, (sources, destinations)."""

    # A table's read returns a few dozen page numbers and takes less than a microsecond, half of it making ctypes arguments
    # and results, so its arguments but one are made here and name one buffer, read under a lock (threads may call at once),
    # and the call keeps the interpreter. It waits for no plan that is being made (both only read the tables), but for a call
    # that changes them: some microseconds of another thread's, or a compaction's pass over all lists.

    def __init__(self, page_count: int, page_tokens: int = 32):
        handle = ctypes.c_void_p()
        lib = _ffi.lib()
        _check(lib.satori_hip_pages_create(page_count, page_tokens, ctypes.byref(handle)))
        self._handle = handle
        self.page_count, self.page_tokens = page_count, page_tokens
        # Held by what takes two calls, or a call and the copies that follow it, and by whatever could change pages between.
        self.changes = threading.RLock()
        self._address, self._room = handle.value, min(page_count, 1024)
        buffer = np.zeros(self._room + 1, np.int32)  # and the count
        self._buffer, self._lock = memoryview(buffer), threading.Lock()
        at = buffer.ctypes.data
        self._read = (ctypes.PyDLL(lib._name).satori_hip_pages_sequence, handle, ctypes.c_void_p(), ctypes.c_void_p(at),
                      ctypes.c_int(self._room), ctypes.c_void_p(at + 4 * self._room))

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._handle

    def open(self) -> int:
        sequence = ctypes.c_int()
        _check(_ffi.lib().satori_hip_pages_open(self._handle, ctypes.byref(sequence)))
        return sequence.value

    def _extend(self, sequences, tokens) -> _Moves:
        ids, counts = _array(sequences), _array(tokens)
        n = len(ids)
        if n != len(counts):
            raise ArgumentException("Lengths differ.")
        moves = _Moves(n)
        with self.changes:
            _check(_ffi.lib().satori_hip_pages_extend(self._address, _address(ids), _address(counts), n, moves.sources,
                                                      moves.destinations, n, moves.counted))
        return moves

    def extend(self, sequences, tokens) -> tuple[np.ndarray, np.ndarray]:
        return self._extend(sequences, tokens).arrays()

    def truncate(self, sequence: int, tokens: int) -> None:
        _check(_ffi.lib().satori_hip_pages_truncate(self._address, sequence, tokens))

    def fork(self, sequence: int, count: int = 1) -> list[int]:
        forks = array("i", bytes(4 * max(count, 1)))
        _check(_ffi.lib().satori_hip_pages_fork(self._address, sequence, count, _address(forks)))
        return forks[:count].tolist()

    def _copy(self, sequence: int) -> tuple[int, _Moves]:
        made = ctypes.c_int()
        with self.changes:
            moves = _Moves(self._describe(sequence)[1])
            _check(_ffi.lib().satori_hip_pages_copy(self._address, sequence, ctypes.byref(made), moves.sources,
                                                    moves.destinations, moves.room, moves.counted))
        return made.value, moves

    def copy(self, sequence: int) -> tuple[int, tuple[np.ndarray, np.ndarray]]:
        made, moves = self._copy(sequence)
        return made, moves.arrays()

    def free(self, sequences) -> None:
        ids = _array(sequences)
        _check(_ffi.lib().satori_hip_pages_free(self._address, _address(ids), len(ids)))

    def _compact(self) -> _Moves:
        with self.changes:
            moves = _Moves(self.page_count - self.free_pages)
            _check(_ffi.lib().satori_hip_pages_compact(self._address, moves.sources, moves.destinations, moves.room,
                                                       moves.counted))
        return moves

    def compact(self) -> tuple[np.ndarray, np.ndarray]:
        return self._compact().arrays()

    @property
    def free_pages(self) -> int:
        count = ctypes.c_int()
        _check(_ffi.lib().satori_hip_pages_free_count(self._handle, ctypes.byref(count)))
        return count.value

    def _describe(self, sequence: int) -> tuple[int, int]:
        tokens, count = ctypes.c_int(), ctypes.c_int()
        _check(_ffi.lib().satori_hip_pages_sequence(self._handle, sequence, ctypes.byref(tokens), None, 0,
                                                    ctypes.byref(count)))
        return tokens.value, count.value

    def tokens(self, sequence: int) -> int:
        return self._describe(sequence)[0]

    def pages(self, sequence: int) -> list[int]:
        read, handle, none, at, room, count = self._read
        buffer = self._buffer
        with self._lock:
            if not read(handle, sequence, none, at, room, count):
                return buffer[:buffer[-1]].tolist()
        length = ctypes.c_int()
        with self.changes:  # a long table: a call of its own size
            count = self._describe(sequence)[1]
            table = np.empty(count, np.int32)
            _check(_ffi.lib().satori_hip_pages_sequence(handle, sequence, None, table.ctypes.data, count,
                                                        ctypes.byref(length)))
        return table[:length.value].tolist()  # (another thread may have shortened it)

    def dispose(self) -> None:
        _check(_ffi.lib().satori_hip_pages_destroy(self._handle))


@dataclass(frozen=True)
class CacheLayout:
    """What a page holds: `page_tokens` positions' keys and values of every layer."""
    layers: int
    kv_heads: int
    head_dim: int
    page_tokens: int = 32
    type: ElementType = ElementType.F16

    @property
    def page_bytes(self) -> int:
        count = ctypes.c_int64()
        _check(_ffi.lib().satori_hip_cache_page_bytes(self.layers, self.kv_heads, self.head_dim, self.page_tokens,
                                                      int(self.type), ctypes.byref(count)))
        return count.value


class PagedCache:
    """A pool of pages on the device with its page table: the calls of PageTable (open, tokens and pages are the table's
    own), with the page bytes moved on `stream` (0: the context stream), which is to be the one that the cache's plans run on
    (or ordered with it): a move reads what they have written and comes before what they write next. The same holds for pages
    that free, truncate and compact give up: the next sequence to get them may be written to while a plan on another stream
    still reads them. Where the device takes no copy (an exception), `copy` leaves no sequence behind; after extend and compact
    the table has changed, and the moves stay due: the next call that moves pages, or sets a plan, makes them first.
    `pool` is a device pointer to page_count * layout.page_bytes bytes; 0: allocated here."""

    def __init__(self, context: HipContext, layout: CacheLayout, page_count: int, pool: int = 0):
        self.context, self.layout, self.page_count = context, layout, page_count
        self.page_bytes = layout.page_bytes
        self.table = PageTable(page_count, layout.page_tokens)
        self._owned, self._due = 0, deque()
        if not pool:
            self._owned = pool = context.alloc(page_count * self.page_bytes)
        self.pool = pool
        self.open, self.pages, self.tokens = self.table.open, self.table.pages, self.table.tokens

    def _move(self, moves: _Moves, stream: int) -> None:
        if moves.count:
            self._due.append(moves)
        if self._due:
            self._settle(stream)

    def _settle(self, stream: int) -> None:
        while self._due:  # (what is copied twice, where a call failed behind its first launch, is the same)
            moves = self._due[0]
            self._copy_pages(moves.sources, moves.destinations, moves.count, stream)
            self._due.popleft()

    def copy_pages(self, sources, destinations, stream: int = 0) -> None:
        """Pool page destinations[i] = pool page sources[i] (moves of a page table's own calls, for instance)."""
        s, d = _array(sources), _array(destinations)
        if len(s) != len(d):
            raise ArgumentException("Lengths differ.")
        with self.table.changes:
            self._settle(stream)
            self._copy_pages(_address(s), _address(d), len(s), stream)

    def _copy_pages(self, sources: int, destinations: int, count: int, stream: int) -> None:
        _check(_ffi.lib().satori_hip_cache_copy_pages(self.context.handle, self.pool, self.page_bytes, self.page_count,
                                                      sources, destinations, count, stream or None))

    def extend(self, sequences, tokens, stream: int = 0) -> None:
        """Makes room for tokens[i] more positions of sequences[i]."""
        with self.table.changes:
            self._move(self.table._extend(sequences, tokens), stream)

    def truncate(self, sequence: int, tokens: int) -> None:
        self.table.truncate(sequence, tokens)

    def fork(self, sequence: int, count: int = 1) -> list[int]:
        return self.table.fork(sequence, count)

    def copy(self, sequence: int, stream: int = 0) -> int:
        with self.table.changes:
            self._settle(stream)
            made, moves = self.table._copy(sequence)
            try:
                self._move(moves, stream)
            except Exception:
                self._due.clear()  # (its own: nothing else was due)
                self.table.free([made])
                raise
        return made

    def free(self, sequences) -> None:
        self.table.free(sequences)

    def compact(self, stream: int = 0) -> None:
        with self.table.changes:
            self._move(self.table._compact(), stream)

    @property
    def free_pages(self) -> int:
        return self.table.free_pages

    def plan(self, heads: int) -> "CachePlan":
        """A plan of batches with `heads` query heads over this cache."""
        return CachePlan(self, heads)

    def dispose(self) -> None:
        """Frees the page table and a pool allocated here; plans are disposed of first."""
        self.table.dispose()
        if self._owned:
            self.context.free(self._owned)
            self._owned = 0


class CachePlan:
    """One batch over a PagedCache (satori_hip_cache_plan). Device pointers are ints; `stream` 0 is the context
    stream."""

    def __init__(self, cache: PagedCache, heads: int):
        layout = cache.layout
        handle = ctypes.c_void_p()
        _check(_ffi.lib().satori_hip_cache_plan_create(cache.context.handle, _pointer(cache.pool), cache.page_count,
                                                       layout.layers, heads, layout.kv_heads, layout.head_dim,
                                                       layout.page_tokens, int(layout.type), ctypes.byref(handle)))
        self.cache, self.heads = cache, heads
        self._handle = handle

    def set(self, sequences: Sequence[int], new_tokens: Sequence[int], stream: int = 0) -> None:
        """The batch's rows: the last new_tokens[i] positions of sequences[i]."""
        ids, counts = _ints(sequences), _ints(new_tokens)
        if ids.size != counts.size:
            raise ArgumentException("Lengths differ.")
        if self.cache._due:
            with self.cache.table.changes:
                self.cache._settle(stream)
        _check(_ffi.lib().satori_hip_cache_plan_set(self._handle, self.cache.table.handle, _at(ids), _at(counts),
                                                    ids.size, _pointer(stream)))

    def append(self, layer: int, q: int, q_bias: int, q_out: int, k: int, k_bias: int, v: int, v_bias: int, base: float,
               rotary: int, rope_table: int = 0, rope_positions: int = 0, stream: int = 0) -> None:
        """Bias, rotation and cache write of every row (biases and rope_table may be 0); q_out may be q."""
        _check(_ffi.lib().satori_hip_cache_append(self._handle, layer, _pointer(q), _pointer(q_bias), _pointer(q_out),
                                                  _pointer(k), _pointer(k_bias), _pointer(v), _pointer(v_bias),
                                                  float(base), rotary, _pointer(rope_table), rope_positions,
                                                  _pointer(stream)))

    def attention(self, layer: int, q: int, out: int, stream: int = 0) -> None:
        """Grouped attention of every row over the positions of its sequence up to its own."""
        _check(_ffi.lib().satori_hip_cache_attention(self._handle, layer, _pointer(q), _pointer(out),
                                                     _pointer(stream)))

    def dispose(self) -> None:
        _check(_ffi.lib().satori_hip_cache_plan_destroy(self._handle))
