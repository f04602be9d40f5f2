"""Low-rank adapters of many requests beside one projection, against y = base + scale up (down x) in 64 bits.

The bound: both products are FP32 sums, of `columns` and of `rank` terms in any order, the scale one more rounding, so with
e = 2^-24 a row's lane is off by at most ((columns + rank + 8) e |scale| sum |up| sum |down x| + e (|base| + |y|))."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.adapters import LowRankAdapters
from satori_amd.cache import ElementType
from test_gpu_cache import NUMPY, Device

pytestmark = pytest.mark.gpu

F32, F16 = ElementType.F32, ElementType.F16
E = 2.0 ** -24


@pytest.fixture
def device(context):
    d = Device(context)
    yield d
    d.close()


class Case:
    def __init__(self, context, device, type_, rows, columns, ranks, seed, offset=0):
        g = rng(seed)
        self.g, self.rows, self.columns = g, rows, columns
        n = NUMPY[type_]
        self.down = [(g.standard_normal((r, columns)) / np.sqrt(columns)).astype(n) for r in ranks]
        self.up = [(g.standard_normal((rows, r)) / np.sqrt(r)).astype(n) for r in ranks]
        self.scales = [np.float32(0.5 + i) for i in range(len(ranks))]
        held = []
        for a in self.down + self.up:  # weights that begin inside an allocation
            p = device(np.concatenate([np.zeros(offset, n), a.reshape(-1)]))
            held.append(p + offset * a.itemsize)
        weights = list(zip(held[:len(ranks)], held[len(ranks):], ranks, self.scales))
        self.adapters = LowRankAdapters(context, rows, columns, weights, type_)

    def check(self, selection, x, base, got):
        for r, a in enumerate(selection):
            if a < 0:
                assert np.array_equal(got[r], base[r]), f"row {r} has no adapter"
                continue
            down, up = self.down[a].astype(np.float64), self.up[a].astype(np.float64)
            scale, x64, b64 = float(self.scales[a]), x[r].astype(np.float64), base[r].astype(np.float64)
            y = b64 + scale * (up @ (down @ x64))
            most = scale * (np.abs(up) @ (np.abs(down) @ np.abs(x64)))
            bound = (self.columns + down.shape[0] + 8) * E * most + E * (np.abs(b64) + np.abs(y))
            err = np.abs(got[r] - y)
            assert np.all(err <= bound), f"row {r} adapter {a}: {err.max()} over {bound.flat[err.argmax()]}"

    def inputs(self, positions):
        return (self.g.standard_normal((positions, self.columns)).astype(np.float32),
                self.g.standard_normal((positions, self.rows)).astype(np.float32))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("rows,columns,ranks,positions", [
    (1536, 1536, [16, 16, 8, 64], 12), (256, 1536, [4], 1), (1, 1, [1], 1), (1, 1, [3, 512], 5), (1001, 1477, [11, 1, 33], 40),
    (64, 8192, [128], 17), (8960, 1536, [16] * 30, 64), (300, 260, [7, 20], 256), (300, 264, [12, 20], 300),
    (40, 100, [2, 5, 6], 777)])
def test_adapters(context, device, type_, rows, columns, ranks, positions):
    case = Case(context, device, type_, rows, columns, ranks, rows + positions)
    selection = case.g.integers(-1, len(ranks), positions)
    x, base = case.inputs(positions)
    dx, db, dy = device(x), device(base), device(np.full_like(base, np.nan))
    case.adapters.apply(selection, dx, db, dy)
    got = context.download(np.zeros_like(base), dy)
    case.check(selection, x, base, got)
    assert np.array_equal(context.download(np.zeros_like(base), db), base)
    case.adapters.apply(selection, dx, db, db)  # in place: the same values
    assert np.array_equal(context.download(np.zeros_like(base), db), got)
    case.adapters.dispose()


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("offset", [1, 4])
def test_weights_and_inputs_inside_allocations(context, device, type_, offset):
    case = Case(context, device, type_, 96, 512, [8, 16], offset, offset=offset)
    x, base = case.inputs(9)
    dx = device(np.concatenate([np.zeros(1, np.float32), x.reshape(-1)])) + 4
    dy = device(np.zeros_like(base))
    selection = [0, 1, 0, 1, 1, -1, 0, 0, 1]
    case.adapters.apply(selection, dx, device(base), dy)
    case.check(selection, x, base, context.download(np.zeros_like(base), dy))
    case.adapters.dispose()


def test_rows_keep_to_themselves(context, device):
    # A row's infinities and NaN reach no other row, and padding of a rank spoils nothing.
    case = Case(context, device, F16, 200, 320, [5, 16], 3)
    x, base = case.inputs(20)
    x[3, 7], x[4, 0], base[5, 1] = np.inf, np.nan, np.nan
    selection = np.array([0, 1] * 10)
    dy = device(np.zeros_like(base))
    case.adapters.apply(selection, device(x), device(base), dy)
    got = context.download(np.zeros_like(base), dy)
    clean = [r for r in range(20) if r not in (3, 4, 5)]
    case.check(selection[clean], x[clean], base[clean], got[clean])
    assert not np.isfinite(got[3]).any() and np.isnan(got[4]).all()
    assert np.isnan(got[5, 1]) and np.isfinite(np.delete(got[5], 1)).all()
    case.adapters.dispose()


def test_a_captured_application_keeps_its_selection(context, device):
    case = Case(context, device, F16, 512, 768, [16, 16, 8], 4)
    x, base = case.inputs(6)
    dx, db, dy, other = device(x), device(base), device(np.zeros_like(base)), device(np.zeros_like(base))
    selection = np.array([0, 1, 2, -1, 1, 0], np.int32)
    context.capture_begin()
    case.adapters.apply(selection, dx, db, dy)
    step = context.capture_end()
    chosen = selection.copy()
    selection[:] = 2  # the caller's array is its own again
    with pytest.raises(S.ArgumentException):
        case.adapters.dispose()
    for _ in range(3):
        x, base = case.inputs(6)
        context.upload(dx, x)
        context.upload(db, base)
        step.execute()
        case.adapters.apply([1] * 6, dx, db, other)
        case.check(chosen, x, base, context.download(np.zeros_like(base), dy))
        case.check([1] * 6, x, base, context.download(np.zeros_like(base), other))
    step.dispose()
    case.adapters.dispose()


def test_refusals(context, device):
    w, x = device(np.zeros(4096, np.float32)), device(np.zeros(4096, np.float32))
    y = device(np.zeros(4096, np.float32))
    for rows, columns, weights in ((0, 8, [(w, w, 4, 1.0)]), (8, -1, [(w, w, 4, 1.0)]), (8, 8, []),
                                   (8, 8, [(w, w, 0, 1.0)]), (8, 8, [(w, w, 513, 1.0)])):
        with pytest.raises(S.ArgumentOutOfRangeException):
            LowRankAdapters(context, rows, columns, weights, F32)
    with pytest.raises(S.ArgumentOutOfRangeException):
        LowRankAdapters(context, 8, 8, [(w, w, 4, 1.0)], 2)
    with pytest.raises(S.ArgumentNullException):
        LowRankAdapters(context, 8, 8, [(0, w, 4, 1.0)], F32)
    with pytest.raises(S.ArgumentException):
        LowRankAdapters(context, 8, 8, [(w + 2, w, 4, 1.0)], F32)
    a = LowRankAdapters(context, 8, 8, [(w, w, 4, 1.0)], F32)
    for selection in ([1], [-2], [0, 5]):
        with pytest.raises(S.ArgumentOutOfRangeException):
            a.apply(selection, x, y, y)
    with pytest.raises(S.ArgumentOutOfRangeException):
        a.apply([], x, y, y)
    with pytest.raises(S.ArgumentNullException):
        a.apply([0], 0, y, y)
    for arguments in ((x, y, x), (x, y, y + 4), (y + 4, x, y)):
        with pytest.raises(S.ArgumentException):
            a.apply([0, 0], *arguments)
    a.dispose()
    a.dispose()
    with pytest.raises(S.ObjectDisposedException):
        a.apply([0], x, y, y)
    own = S.HipContext(0)
    p = own.alloc(256)
    held = LowRankAdapters(own, 8, 8, [(p, p, 4, 1.0)], F32)
    with pytest.raises(S.ArgumentException):
        own.dispose()
    held.dispose()
    own.free(p)
    own.dispose()
