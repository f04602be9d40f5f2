"""Low-rank adapters where every adapted row counts: single rows and the smallest shapes, whose one row has an adapter in each
of them; bounds and helpers of test_gpu_adapters.py."""
from __future__ import annotations

import numpy as np
import pytest

from satori_amd.cache import ElementType
from test_gpu_adapters import Case, device  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

F32, F16 = ElementType.F32, ElementType.F16


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("rows,columns,ranks", [
    (256, 1536, [4]), (1, 1, [1]), (1536, 1536, [16]), (1, 8192, [512]), (11008, 96, [64]), (33, 4097, [17, 3]), (5, 2, [1, 16])])
def test_a_single_row(context, device, type_, rows, columns, ranks):  # noqa: F811
    case = Case(context, device, type_, rows, columns, ranks, rows * columns)
    for adapter in range(len(ranks)):
        x, base = case.inputs(1)
        db, dy = device(base), device(np.full_like(base, np.nan))
        case.adapters.apply([adapter], device(x), db, dy)
        got = context.download(np.zeros_like(base), dy)
        case.check([adapter], x, base, got)
        # What is added is no smaller than the check allows to be missing.
        down, up = case.down[adapter].astype(np.float64), case.up[adapter].astype(np.float64)
        added = np.abs(up @ (down @ x[0].astype(np.float64))).max() * float(case.scales[adapter])
        assert added > 1e-3 and not np.array_equal(got, base)
        case.adapters.apply([adapter], device(x), db, db)
        assert np.array_equal(context.download(np.zeros_like(base), db), got)
    case.adapters.dispose()


@pytest.mark.parametrize("rank", [8, 40])  # one launch, two
def test_rows_without_an_adapter_keep_their_bits(context, device, rank):  # noqa: F811
    case = Case(context, device, F16, 70, 300, [rank], rank)
    x, base = case.inputs(5)
    base[1:4, ::3], base[1, 1], base[3, 2] = -0.0, -np.inf, np.float32(1e-45)
    dy = device(np.full_like(base, np.nan))
    case.adapters.apply([0, -1, -1, -1, 0], device(x), device(base), dy)
    got = context.download(np.zeros_like(base), dy)
    assert np.array_equal(got[1:4].view(np.uint32), base[1:4].view(np.uint32))
    case.check([0, 0], x[[0, 4]], base[[0, 4]], got[[0, 4]])
    case.adapters.dispose()
