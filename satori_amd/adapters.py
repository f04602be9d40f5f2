"""Low-rank adapters of many requests beside one projection (satori_hip_adapters_*)."""
from __future__ import annotations

import ctypes

import numpy as np

from . import HipContext, _check, _ffi
from .cache import ElementType, _at, _ints, _pointer


class LowRankAdapters:
    """The adapters that rows of a projection [rows][columns] can have: weights[i] = (down, up, rank, scale), down
    [rank][columns] and up [rows][rank] being device pointers that the caller keeps alive."""

    def __init__(self, context: HipContext, rows: int, columns: int, weights: list[tuple[int, int, int, float]],
                 type: ElementType = ElementType.F16):
        count = len(weights)
        down = (ctypes.c_void_p * count)(*(w[0] for w in weights))
        up = (ctypes.c_void_p * count)(*(w[1] for w in weights))
        ranks, scales = _ints([w[2] for w in weights]), np.array([w[3] for w in weights], np.float32)
        handle = ctypes.c_void_p()
        _check(_ffi.lib().satori_hip_adapters_create(context.handle, rows, columns, int(type), count, down, up,
                                                     _at(ranks), _at(scales), ctypes.byref(handle)))
        self.context, self.rows, self.columns, self.count = context, rows, columns, count
        self._handle = handle

    def apply(self, selection, x: int, base: int, y: int, stream: int = 0) -> None:
        """y[r] = base[r] + scale * up (down x[r]) with the adapter selection[r] of each row (-1: none)."""
        chosen = _ints(selection)
        _check(_ffi.lib().satori_hip_adapters_apply(self._handle, _at(chosen), chosen.size, _pointer(x), _pointer(base),
                                                    _pointer(y), _pointer(stream)))

    def dispose(self) -> None:
        _check(_ffi.lib().satori_hip_adapters_destroy(self._handle))
