"""Rotary positions of rows (satori_hip_rotation_*): both layouts, part of a head, frequencies scaled for long contexts."""
from __future__ import annotations

import ctypes
import enum

import numpy as np

from . import HipContext, _check, _ffi
from .cache import ElementType, _at


class RotaryLayout(enum.IntEnum):
    HALF = 0         # pairs of lanes (k, k + dimensions / 2)
    INTERLEAVED = 1  # (2 k, 2 k + 1)


class RotaryScaling(enum.IntEnum):
    NONE = 0
    LINEAR = 1
    NTK = 2
    YARN = 3
    WAVELENGTH = 4


def rotary_frequencies(dimensions: int, base: float, scaling: RotaryScaling = RotaryScaling.NONE, factor: float = 1.0,
                       original_positions: int = 0, low: float = 1.0, high: float = 32.0) -> tuple[np.ndarray, float]:
    """The frequencies of dimensions / 2 pairs and the magnitude (satori_hip_rotary_frequencies has the formulas)."""
    frequencies, magnitude = np.zeros(max(dimensions // 2, 1)), ctypes.c_double()
    _check(_ffi.lib().satori_hip_rotary_frequencies(dimensions, float(base), int(scaling), float(factor), original_positions,
                                                    float(low), float(high), _at(frequencies), ctypes.byref(magnitude)))
    return frequencies, magnitude.value


class Rotation:
    """Frequencies on the device, with a table of the first `positions` positions' sines and cosines (others are computed in
    the launch, to the same bits)."""

    def __init__(self, context: HipContext, frequencies, magnitude: float = 1.0,
                 layout: RotaryLayout = RotaryLayout.HALF, positions: int = 0):
        values = np.ascontiguousarray(frequencies, np.float64).reshape(-1)
        handle = ctypes.c_void_p()
        _check(_ffi.lib().satori_hip_rotation_create(context.handle, int(layout), 2 * values.size, _at(values),
                                                     float(magnitude), positions, ctypes.byref(handle)))
        self.context, self.dimensions, self._handle = context, 2 * values.size, handle

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._handle

    def apply(self, x: int, positions: int, rows: int, heads: int, head_dim: int, out: int = 0, stride: int = 0,
              out_stride: int = 0, type: ElementType = ElementType.F32, stream: int = 0) -> None:
        """Turns `rows` rows of `heads` heads at device pointer x by positions[row] (32-bit, on the device), into `out` or in
        place. Strides are elements from row to row; 0: rows lie side by side (in place: x's own)."""
        width = heads * head_dim
        if not out or out == x:
            out, out_stride = x, out_stride or stride
        _check(_ffi.lib().satori_hip_rotation_apply(self._handle, type, x, stride or width, out, out_stride or width, rows, heads,
                                                    head_dim, positions, stream))

    def dispose(self) -> None:
        _check(_ffi.lib().satori_hip_rotation_destroy(self._handle))
