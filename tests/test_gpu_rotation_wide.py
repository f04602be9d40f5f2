"""Rotations at sizes that change how a launch works: heads of many pairs, rows past a launch, and rows named as their own output."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.rotary import Rotation, RotaryLayout, rotary_frequencies
from test_gpu_cache import F16, F32, NUMPY, device  # noqa: F401  (device: a fixture)
from test_gpu_rotation import check, near
from test_gpu_trees import rotated

pytestmark = pytest.mark.gpu


def test_rows_that_are_their_own_output(context, device):
    # `out` that is x turns in place, with x's stride where no other is named.
    g = rng(1)
    rows, heads, head_dim, stride = 5, 3, 16, 61
    x = g.standard_normal(rows * stride).astype(np.float32)
    at = device(np.arange(rows, dtype=np.int32))
    rotation = Rotation(context, *rotary_frequencies(head_dim, 1e4))
    named, unnamed = device(x), device(x)
    rotation.apply(named, at, rows, heads, head_dim, out=named, stride=stride)
    rotation.apply(unnamed, at, rows, heads, head_dim, stride=stride)
    got = context.download(np.zeros_like(x), named)
    assert not np.array_equal(got, x)
    assert np.array_equal(got, context.download(np.zeros_like(x), unnamed))
    with pytest.raises(S.ArgumentException):
        rotation.apply(named, at, rows, heads, head_dim, out=named, stride=stride, out_stride=stride + 1)
    rotation.dispose()
