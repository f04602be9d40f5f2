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


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("layout", list(RotaryLayout))
@pytest.mark.parametrize("rows,heads,head_dim,rotary", [(3, 2, 700, 514), (2, 3, 700, 600), (5, 1, 1100, 1026), (2, 5, 1030, 1030),
                                                        (3, 1, 521, 516)])
def test_heads_of_more_pairs_than_a_workgroup(context, device, type_, layout, rows, heads, head_dim, rotary):
    # 256 pairs a workgroup: the parts behind the first begin at other lanes, the last is shorter, and it alone copies what lies behind.
    positions = rng(rotary).integers(0, 5000, rows)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, table=2500, seed=1)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, stride=heads * head_dim + 13, place=1, in_place=True,
          seed=2)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, stride=heads * head_dim + 5,
          out_stride=heads * head_dim + 2, place=3, table=5000, seed=3)


@pytest.mark.parametrize("type_", [F32, F16])
def test_more_rows_than_a_launch_takes(context, device, type_):
    # A launch takes 2^22 rows: the next one begins at its own rows, positions and places.
    rows = (1 << 22) + 37
    g = rng(2)
    x = g.standard_normal((rows, 1, 3)).astype(NUMPY[type_])
    positions = g.integers(0, 5000, rows).astype(np.int32)
    frequencies = np.array([0.013])
    rotation = Rotation(context, frequencies, 1.25, RotaryLayout.HALF, 3000)
    out = device(np.full((rows, 5), 7, NUMPY[type_]))
    rotation.apply(device(x), device(positions), rows, 1, 3, out, out_stride=5, type=type_)
    got = context.download(np.zeros((rows, 5), NUMPY[type_]), out)
    want = rotated(x, positions, frequencies, 1.25, False)
    assert np.all(near(got[:, :3], want[:, 0], type_, 2.0 ** -36))
    assert np.array_equal(got[:, 2], x[:, 0, 2]) and np.all(got[:, 3:] == 7)
    rotation.dispose()
