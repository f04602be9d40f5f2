"""Rotated rows are rounded once, from the sums in 64 bits to the rows' type."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import rng
from satori_amd.rotary import Rotation, RotaryLayout
from test_gpu_cache import F16, device  # noqa: F401  (device: a fixture)
from test_gpu_trees import rotated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("table", [0, 1])
@pytest.mark.parametrize("layout", list(RotaryLayout))
@pytest.mark.parametrize("head_dim", [64, 6])  # whole packs, and pairs one by one
def test_sums_beside_a_border_of_f16(context, device, layout, head_dim, table):
    # At position 0 (sine 0, cosine 1) a lane becomes itself times the magnitude, exactly so in 64 bits for these: a border between
    # two F16 numbers and 2^-40 of it more or less, which FP32 cannot tell from the border. Lanes are signed powers of two
    # and their 3 / 2, down to where F16's steps stay the same (subnormal results, whose borders lie elsewhere).
    lanes = np.array([s * m * 2.0 ** e for e in range(-24, 15) for m in (1.0, 1.5) for s in (1, -1)])
    lanes = lanes[lanes.astype(np.float16).astype(np.float64) == lanes]
    heads = -(-len(lanes) // head_dim)
    x = np.resize(lanes, (1, heads, head_dim)).astype(np.float16)
    for magnitude in (1 + 2.0 ** -11 + 2.0 ** -40, 1 + 2.0 ** -11 - 2.0 ** -40, 1 + 3 * 2.0 ** -11 + 2.0 ** -40,
                      1 + 3 * 2.0 ** -11 - 2.0 ** -40, 1 + 2.0 ** -11, 1 + 2.0 ** -10 + 2.0 ** -40, 1.5 + 2.0 ** -40):
        rotation = Rotation(context, np.ones(head_dim // 2), magnitude, layout, table)
        d = device(x)
        rotation.apply(d, device(np.zeros(1, np.int32)), 1, heads, head_dim, type=F16)
        got = context.download(np.zeros_like(x), d)
        with np.errstate(over="ignore"):  # (from 65520 on: infinite)
            want = (x.astype(np.float64) * magnitude).astype(np.float16)
        assert np.array_equal(got, want)
        rotation.dispose()


def test_many_values_have_the_bits_of_the_sums_in_64_bits(context, device):
    # A million lanes turned by some angles, of which some 60 lie where a second rounding would be seen. What the device's sines
    # and cosines may differ by, 2^-52 of the sums' parts, moves one of a million over a border with a chance of about 2^-18.
    x = (rng(3).standard_normal((2, 4096, 128)) * 50).astype(np.float16)
    magnitude, frequencies = 1.2345678901234567, np.linspace(0.3, 1.2, 64)
    rotation = Rotation(context, frequencies, magnitude)
    d = device(x)
    rotation.apply(d, device(np.array([1, 5], np.int32)), 2, 4096, 128, type=F16)
    got = context.download(np.zeros_like(x), d)
    sums = rotated(x, [1, 5], frequencies, magnitude, False)
    want = sums.astype(np.float16)
    assert np.count_nonzero(sums.astype(np.float32).astype(np.float16) != want) > 20
    assert np.array_equal(got, want)
    rotation.dispose()
