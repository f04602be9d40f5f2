"""Rotations of rows of heads against 64 bits: layouts, types, parts of heads, strides, places, tables, captured calls, and what
is refused."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.rotary import Rotation, RotaryLayout, RotaryScaling, rotary_frequencies
from test_gpu_cache import F16, F32, NUMPY, device  # noqa: F401  (device: a fixture)
from test_gpu_trees import rotated

pytestmark = pytest.mark.gpu


def near(got, want, type_, magnitudes):
    # FP64 until the one rounding (2^-24 or 2^-11 of the value, or half the smallest F16 step), plus what an angle's product and
    # sine leave open: 2^-51 of the angle, under 2^-20 of the lanes for positions below 2^31.
    rel = 2.0 ** -24 if type_ == F32 else 2.0 ** -11
    return np.abs(got.astype(np.float64) - want) <= 1.001 * rel * np.abs(want) + (2.0 ** -25 if type_ == F16 else 0) + magnitudes


def check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, stride=0, out_stride=0, place=0, table=0,
          in_place=False, seed=0):
    g = rng(seed + head_dim + rows)
    width = heads * head_dim
    stride, out_stride = stride or width, out_stride or width
    frequencies, magnitude = rotary_frequencies(rotary, 1e4, RotaryScaling.LINEAR, 2.0)
    magnitude = 1.25
    memory = g.standard_normal(place + (rows - 1) * stride + width + 9).astype(NUMPY[type_])
    x = np.lib.stride_tricks.as_strided(memory[place:], (rows, width), (stride * memory.itemsize, memory.itemsize))
    source = x.copy()
    at = np.array(positions, np.int32)
    rotation = Rotation(context, frequencies, magnitude, layout, table)
    dx = device(memory)
    address = dx + place * memory.itemsize
    if in_place:
        rotation.apply(address, device(at), rows, heads, head_dim, stride=stride, type=type_)
        got = context.download(memory.copy(), dx)
    else:
        target = np.full(place + (rows - 1) * out_stride + width + 9, 7, NUMPY[type_])
        out = device(target)
        rotation.apply(address, device(at), rows, heads, head_dim, out + place * memory.itemsize, stride, out_stride, type_)
        got = context.download(target.copy(), out)
        memory, stride = target, out_stride
    result = np.lib.stride_tricks.as_strided(got[place:], (rows, width), (stride * got.itemsize, got.itemsize)).copy()
    want = rotated(source.reshape(rows, heads, head_dim), positions, frequencies, magnitude, layout == RotaryLayout.INTERLEAVED)
    slack = 16 * (2.0 ** -50 * np.abs(at.astype(np.float64)) + 2.0 ** -49)[:, None, None]
    assert np.all(near(result.reshape(want.shape), want, type_, slack))
    # The lanes behind the rotated ones are copied; what lies between rows stays.
    assert np.array_equal(result.reshape(want.shape)[..., rotary:], source.reshape(want.shape)[..., rotary:])
    view = np.lib.stride_tricks.as_strided(got[place:], (rows, width), (stride * got.itemsize, got.itemsize))
    back = np.lib.stride_tricks.as_strided(memory[place:], (rows, width), (stride * got.itemsize, got.itemsize))
    view[:] = back
    assert np.array_equal(got, memory)
    context.synchronize()
    rotation.dispose()
    return result


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("layout", list(RotaryLayout))
@pytest.mark.parametrize("rows,heads,head_dim,rotary", [
    (1, 1, 2, 2), (1, 12, 128, 128), (7, 5, 80, 80), (3, 2, 33, 32), (300, 9, 64, 26), (5, 4, 128, 42), (2, 3, 256, 256), (65, 1, 7, 6),
    (4, 6, 576, 64)])
def test_rows_of_heads(context, device, type_, layout, rows, heads, head_dim, rotary):
    g = rng(rows * heads)
    positions = g.integers(0, 5000, rows)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, table=2500, seed=1)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, stride=heads * head_dim + 13, place=1, in_place=True,
          seed=2)
    check(context, device, type_, layout, rows, heads, head_dim, rotary, positions, stride=heads * head_dim + 5,
          out_stride=heads * head_dim + 2, place=3, table=5000, seed=3)


@pytest.mark.parametrize("layout", list(RotaryLayout))
def test_positions_far_and_before_the_first(context, device, layout):
    positions = [0, 1, -1, -100000, 2 ** 31 - 1, -2 ** 31, 10 ** 6, 131071]
    check(context, device, F32, layout, len(positions), 3, 64, 64, positions, table=1000)


@pytest.mark.parametrize("layout", list(RotaryLayout))
@pytest.mark.parametrize("type_", [F32, F16])
def test_a_table_gives_the_same_bits(context, device, layout, type_):
    g = rng(6)
    x = g.standard_normal((200, 4, 96)).astype(NUMPY[type_])
    positions = device(g.integers(0, 40000, 200).astype(np.int32))
    frequencies = rotary_frequencies(96, 1e6, RotaryScaling.YARN, 4.0, 32768)
    results = []
    for table in (0, 1, 20000, 40000):
        rotation = Rotation(context, *frequencies, layout, table)
        out = device(np.zeros_like(x))
        rotation.apply(device(x), positions, 200, 4, 96, out, type=type_)
        results.append(context.download(np.zeros_like(x), out))
        rotation.dispose()
    for r in results[1:]:
        assert np.array_equal(results[0], r)


def test_rows_behind_the_fourth_gibibyte(context, device):
    rows, heads, head_dim, stride = 4, 2, 64, 1_500_000_001
    rotation = Rotation(context, *rotary_frequencies(64, 1e4), RotaryLayout.INTERLEAVED)
    g = rng(9)
    x = g.standard_normal((rows, heads * head_dim)).astype(np.float16)
    p = context.alloc(((rows - 1) * stride + heads * head_dim) * 2)
    for r in range(rows):
        context.upload(p + r * stride * 2, x[r])
    positions = [3, 1000, 77, 5]
    rotation.apply(p, device(np.array(positions, np.int32)), rows, heads, head_dim, stride=stride, type=F16)
    got = np.stack([context.download(np.zeros(heads * head_dim, np.float16), p + r * stride * 2) for r in range(rows)])
    context.free(p)
    want = rotated(x.reshape(rows, heads, head_dim), positions, rotary_frequencies(64, 1e4)[0], 1.0, True)
    assert np.all(near(got.reshape(want.shape), want, F16, 2.0 ** -30))
    rotation.dispose()


def test_values_that_are_no_numbers(context, device):
    # An infinite lane makes its pair infinite or NaN and nothing else.
    x = np.ones((2, 2, 8), np.float32)
    x[0, 1, 1], x[1, 0, 6] = np.inf, np.nan
    rotation = Rotation(context, *rotary_frequencies(8, 1e4))
    d = device(x)
    rotation.apply(d, device(np.array([5, 0], np.int32)), 2, 2, 8)
    got = context.download(np.zeros_like(x), d)
    spoiled = np.zeros(x.shape, bool)
    spoiled[0, 1, [1, 5]] = spoiled[1, 0, [2, 6]] = True
    assert np.array_equal(~np.isfinite(got), spoiled)
    rotation.dispose()


def test_captured_calls_read_positions_when_they_run(context, device):
    g = rng(10)
    x = g.standard_normal((6, 3, 32)).astype(np.float32)
    dx, out, positions = device(x), device(np.zeros_like(x)), device(np.zeros(6, np.int32))
    rotation = Rotation(context, *rotary_frequencies(32, 1e4), positions=50)
    context.capture_begin()
    rotation.apply(dx, positions, 6, 3, 32, out)
    step = context.capture_end()
    with pytest.raises(S.ArgumentException):
        rotation.dispose()
    for seed in range(4):
        at = rng(seed).integers(0, 100, 6).astype(np.int32)
        context.upload(positions, at)
        step.execute()
        got = context.download(np.zeros_like(x), out)
        rotation.apply(dx, positions, 6, 3, 32, out)
        assert np.array_equal(got, context.download(np.zeros_like(x), out))
        assert np.all(near(got, rotated(x, at, rotary_frequencies(32, 1e4)[0], 1.0, False), F32, 2.0 ** -40))
    step.dispose()
    rotation.dispose()


def test_refused_calls(context, device):
    for bad in (dict(frequencies=[]), dict(frequencies=[np.inf]), dict(frequencies=[np.nan]), dict(frequencies=[1.0], magnitude=np.inf),
                dict(frequencies=[1.0], layout=2), dict(frequencies=[1.0], positions=-1), dict(frequencies=np.ones(32769))):
        with pytest.raises(S.ArgumentOutOfRangeException):
            Rotation(context, **bad)
    with pytest.raises(S.OutOfMemoryException):
        Rotation(context, np.ones(32768), positions=2 ** 31 - 1)
    rotation = Rotation(context, [1.0, 0.5])
    x, at = device(np.zeros(64, np.float32)), device(np.zeros(4, np.int32))
    call = lambda **k: rotation.apply(**{**dict(x=x, positions=at, rows=2, heads=2, head_dim=4), **k})  # noqa: E731
    call(rows=0)
    for bad in (dict(rows=-1), dict(heads=0), dict(head_dim=3), dict(head_dim=0), dict(stride=7), dict(out=x + 128, out_stride=7),
                dict(heads=2 ** 30), dict(type=2), dict(stride=2 ** 62)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            call(**bad)
    for bad in (dict(out=x + 4), dict(out=x, out_stride=9), dict(x=x + 2), dict(positions=at + 2), dict(out=x + 128 + 1),
                dict(positions=x + 4)):
        with pytest.raises(S.ArgumentException):
            call(**bad)
    for bad in (dict(x=0), dict(positions=0)):
        with pytest.raises(S.ArgumentNullException):
            call(**bad)
    context.synchronize()
    rotation.dispose()
    rotation.dispose()
    with pytest.raises(S.ObjectDisposedException):
        call()
    context.capture_begin()
    with pytest.raises(S.InvalidOperationException):
        Rotation(context, [1.0])
    context.capture_end().dispose()
    handle = ctypes.c_void_p()
    assert S._ffi.lib().satori_hip_rotation_create(context.handle, 0, 2, None, 1.0, 0, ctypes.byref(handle)) == 10


def test_two_rotations_on_two_streams(context, device):
    other = S.HipContext(0)
    g = rng(11)
    x = g.standard_normal((1000, 8, 128)).astype(np.float32)
    at = device(np.arange(1000, dtype=np.int32))
    stream = ctypes.c_void_p()
    assert S._ffi.lib().satori_hip_context_stream(other.handle, ctypes.byref(stream)) == 0
    rotations = [Rotation(context, *rotary_frequencies(128, base)) for base in (1e4, 1e6)]
    outs = [device(np.zeros_like(x)) for _ in rotations]
    dx = device(x)
    for r, o, s in zip(rotations, outs, (0, stream.value)):
        r.apply(dx, at, 1000, 8, 128, o, stream=s)
    other.synchronize()
    for base, o in zip((1e4, 1e6), outs):
        got = context.download(np.zeros_like(x), o)
        assert np.all(near(got, rotated(x, np.arange(1000), rotary_frequencies(128, base)[0], 1.0, False), F32, 2.0 ** -36))
    for r in rotations:
        r.dispose()
    other.dispose()
