"""Trees of drafted tokens and rotary frequencies, what of them is the host's: plans of trees under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/trees_sanitize.cpp), the frequencies against their formulas, and refusals."""
from __future__ import annotations

import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import satori_amd as S
from satori_amd.rotary import RotaryScaling, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the sanitizer harness")
def test_plans_of_trees_under_address_and_undefined_behaviour_sanitizers(tmp_path):
    exe = str(tmp_path / "trees_sanitize")
    sources = [os.path.join(ROOT, "tests", "trees_sanitize.cpp"), os.path.join(ROOT, "satori_amd", "csrc", "pages.cpp")]
    build = subprocess.run(
        ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
         "-fno-sanitize-recover=all", "-static-libasan", "-static-libubsan", *sources, "-o", exe],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-4000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    run = subprocess.run([exe], capture_output=True, text=True, timeout=900, env=env)
    assert run.returncode == 0, run.stdout[-2000:] + run.stderr[-6000:]
    assert run.stdout.rstrip().endswith("ok"), run.stdout[-2000:]
    assert "runtime error" not in run.stderr and "AddressSanitizer" not in run.stderr, run.stderr[-6000:]


# ---- frequencies ----

def expected(r, base, scaling, s, original, low, high):
    plain = [base ** (-2 * k / r) for k in range(r // 2)]
    if scaling == RotaryScaling.LINEAR:
        return [f / s for f in plain], 1.0
    if scaling == RotaryScaling.NTK:
        return [(base * s ** (r / (r - 2))) ** (-2 * k / r) for k in range(r // 2)], 1.0
    if scaling == RotaryScaling.YARN:
        def pair(turns):
            return r * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
        first, last = max(0, math.floor(pair(high))), min(r - 1, math.ceil(pair(low)))
        part = [min(1, max(0, (k - first) / max(0.001, last - first))) for k in range(r // 2)]
        return [f * (1 - p) + f / s * p for f, p in zip(plain, part)], 1 + 0.1 * math.log(s)
    if scaling == RotaryScaling.WAVELENGTH:
        part = [min(1, max(0, (original * f / (2 * math.pi) - low) / (high - low))) for f in plain]
        return [f * p + f / s * (1 - p) for f, p in zip(plain, part)], 1.0
    return plain, 1.0


@pytest.mark.parametrize("scaling", list(RotaryScaling))
@pytest.mark.parametrize("r,base,s,original,low,high", [
    (128, 1e6, 4.0, 32768, 1.0, 32.0), (64, 10000.0, 8.0, 8192, 1.0, 4.0), (4, 10000.0, 1.0, 1, 1.0, 32.0),
    (80, 500000.0, 1.37, 2048, 0.5, 7.0), (256, 1.5, 16.0, 100000, 1.0, 32.0)])
def test_frequencies_follow_their_formulas(scaling, r, base, s, original, low, high):
    got, magnitude = rotary_frequencies(r, base, scaling, s, original, low, high)
    want, factor = expected(r, base, scaling, s, original, low, high)
    # Each takes a power and a handful of products and sums of numbers of one sign, some 2^-52 each; a power's own error, and that
    # of the base and the exponent it is taken of, is at most 1 + ln(f) of those.
    worst = 16 * (1 + abs(np.log(want))) * 2.0 ** -52
    assert got.shape == (r // 2,) and np.all(np.abs(got / want - 1) <= worst)
    assert abs(magnitude / factor - 1) <= 1e-15


def test_scaled_frequencies_keep_what_they_promise():
    plain, _ = rotary_frequencies(128, 1e6)
    for scaling in (RotaryScaling.YARN, RotaryScaling.WAVELENGTH):
        scaled, _ = rotary_frequencies(128, 1e6, scaling, 4.0, 32768, 1.0, 32.0)
        turns = 32768 * plain / (2 * np.pi)
        assert np.array_equal(scaled[turns > 64], plain[turns > 64])
        assert np.allclose(scaled[turns < 0.5], plain[turns < 0.5] / 4, rtol=1e-15)
    scaled, _ = rotary_frequencies(128, 1e6, RotaryScaling.NTK, 4.0)
    assert scaled[0] == 1 and abs(scaled[-1] / (plain[-1] / 4) - 1) < 1e-13


@pytest.mark.parametrize("arguments", [
    (0, 1e4), (-2, 1e4), (7, 1e4), (8, 0.0), (8, -1.0), (8, math.inf), (8, math.nan), (8, 1e4, 5), (8, 1e4, -1),
    (8, 1e4, 1, 0.5), (8, 1e4, 1, math.nan), (8, 1e4, 1, math.inf), (2, 1e4, 2, 2.0), (8, 1e4, 3, 2.0, 0), (8, 1.0, 3, 2.0, 100),
    (8, 1e4, 3, 2.0, 100, 0.0, 4.0), (8, 1e4, 4, 2.0, 100, 4.0, 4.0), (8, 1e4, 4, 2.0, 100, 1.0, math.inf),
    (8, 1e4, 4, 2.0, -5)])
def test_frequencies_that_make_no_sense_are_refused(arguments):
    with pytest.raises(S.ArgumentOutOfRangeException):
        rotary_frequencies(*arguments)


def test_null_arguments_are_refused():
    lib, one = S._ffi.lib(), ctypes.c_double()
    for frequencies, magnitude in ((None, ctypes.byref(one)), (ctypes.byref(one), None)):
        assert lib.satori_hip_rotary_frequencies(2, 1e4, 0, 1.0, 0, 1.0, 32.0, frequencies, magnitude) == 10
    handle = ctypes.c_void_p()
    # (without a context, before anything is asked of a device)
    assert lib.satori_hip_rotation_create(None, 0, 2, ctypes.byref(one), 1.0, 0, ctypes.byref(handle)) == 10
    assert lib.satori_hip_rotation_create(None, 0, 2, ctypes.byref(one), 1.0, 0, None) == 10
    assert lib.satori_hip_logit_rules_create(None, 10, 0, 0, ctypes.byref(handle)) == 10
    assert lib.satori_hip_logit_rules_create(None, 10, 0, 0, None) == 10
    for name in ("rotation_destroy", "logit_rules_destroy"):
        assert getattr(lib, "satori_hip_" + name)(None) == 0
    assert lib.satori_hip_rotation_apply(None, 0, None, 0, None, 0, 1, 1, 1, None, None) == 10
    assert lib.satori_hip_logit_rules_apply(None, None, None) == 10
    assert lib.satori_hip_logit_rules_set_biases(None, 0, None, None, 0, None) == 10
    assert lib.satori_hip_cache_plan_set_tree(None, None, None, None, None, 0, None) == 10
    assert lib.satori_hip_cache_append_rotated(None, 0, *[None] * 9) == 10
    assert lib.satori_hip_cache_keep(None, None, None, 0, None) == 10
