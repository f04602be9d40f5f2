"""The paged cache's host code under AddressSanitizer and UndefinedBehaviorSanitizer (no GPU): tests/pages_sanitize.cpp is
built with g++ together with satori_amd/csrc/pages.cpp and run; it makes random calls and checks every plan's image against
what the kernels assume of it."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the sanitizer harness")
def test_pages_and_plans_under_address_and_undefined_behaviour_sanitizers(tmp_path):
    exe = str(tmp_path / "pages_sanitize")
    sources = [os.path.join(ROOT, "tests", "pages_sanitize.cpp"), os.path.join(ROOT, "satori_amd", "csrc", "pages.cpp")]
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
