"""What a batch's plan asks for (plan_batch of satori_amd/csrc/pages.cpp), without a GPU: tests/plan_memory.cpp is built with
g++ under AddressSanitizer and UndefinedBehaviorSanitizer together with pages.cpp; a check a test."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the harness")


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "plan_memory")
    sources = [os.path.join(ROOT, "tests", "plan_memory.cpp"), os.path.join(ROOT, "satori_amd", "csrc", "pages.cpp")]
    build = subprocess.run(
        ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
         "-fno-sanitize-recover=all", "-static-libasan", "-static-libubsan", "-pthread", *sources, "-o", exe],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-4000:]
    return exe


def run(exe, what):
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    done = subprocess.run([exe, what], capture_output=True, text=True, timeout=600, env=env)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-6000:]
    assert done.stdout.rstrip().endswith("ok"), done.stdout[-2000:]


def test_rows_of_one_part_ask_for_no_partial_results(harness):
    run(harness, "partials")


def test_a_plan_has_room_for_every_smaller_batch(harness):
    run(harness, "smaller")


def test_lists_are_read_beside_a_plan(harness):
    run(harness, "readers")


def test_a_sequence_as_long_as_positions_are_counted(harness):
    run(harness, "longest")
