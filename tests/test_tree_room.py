"""How many rows a batch with a tree may have (plan_batch of satori_amd/csrc/pages.cpp), without a GPU: tests/tree_room.cpp."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ builds the harness")
def test_a_tree_beside_prompts_of_any_length(tmp_path):
    exe = str(tmp_path / "tree_room")
    sources = [os.path.join(ROOT, "tests", "tree_room.cpp"), os.path.join(ROOT, "satori_amd", "csrc", "pages.cpp")]
    build = subprocess.run(["g++", "-std=c++17", "-O1", *sources, "-pthread", "-o", exe], capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-2000:] + run.stderr[-6000:]
    assert run.stdout.rstrip().endswith("ok")
