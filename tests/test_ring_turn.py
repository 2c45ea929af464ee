"""The block-scaled product's epilogue after a wait that ran out, checked on the CPU with the kernel's own turn (tests/ring_turn_host.cpp):
no wait is made to run out on a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_tile_behind_a_wait_that_ran_out_is_taken_for_whole(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++ to build the host harness")
    exe = str(tmp_path / "ring_turn_host")
    build = subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-o", exe, os.path.join(ROOT, "tests", "ring_turn_host.cpp")],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.startswith("ok"), run.stdout[-2000:]
