"""Rows of the output that the blocks of the few-token layer's second kernel own, checked on the CPU with the kernel's own function
(tests/row_slice_host.cpp): hidden sizes below the number of blocks leave some without any."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_and_pieces(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++ to build the host harness")
    exe = str(tmp_path / "row_slice_host")
    build = subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-o", exe, os.path.join(ROOT, "tests", "row_slice_host.cpp")],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.startswith("ok"), (run.returncode, run.stdout[-2000:])
