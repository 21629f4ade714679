"""Where the matrix products read: every 16-byte read of every tile, on the CPU, with the
kernels' own address arithmetic (``slideformer_amd/csrc/tile_range.h``)."""
from __future__ import annotations

import os
import shutil
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_tile_reads_outside_its_matrix(tmp_path):
    gxx = shutil.which("g++")
    assert gxx, "g++ not found"
    exe = str(tmp_path / "tile_range")
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I",
                    os.path.join(REPO, "slideformer_amd", "csrc"), "-o", exe,
                    os.path.join(REPO, "tests", "native", "tile_range_driver.cpp")], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout
    walks, excluded = (int(word) for word in run.stdout.replace(" reads excluded", "").split(" walks, "))
    assert walks > 10000 and excluded > 0, run.stdout
