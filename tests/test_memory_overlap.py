"""Whether tensors' heads share memory (``slideformer_amd/csrc/memory_overlap.h``), against counting every byte, on the
CPU."""
from __future__ import annotations

import os
import shutil
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_shared_bytes_are_found_and_no_others(tmp_path):
    gxx = shutil.which("g++")
    assert gxx, "g++ not found"
    exe = str(tmp_path / "memory_overlap")
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(REPO, "slideformer_amd", "csrc"), "-o", exe,
                    os.path.join(REPO, "tests", "native", "memory_overlap_driver.cpp")], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    cases, sharing = (int(run.stdout.split()[k]) for k in (0, 2))
    assert cases == 200000 and cases // 10 < sharing < cases * 9 // 10, run.stdout
