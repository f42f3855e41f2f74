"""The tile walk of the persistent kernels (laya-cuda_amd/csrc/ring_walk.hpp, shared with the kernel), on the CPU by
tests/ring_walk.cpp (no GPU)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_every_tile_is_taken_once(tmp_path):
    exe = tmp_path / "ring_walk"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'laya-cuda_amd' / 'csrc'}", str(ROOT / "tests" / "ring_walk.cpp"), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    assert int(run.stdout.split()[1]) > 1000000
