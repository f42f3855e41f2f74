"""The 8-bit product's planner (laya-cuda_amd/csrc/linear8_plan.hpp), on the CPU by tests/linear8_plan.cpp (no GPU)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_plans_are_valid_and_reach_every_tile(tmp_path):
    exe = tmp_path / "linear8_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'laya-cuda_amd' / 'csrc'}", str(ROOT / "tests" / "linear8_plan.cpp"), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    assert int(run.stdout.split()[1]) > 500000
