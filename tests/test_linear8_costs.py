"""The 8-bit product's planner against measured times (laya-cuda_amd/csrc/linear8_cost_data.json.gz; no GPU): on products that its
constants were not fitted to, the tile it takes is near the best one."""
import gzip
import json
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "laya-cuda_amd" / "csrc"
sys.path.insert(0, str(CSRC))
import tune_linear8_costs as T  # noqa: E402

DATA = json.loads(gzip.decompress((CSRC / "linear8_cost_data.json.gz").read_bytes()))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
@pytest.mark.parametrize("fast,most,mean", [(False, 1.05, 1.005), (True, 1.2, 1.01)])
def test_held_out_products_take_a_tile_near_the_best(tmp_path, fast, most, mean):
    exe = tmp_path / "linear8_choice"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(Path(__file__).with_name("linear8_choice.cpp")), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    lines = []
    for M, N, K, out, act, res, _ in DATA["held_out"]:
        cols = N // 2 if act > 2 else N
        lines.append(f"{M} {T.padded(cols) if out == T.E4M3 else cols} {-(-K // 128)} {act > 2:d} {out == T.E4M3:d} "
                     f"{out == T.F32 or not fast:d} {T.legal(T.RING, (M, N, K, out, act, res)):d}")
    run = subprocess.run([str(exe)], input="\n".join(lines), capture_output=True, text=True, timeout=60, check=True)
    picks = [int(v) for v in run.stdout.split()]
    assert len(picks) == len(DATA["held_out"]) >= 100
    ratios = []
    for pick, (*case, timed) in zip(picks, DATA["held_out"]):
        assert pick == T.choose(T.present(), tuple(case), fast)  # the script's model is the header's
        us = {t: v for t, v in timed if fast or not (t == T.FAST_RING or t in T.TILES and T.TILES[t][2])}
        ratios.append(us[pick] / min(us.values()))
    assert max(ratios) <= most and sum(ratios) / len(ratios) <= mean
