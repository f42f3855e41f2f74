"""The 8-bit product's cost constants (linear8_plan.hpp): sweep, fit and check.

    python laya-cuda_amd/csrc/tune_linear8_costs.py sweep --seed 31 --count 260 --out <file>   (on the GPU)
    python laya-cuda_amd/csrc/tune_linear8_costs.py fit                                        (anywhere)

`sweep` times products of random sizes, types, activations and residuals on every tile that makes the output and is not
estimated at over four times the best: graph replays over three sets of operands in turn (out of L2).  `fit` reads
linear8_cost_data.json.gz beside this file and prints the constants and how far their choice is from the best
tile measured, with and without the 8-bit unit.  The data holds two lists of [M, N, K, out type, activation, residual type or
-1, [[tile, us], ...]]: "fitted", sweep --seed 31 --count 260, and "held_out", sweep --seed 47 --count 120.
"""
import argparse
import gzip
import json
import math
import random
import re
import sys
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent
CUS, F32, E4M3, FAST_RING, RING = 256, 0, 3, 13, 14


def table():
    """linear8_plan.hpp's tiles: number -> (rows, columns, 8-bit unit, workgroups a CU, constants)."""
    rows = re.findall(r"^ *LAYA_T\((\d+), (\d+), (\d+), [\d, ]+(true|false), (\d), ([\d.]+)f, ([\d.]+)f, ([\d.]+)f\)",
                      (HERE / "linear8_plan.hpp").read_text(), re.M)
    return {int(r[0]): (int(r[1]), int(r[2]), r[3] == "true", int(r[4]), [float(v) for v in r[5:]]) for r in rows}


def rings():
    """Its rings' constants: number -> list."""
    text = (HERE / "linear8_plan.hpp").read_text()
    return {ring: [float(v) for v in re.search(name + r"\[\] = \{([^}]*)\}", text)[1].replace("f", "").split(",")]
            for ring, name in ((FAST_RING, "kFastRingCost"), (RING, "kRingCost"))}


TILES = table()


def problems(seed, count):
    rng = random.Random(seed)

    def size():
        return rng.choice([768, 1024, 2304, 4096, int(math.exp(rng.uniform(math.log(64), math.log(4096))))])

    out = []
    while len(out) < count:
        M, N, K = int(round(math.exp(rng.uniform(0, math.log(65536))))), size(), size()
        act = rng.choice([0, 0, 1, 2, 3, 4])
        N = -(-N // 32) * 32 if act > 2 else N
        case = (M, N, K, rng.choice([0, 1, 2, 2, 3, 3]), act, rng.choice([-1, -1, 0, 2]))
        if M * N * K <= 1 << 38:
            out.append(case)
    return out


def padded(v):
    return -(-v // 128) * 128


def legal(tile, case):
    """linear8_plan.hpp's tile8_valid, and the ring's gate for aligned arrays."""
    M, N, K, out, act, res = case
    gated = act > 2
    cols = N // 2 if gated else N
    if tile >= FAST_RING:
        whole = out == E4M3 and (res < 0 or cols % 4 == 0) or out == F32 and cols % 4 == 0 or out in (1, 2) and cols % 8 == 0
        return whole and K > 128 and (tile == RING or out != F32)
    bm, bn, fast, _, _ = TILES[tile]
    return not (out == F32 and fast or gated and bn % 32 or out == E4M3 and (bn // 2 if gated else bn) % 32)


def features(tile, case):
    """What the constants of a tile, or of a ring, multiply."""
    M, N, K, out, act, res = case
    cols, n = N // 2 if act > 2 else N, -(-K // 128)
    span = padded(cols) if out == E4M3 else cols
    bm, bn, _, occ, _ = TILES.get(tile, (256, 256, None, 1, None))
    oc = bn // 2 if act > 2 else bn
    tiles = -(-span // oc) * -(-M // bm)
    if tile >= FAST_RING:
        full, rounds = min(tiles / CUS, 1), -(-tiles // CUS)
        return [1, full, n, rounds - 1, (rounds - 1) * n]
    share = 0.75 if tiles <= CUS and occ == 2 else 1.0
    rounds = -(-tiles // (CUS * occ)) * share
    return [1, rounds, rounds * n]


def present():
    return {**{tile: t[4] for tile, t in TILES.items()}, **rings()}


def choose(costs, case, fast):
    """The least estimated time of the tiles that the call may take, with the fast unit's or without."""
    def estimate(tile):
        return float(np.dot(costs[tile], features(tile, case)))
    return min((t for t in costs if legal(t, case) and (fast or not (t == FAST_RING or t in TILES and TILES[t][2]))), key=estimate)


def sweep(args):
    import torch
    sys.path.insert(0, str(HERE.parent))
    from laya_cuda import _lib
    lib, costs, types = _lib.load(), present(), {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
    rows = []
    for case in problems(args.seed, args.count):
        M, N, K, out, act, res = case
        cols, ld = N // 2 if act > 2 else N, padded(K)
        # Codes under 2 in magnitude: no NaNs.
        sets = [[torch.randint(0, 256, (r, ld), device="cuda", dtype=torch.uint8) & 0xbf for r in (M, N)]
                + [torch.full((r, ld // 32), 122, device="cuda", dtype=torch.uint8) for r in (M, N)] for _ in range(3)]
        bias = torch.zeros(N, device="cuda")
        residual = torch.zeros(M, cols, device="cuda", dtype=types[res]) if res >= 0 else None
        o = torch.empty(M, padded(cols), dtype=torch.uint8, device="cuda") if out == E4M3 else torch.empty(M, cols, dtype=types[out], device="cuda")
        scales = torch.empty(M, padded(cols) // 32, dtype=torch.uint8, device="cuda") if out == E4M3 else None

        def launch(i, tile):
            x, w, xs, ws = (t.data_ptr() for t in sets[i % 3])
            return lib.laya_op_linear8(x, xs, w, ws, bias.data_ptr(), residual.data_ptr() if res >= 0 else None, max(res, 0),
                                       o.data_ptr(), scales.data_ptr() if out == E4M3 else None, out, act, M, N, K, tile,
                                       torch.cuda.current_stream().cuda_stream)

        def time(tile):
            n = max(9, min(48, int(1e11 / (M * N * K))))
            _lib.check(launch(0, tile))
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                for i in range(n):
                    launch(i, tile)
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            graph.replay()
            us = []
            for _ in range(5):
                start.record()
                graph.replay()
                end.record()
                end.synchronize()
                us.append(start.elapsed_time(end) * 1e3 / n)
            return sorted(us)[2]

        tiles = [t for t in costs if legal(t, case)]
        estimate = {t: float(np.dot(costs[t], features(t, case))) for t in tiles}
        timed = [[t, round(time(t), 2)] for t in tiles if estimate[t] < 4 * min(estimate.values())]
        rows.append([*case, timed])
        print(*case, min((us, t) for t, us in timed), flush=True)
    Path(args.out).write_text(json.dumps(rows))


def fit(data):
    from scipy.optimize import least_squares
    out = {}
    for tile in present():
        A, us = [], []
        for *case, timed in data:
            best = min(t[1] for t in timed)
            for t, took in timed:
                if t == tile and took < 3 * best:  # where it may be the choice
                    A.append(features(t, tuple(case)))
                    us.append(took)
        A, us = np.array(A, float), np.array(us)
        start = np.array(present()[tile])
        found = least_squares(lambda x: (A @ x) / us - 1, start, bounds=([0] * len(start), [60] * len(start)), loss="soft_l1",
                              f_scale=0.1)
        out[tile] = found.x
    return out


def regret(costs, data, fast):
    """Mean, 95th percentile and largest ratio of the chosen tile's time to the best one's."""
    ratios = []
    for *case, timed in data:
        us = {t: v for t, v in timed if fast or not (t == FAST_RING or t in TILES and TILES[t][2])}
        pick = choose(costs, tuple(case), fast)
        ratios.append(us[pick] / min(us.values()) if pick in us else 4.0)  # not timed: estimated far off the best
    return f"mean {np.mean(ratios):.4f}, 95th percentile {np.quantile(ratios, .95):.3f}, largest {max(ratios):.3f} of {len(ratios)}"


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("do", choices=["sweep", "fit"])
    ap.add_argument("--seed", type=int, default=31)
    ap.add_argument("--count", type=int, default=260)
    ap.add_argument("--out", default="sweep.json")
    args = ap.parse_args()
    if args.do == "sweep":
        return sweep(args)
    data = json.loads(gzip.decompress((HERE / "linear8_cost_data.json.gz").read_bytes()))
    found = fit(data["fitted"])
    for name, costs in (("as built", present()), ("fitted", found)):
        for fast in (False, True):
            print(name, "fast" if fast else "exact", "| fitted:", regret(costs, data["fitted"], fast), "| held out:",
                  regret(costs, data["held_out"], fast))
    for tile, cost in found.items():
        print(tile, ", ".join("%.3ff" % v for v in cost))


if __name__ == "__main__":
    main()
