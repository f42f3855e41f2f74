"""The first calls of a process on 8-bit rows, made while a graph captures: what a call sets up once is no part of the graph
and does not break it."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
SCRIPT = """
import torch as t
from laya_cuda import _lib
lib = _lib.load()
M, N, K = 300, 512, 384
gen = t.Generator(device="cuda").manual_seed(1)
x = t.randn(M, K, device="cuda", generator=gen)
w = t.randn(N, K, device="cuda", generator=gen)
byte = lambda *s: t.zeros(*s, dtype=t.uint8, device="cuda")
xc, xs, wc, ws = byte(M, K), byte(M, K // 32), byte(N, K), byte(N, K // 32)
ones, out = t.ones(K, device="cuda"), t.zeros(M, N, device="cuda")


def calls(out, tile):
    s = t.cuda.current_stream().cuda_stream
    p = lambda v: v.data_ptr()
    _lib.check(lib.laya_op_norm8(p(x), None, 0, 1, 0, None, p(ones), None, 1e-5, 1, None, None, p(xc), p(xs), M, K, s))
    _lib.check(lib.laya_op_quantize8(p(w), 0, K, p(wc), p(ws), N, K, s))
    _lib.check(lib.laya_op_linear8(p(xc), p(xs), p(wc), p(ws), None, None, 0, p(out), None, 0, 0, M, N, K, tile, s))


t.cuda.synchronize()
graph = t.cuda.CUDAGraph()
with t.cuda.graph(graph):
    calls(out, TILE)
for turn in range(3):
    x.copy_(t.randn(M, K, device="cuda", generator=gen))
    out.zero_()
    graph.replay()
    t.cuda.synchronize()
    want = t.empty_like(out)
    calls(want, TILE)
    t.cuda.synchronize()
    assert t.equal(out, want) and out.abs().sum() > 0
print("replayed")
"""


@pytest.mark.parametrize("tile", [-1, 14])
def test_first_calls_inside_a_capture(gpu, tile):
    env = {**os.environ, "PYTHONPATH": str(ROOT / "laya-cuda_amd")}
    run = subprocess.run([sys.executable, "-c", SCRIPT.replace("TILE", str(tile))], env=env, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "replayed" in run.stdout, run.stderr[-2000:]
