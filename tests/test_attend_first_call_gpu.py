"""The first calls of a process on rotary positions, document bounds and attention, made while a graph captures; replays against eager
calls, with other inputs and lengths each time."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
SCRIPT = """
import ctypes as ct
import torch as t
from laya_cuda import _lib
lib = _lib.load()
rows, heads, dim, n = 700, 4, 64, 2
gen = t.Generator(device="cuda").manual_seed(1)
x = t.randn(rows, 3 * heads, dim, device="cuda", generator=gen).half()
turned, out = t.zeros_like(x), t.zeros(rows, heads, dim, device="cuda", dtype=t.float16)
i32 = lambda v: t.tensor(v, dtype=t.int32, device="cuda")
starts, lengths, positions = i32([0, 350]), i32([350, 349]), i32(list(range(350)) * 2)
ids, bounds = i32([i // 60 for i in range(rows)]), t.zeros(rows, 2, dtype=t.int32, device="cuda")
turns = (10000.0 ** (-t.arange(32, dtype=t.float64) / 32) / 6.283185307179586).cuda()
p = lambda v: v.data_ptr()
call = _lib.LayaAttend(struct_bytes=ct.sizeof(_lib.LayaAttend), dtype=_lib.F16, q=p(turned), k=p(turned) + 2 * heads * dim,
                       v=p(turned) + 4 * heads * dim, out=p(out), q_row=3 * heads * dim, q_head=dim, k_row=3 * heads * dim, k_head=dim,
                       v_row=3 * heads * dim, v_head=dim, out_row=heads * dim, out_head=dim, heads=heads, kv_heads=heads, dim=dim,
                       q_rows=rows, k_rows=rows, n_seq=n, max_q=350, max_k=350, q_starts=p(starts), q_lengths=p(lengths),
                       k_starts=p(starts), k_lengths=p(lengths), scale=0.125, cap=20.0, before=-1, after=-1, bounds=p(bounds), kernel=KERNEL)
need = lib.laya_attend_workspace(ct.byref(call))
workspace = t.empty(max(need, 16), dtype=t.uint8, device="cuda")


def calls():
    s = t.cuda.current_stream().cuda_stream
    _lib.check(lib.laya_op_rotary(p(x), 3 * heads * dim, dim, p(turned), 3 * heads * dim, dim, _lib.F16, p(positions), p(turns), 1.0, 0, 1,
                                  rows, 3 * heads, dim, dim, s))
    _lib.check(lib.laya_op_document_bounds(p(ids), p(starts), p(lengths), n, rows, 350, p(bounds), s))
    _lib.check(lib.laya_op_attend(ct.byref(call), p(workspace), workspace.numel(), s))


t.cuda.synchronize()
graph = t.cuda.CUDAGraph()
with t.cuda.graph(graph):
    calls()
for turn in range(3):
    x.copy_(t.randn(x.shape, device="cuda", generator=gen))
    lengths.copy_(i32([350 - 100 * turn, 349 - turn]))
    out.zero_()
    graph.replay()
    t.cuda.synchronize()
    got, seen = out.clone(), bounds.clone()
    out.zero_()
    calls()
    t.cuda.synchronize()
    assert t.equal(out, got) and t.equal(seen, bounds) and out.abs().sum() > 0
print("replayed")
"""


@pytest.mark.parametrize("kernel", [1, 2])
def test_first_calls_inside_a_capture(gpu, kernel):
    env = {**os.environ, "PYTHONPATH": str(ROOT / "laya-cuda_amd")}
    run = subprocess.run([sys.executable, "-c", SCRIPT.replace("KERNEL", str(kernel))], env=env, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "replayed" in run.stdout, run.stderr[-2000:]
