"""laya_op_linear, laya_op_rotary and laya_op_attend beside the fused path of the encoder (laya_op_qkv, laya_op_attention): the same queries,
keys and values from both, and the same outputs from the same queries, keys and values, in bounds that no other output meets.

Queries and keys: the fused epilogue rotates the product's fp32 sums and rounds once; the other path rounds the sums, which moves a
turned pair by up to h (|a| + |b|), and rounds again.  Sums of K products in any order differ by 2 K u of sum |x||w|; sine, cosine and
the products add (5e-8 + 10 u) (|a| + |b|), the fused path's tables being rounded to fp32.  Outputs: each path is within the bound of
attend_reference.py of its own inputs in 64 bits, so two paths over the same ones are within twice it.
"""
import ctypes as ct

import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib

HEADS, DIM, LENGTHS = 4, 64, [96, 150, 33]
WIDTH = HEADS * DIM
SPANS = [-(-n // 16) * 16 for n in LENGTHS]  # the fused path's sequences begin at whole 16 rows
STARTS = np.cumsum([0] + SPANS)[:-1]
ROWS = sum(SPANS) + 16


def halves(x, kind):
    import torch as t
    return t.from_numpy(x).to({"f16": t.float16, "bf16": t.bfloat16}[kind]).double().numpy()


def inputs(kind, seed=4):
    rng = np.random.default_rng(seed)
    x = halves(rng.normal(0, 1, (ROWS, WIDTH)), kind)
    w = halves(rng.normal(0, WIDTH ** -0.5, (3 * WIDTH, WIDTH)), kind)
    positions = np.zeros(ROWS, np.int32)
    for a, n in zip(STARTS, LENGTHS):
        positions[a:a + n] = np.arange(n)
    return x, w, positions, 10000.0 ** (-np.arange(0, DIM, 2) / DIM) / (2 * np.pi)


def attended(q, k, v, window, kind):
    """64 bits, and the bound, of every sequence's rows; q, k, v [rows][heads][dim]."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for a, n in zip(STARTS, LENGTHS):
        rows = slice(a, a + n)
        out[rows], bound[rows] = A.attend(q[rows], k[rows], v[rows], 0.125, before=window, after=window, kind=kind)
    return out, bound


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("window", [-1, 20])
def test_the_bound_tells_other_outputs(kind, window):
    """Zeros, heads in another order, a sequence's keys one place off, and half of the window too many: most values pass twice the bound."""
    x, w, positions, turns = inputs(kind)
    packed = (x @ w.T).reshape(ROWS, 3, HEADS, DIM)
    q, k = (halves(A.rotate(packed[:, i], positions, turns), kind) for i in (0, 1))
    v = halves(packed[:, 2], kind)
    want, bound = attended(q, k, v, window, kind)
    real = np.concatenate([np.arange(a, a + n) for a, n in zip(STARTS, LENGTHS)])
    wrong = {"zeros": np.zeros_like(want), "heads": want[:, [1, 0, 3, 2]], "keys": attended(q, np.roll(k, 1, 0), v, window, kind)[0]}
    if window >= 0:
        wrong["window"] = attended(q, k, v, window + 10, kind)[0]
    for name, other in wrong.items():
        passed = (np.abs(other - want) > 2 * bound)[real].mean()
        assert passed > 0.5, (name, passed)
    assert (bound[real] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("window", [-1, 20])
@pytest.mark.parametrize("kernel", [_lib.ATTEND_MANY, _lib.ATTEND_FEW], ids=["many", "few"])
def test_both_paths_agree(gpu, kind, window, kernel):
    import torch as t
    lib, code, h = _lib.load(), {"f16": _lib.F16, "bf16": _lib.BF16}[kind], A.HALF[kind]
    dtype = {"f16": t.float16, "bf16": t.bfloat16}[kind]
    x, w, positions, turns = inputs(kind)
    stream = ct.c_void_p(t.cuda.current_stream().cuda_stream)
    up = lambda a: t.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
    at = lambda a: a.data_ptr()  # noqa: E731
    xd, wd, p, f = up(x).to(dtype), up(w).to(dtype), up(positions), up(turns)

    angle = 2 * np.pi * np.arange(max(LENGTHS))[:, None] * turns
    cos, sin = up(np.cos(angle).astype(np.float32)), up(np.sin(angle).astype(np.float32))
    q, k = (t.empty(HEADS, ROWS, DIM, dtype=dtype, device=gpu) for _ in range(2))
    vt = t.empty(HEADS, DIM, ROWS, dtype=dtype, device=gpu)
    _lib.check(lib.laya_op_qkv(at(xd), at(wd), None, at(q), at(k), at(vt), at(cos), at(sin), at(p), code, ROWS, WIDTH, -1, stream))
    v = vt.transpose(1, 2).contiguous()

    packed = t.empty(ROWS, 3 * HEADS, DIM, dtype=dtype, device=gpu)
    _lib.check(lib.laya_op_linear(at(xd), at(wd), None, at(packed), 1, code, ROWS, 3 * WIDTH, WIDTH, 1, -1, stream))
    _lib.check(lib.laya_op_rotary(at(packed), 3 * WIDTH, DIM, at(packed), 3 * WIDTH, DIM, code, at(p), at(f), 1.0, 0, 1, ROWS, 2 * HEADS,
                                  DIM, DIM, stream))
    t.cuda.synchronize()
    wide = packed.double().cpu().numpy().reshape(ROWS, 3, HEADS, DIM)
    sums, sizes = ((a @ b.T).reshape(ROWS, 3, HEADS, DIM) for a, b in ((x, w), (np.abs(x), np.abs(w))))
    slack = 2 * WIDTH * A.U * sizes
    pair = np.abs(sums) + slack
    pair = pair[..., :DIM // 2] + pair[..., DIM // 2:]
    pair = np.concatenate([pair, pair], -1)
    pair_slack = np.concatenate([slack[..., :DIM // 2] + slack[..., DIM // 2:]] * 2, -1)
    for i, fused in enumerate((q, k)):
        fused = fused.double().cpu().numpy().transpose(1, 0, 2)
        allowed = (h + 5e-8 + 10 * A.U) * pair[:, i] + pair_slack[:, i] + h * (np.abs(fused) + np.abs(wide[:, i])) + 2.0 ** -24
        assert (np.abs(fused - wide[:, i]) <= allowed).all()
    values = v.double().cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(values - wide[:, 2]) <= slack[:, 2] + h * (np.abs(values) + np.abs(wide[:, 2])) + 2.0 ** -24).all()

    tiles = np.zeros((ROWS // 16, 4), np.int32)
    a32, l32, ip = STARTS.astype(np.int32), np.array(LENGTHS, np.int32), ct.POINTER(ct.c_int32)
    used = lib.laya_attention_tiles(a32.ctypes.data_as(ip), l32.ctypes.data_as(ip), len(LENGTHS), ROWS, lib.laya_attention_block(1, 4),
                                    tiles.ctypes.data_as(ip), ROWS // 16)
    assert used > 0
    listed, fused = up(tiles), t.empty(ROWS, HEADS, DIM, dtype=dtype, device=gpu)
    _lib.check(lib.laya_op_attention(at(q), at(k), at(vt), at(fused), at(listed), ROWS, HEADS, ROWS // 16, 1, 4, window, code, stream))

    starts, lengths, out = up(a32), up(l32), t.zeros(ROWS, HEADS, DIM, dtype=dtype, device=gpu)
    call = _lib.LayaAttend(struct_bytes=ct.sizeof(_lib.LayaAttend), dtype=code, q=at(q), k=at(k), v=at(v), out=at(out), q_row=DIM,
                           q_head=ROWS * DIM, k_row=DIM, k_head=ROWS * DIM, v_row=DIM, v_head=ROWS * DIM, out_row=WIDTH, out_head=DIM,
                           heads=HEADS, kv_heads=HEADS, dim=DIM, q_rows=ROWS, k_rows=ROWS, n_seq=len(LENGTHS), max_q=max(LENGTHS),
                           max_k=max(LENGTHS), q_starts=at(starts), q_lengths=at(lengths), k_starts=at(starts), k_lengths=at(lengths),
                           scale=0.125, before=window, after=window, kernel=kernel)
    assert lib.laya_attend_workspace(ct.byref(call)) == 0
    _lib.check(lib.laya_op_attend(ct.byref(call), None, 0, stream))
    t.cuda.synchronize()
    got, other = out.double().cpu().numpy(), fused.double().cpu().numpy()
    want, bound = attended(*(y.double().cpu().numpy().transpose(1, 0, 2) for y in (q, k, v)), window, kind)
    assert (np.abs(got - want) <= bound).all()
    real = np.concatenate([np.arange(a, a + n) for a, n in zip(STARTS, LENGTHS)])
    assert (np.abs(got - other) <= 2 * bound)[real].all(), np.max((np.abs(got - other) - 2 * bound)[real])
