"""Which tiles take which call of laya_op_linear8, against the rule written out here: a tile refused by mistake, or taken by
one, shows."""
import numpy as np
import pytest

import rows8_reference as R
from laya_cuda import _lib
from test_rows8_gpu import CODE, Rows8, check, dtype, f64, operands, p, stream, torch, up

pytestmark = pytest.mark.gpu

# rows, columns, 8-bit unit of the ordinary tiles; 13 and 14 are the rings
TILES = [(16, 16, False), (16, 32, False), (16, 64, False), (64, 32, False), (64, 64, False), (64, 64, True), (64, 64, False), (64, 64, True),
         (64, 128, True), (128, 128, True), (128, 128, True), (128, 128, False), (128, 128, False)]


def expected(out, act, cols, K, residual, aligned=True):
    gated = act in ("geglu", "swiglu")
    taken = {-1, -2}
    for tile, (_, bn, fast) in enumerate(TILES):
        if not (out == "f32" and fast or gated and bn % 32 or out == "e4m3" and (bn // 2 if gated else bn) % 32):
            taken.add(tile)
    whole = {"f32": cols % 4 == 0, "f16": cols % 8 == 0, "bf16": cols % 8 == 0, "e4m3": not residual or cols % 4 == 0}[out]
    if whole and aligned and K > 128:
        taken |= {14} if out == "f32" else {13, 14}
    return taken


@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("act,N", [("none", 256), ("gelu", 100), ("relu", 52), ("none", 33), ("geglu", 192), ("swiglu", 1056)])
@pytest.mark.parametrize("K", [100, 300])
@pytest.mark.parametrize("residual", [False, True])
def test_the_tiles_that_take_a_call(gpu, out, act, N, K, residual):
    t, lib = torch(), _lib.load()
    M, cols = 37, N // 2 if act in ("geglu", "swiglu") else N
    x, w = operands(gpu, np.random.default_rng(N + K), M, N, K)
    res = t.zeros(M, cols, device=gpu) if residual else None
    o = Rows8(gpu, M, cols) if out == "e4m3" else t.empty(M, cols, dtype=dtype(out), device=gpu)
    outs = (p(o.codes), p(o.scales)) if out == "e4m3" else (p(o), None)
    taken = set()
    for tile in range(-4, 64):
        code = lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, p(res), 0, *outs, CODE[out],
                                   ["none", "gelu", "relu", "geglu", "swiglu"].index(act), M, N, K, tile, stream())
        if code == _lib.OK:
            taken.add(tile)
        else:
            assert code == _lib.EINVAL and "no such tile" in _lib.error(None)
    t.cuda.synchronize()
    assert taken == expected(out, act, cols, K, residual)


@pytest.mark.parametrize("out", ["f32", "bf16", "e4m3"])
def test_alignments_that_the_rings_need(gpu, out):
    """A bias on any 4 bytes is taken; an output off 16 bytes takes another tile and gets the same values."""
    t, lib = torch(), _lib.load()
    M, N, K = 300, 512, 384
    x, w = operands(gpu, np.random.default_rng(3), M, N, K)
    bias = up(np.random.default_rng(4).normal(0, 1, N + 1).astype(np.float32), gpu)
    want = x.values @ w.values.T + f64(bias)[1:]

    def run(tile, shift=0):
        if out == "e4m3":
            o = Rows8(gpu, M, N)
            code = lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), p(bias[1:]), None, 0, p(o.codes), p(o.scales),
                                       _lib.E4M3, 0, M, N, K, tile, stream())
            return code, lambda: R.decode(*o.host(), N)
        o = t.empty(M * N + shift, dtype=dtype(out), device=gpu)[shift:]
        code = lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), p(bias[1:]), None, 0, p(o), None, CODE[out], 0,
                                   M, N, K, tile, stream())
        return code, lambda: f64(o).reshape(M, N)

    # A code's half step, or the smallest code's at the block's scale (tops here are under 8).
    tol = np.abs(want) * {"f32": 2.0 ** -20, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}[out] + {"f32": 1e-5, "bf16": 1e-5, "e4m3": 2.0 ** -10 * 8 / 224 * 2}[out]
    for tile in (-1, 14):
        code, got = run(tile)
        check(code)
        assert (np.abs(got() - want) <= tol).all()
    if out != "e4m3":
        for shift in (1, 2) if out == "bf16" else (1, 3):
            assert run(14, shift)[0] == _lib.EINVAL
            code, got = run(-1, shift)
            check(code)
            assert (np.abs(got() - want) <= tol).all()
