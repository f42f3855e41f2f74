"""8-bit rows on the GPU: quantising and reading back bit for bit, the norm and the product against 64 bits.

Tolerances count roundings (u = 2^-24, half a unit of fp32 relative to the value):
  * norm: a row's sums add at most 32 registers and 6 + 4 lane and wave partials, so they are within 48 u of the sum of
    magnitudes; 64 u covers the variance, the root and the division, and three multiplications and additions;
  * product, exact tiles: every 32-code step adds 32 products to fp32 accumulators in a tree of at most 6 levels, so a sum is
    within (steps + 6) 2 u of the sum of magnitudes (2 u: additions inside the matrix unit may truncate);
  * product, 8-bit matrix unit: it aligns a group's products before it adds them; on 256 sums of 4,096 products the error
    was at most 2^-14 of the root of the products' sum of squares; 2^-11 of it leaves 8 times that for longer tails;
  * then half a step of the output's type.
"""
import ctypes as ct

import numpy as np
import pytest

import rows8_reference as R
from laya_cuda import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
CODE = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16, "e4m3": _lib.E4M3}
ACT = {"none": 0, "gelu": 1, "relu": 2, "geglu": 3, "swiglu": 4}


def torch():
    import torch as t
    return t


def dtype(name):
    t = torch()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[name]


def p(x):
    return None if x is None else ct.c_void_p(x.data_ptr())


def stream():
    return ct.c_void_p(torch().cuda.current_stream().cuda_stream)


def check(code):
    _lib.check(code)


def up(x, gpu):
    return torch().from_numpy(np.ascontiguousarray(x)).to(gpu)


def f64(x):
    return x.double().cpu().numpy()


GUARD = 0x5a


class Rows8:
    """Device 8-bit rows with a guard row behind the last."""

    def __init__(self, gpu, rows, width):
        t, ld = torch(), R.width8(width)
        self.rows, self.width = rows, width
        self.codes = t.full((rows + 1, ld), GUARD, dtype=t.uint8, device=gpu)
        self.scales = t.full((rows + 1, ld // 32), GUARD, dtype=t.uint8, device=gpu)

    def host(self):
        codes, scales = self.codes.cpu().numpy(), self.scales.cpu().numpy()
        assert (codes[-1] == GUARD).all() and (scales[-1] == GUARD).all()
        return codes[:-1], scales[:-1]

    @classmethod
    def of(cls, gpu, x):
        self = cls(gpu, *x.shape)
        codes, scales = R.encode(x)
        self.codes[:-1], self.scales[:-1] = up(codes, gpu), up(scales, gpu)
        self.values = R.decode(codes, scales, x.shape[1])
        return self


def mixed(rng, rows, width):
    """Values over many magnitudes, with blocks of zeros, ties, denormals and the largest floats."""
    x = (rng.normal(0, 1, (rows, width)) * np.exp2(rng.integers(-30, 30, (rows, 1)))).astype(np.float32)
    x[rng.random((rows, width)) < .05] = 0
    x[0, : min(width, 32)] = 0
    if rows > 2:
        x[1] = np.float32(1.0625) * np.exp2(rng.integers(-3, 3, width))  # halfway between two codes
        x[2] = np.float32(2.0 ** -140) * rng.integers(-900, 900, width)
    if rows > 4:
        x[3] = np.float32(3.0e38) * np.sign(rng.normal(0, 1, width))
    return x


# ---------------- quantise, read back ----------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,extra", [(1, 1, 0), (3, 31, 1), (5, 128, 0), (7, 129, 3), (64, 768, 0), (33, 1000, 24),
                                              (2, 4095, 0), (1000, 260, 4)])
def test_quantize_is_bit_exact(gpu, kind, rows, width, extra):
    t, lib = torch(), _lib.load()
    rng = np.random.default_rng(rows * 5000 + width)
    x = up(mixed(rng, rows, width), gpu).to(dtype(kind))
    if kind == "f16":
        x = x.clamp(-60000, 60000)
    held = t.full((rows, width + extra), float("nan"), dtype=x.dtype, device=gpu)  # NaNs between the rows
    held[:, :width] = x
    out = Rows8(gpu, rows, width)
    check(lib.laya_op_quantize8(p(held), CODE[kind], width + extra, p(out.codes), p(out.scales), rows, width, stream()))
    codes, scales = out.host()
    want, want_scales = R.encode(f64(x))
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_that_is_not_finite_reads_back_as_nans(gpu, bad):
    t, lib = torch(), _lib.load()
    x = np.random.default_rng(3).normal(0, 1, (4, 200)).astype(np.float32)
    x[1, 37] = x[3, 199] = bad
    out = Rows8(gpu, 4, 200)
    held = up(x, gpu)
    check(lib.laya_op_quantize8(p(held), _lib.F32, 200, p(out.codes), p(out.scales), 4, 200, stream()))
    back = t.zeros(4, 200, device=gpu)
    check(lib.laya_op_dequantize8(p(out.codes), p(out.scales), p(back), _lib.F32, 200, 4, 200, stream()))
    nan = np.zeros((4, 200), bool)
    nan[1, 32:64] = nan[3, 192:] = True
    np.testing.assert_array_equal(np.isnan(f64(back)), nan)
    np.testing.assert_array_equal(f64(back), R.decode(*R.encode(x), 200))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,extra", [(1, 1, 0), (9, 127, 2), (16, 1024, 0), (5, 1000, 24), (257, 514, 0)])
def test_dequantize_every_code_and_leaves_the_gaps(gpu, kind, rows, width, extra):
    t, lib = torch(), _lib.load()
    rng = np.random.default_rng(width)
    codes = rng.integers(0, 256, (rows, R.width8(width))).astype(np.uint8)
    scales = rng.integers(110, 140, (rows, R.width8(width) // 32)).astype(np.uint8)
    scales[0, 0] = 255
    if rows > 4:
        scales[1], scales[2] = 0, 247
    out = t.full((rows, width + extra), 7.0, dtype=dtype(kind), device=gpu)
    c, s = up(codes, gpu), up(scales, gpu)
    check(lib.laya_op_dequantize8(p(c), p(s), p(out), CODE[kind], width + extra, rows, width, stream()))
    want = t.from_numpy(R.decode(codes, scales, width)).to(dtype(kind))
    got = out.cpu()
    assert (got[:, width:] == 7).all()
    np.testing.assert_array_equal(got[:, :width].float().numpy(), want.float().numpy())


def test_quantize_offsets_past_32_bits(gpu):
    """Rows 2^21 elements apart: the last starts past 2^32 elements; the first and the last come out right."""
    t, lib = torch(), _lib.load()
    rows, stride, width = 2100, 1 << 21, 96
    x = t.zeros(rows * stride, dtype=t.bfloat16, device=gpu)
    v = t.randn(rows, width, device=gpu, generator=t.Generator(device=gpu).manual_seed(1)).to(t.bfloat16)
    x.view(rows, stride)[:, :width] = v
    out = Rows8(gpu, rows, width)
    check(lib.laya_op_quantize8(p(x), _lib.BF16, stride, p(out.codes), p(out.scales), rows, width, stream()))
    codes, scales = out.host()
    want, want_scales = R.encode(f64(v))
    np.testing.assert_array_equal(codes, want)
    np.testing.assert_array_equal(scales, want_scales)
    check(lib.laya_op_dequantize8(p(out.codes), p(out.scales), p(x), _lib.BF16, stride, rows, width, stream()))
    np.testing.assert_array_equal(f64(x.view(rows, stride)[:, :width]), R.decode(want, want_scales, width))
    assert int((x.view(rows, stride)[:, width:] != 0).sum()) == 0


# ---------------- residual add and norm ----------------

def run_norm(gpu, rng, rows, width, kind, branch, splits, bias, beta, alias=None, shift=0, scale=1.0):
    t, lib = torch(), _lib.load()
    normal = lambda *s: rng.normal(0, 1, s).astype(np.float32)  # noqa: E731
    # shift: elements by which every array is moved off its allocation's alignment
    def place(x):
        held = t.empty(x.size + shift, dtype=t.float32, device=gpu)
        held[shift:] = up(x.reshape(-1), gpu)
        return held[shift:].view(x.shape)
    residual = place(normal(rows, width) * scale)
    gap = 0 if splits == 1 else 12
    parts = None
    if branch:
        parts = t.full((splits, rows * width + gap), float("nan"), dtype=dtype(branch), device=gpu)
        parts[:, :rows * width] = up(normal(splits, rows * width), gpu).to(dtype(branch))
    b = place(normal(width)) if bias else None
    gamma, be = place(1 + .1 * normal(width)), place(.1 * normal(width)) if beta else None
    before = f64(residual)
    total = t.full((rows + 1, width), 3.0, device=gpu)
    out32 = t.full((rows + 1, width), 3.0, device=gpu)
    s_out = residual if alias == "sum" else total
    y_out = residual if alias == "out32" else out32
    out = Rows8(gpu, rows, width)
    check(lib.laya_op_norm8(p(residual), p(parts), CODE[branch or "f32"], splits, rows * width + gap, p(b), p(gamma), p(be),
                            1e-5, kind, p(s_out), p(y_out), p(out.codes), p(out.scales), rows, width, stream()))
    codes, scales = out.host()
    for held in (total, out32):
        assert (held[rows:] == 3).all()
    got_sum, got = s_out.cpu().numpy()[:rows], y_out.cpu().numpy()[:rows]
    # The sum's order: partials, bias, residual, one fp32 rounding each.
    want_sum = before.astype(np.float32)
    if branch:
        acc = parts[0, :rows * width].float().cpu().numpy().reshape(rows, width)
        for i in range(1, splits):
            acc = acc + parts[i, :rows * width].float().cpu().numpy().reshape(rows, width)
        if bias:
            acc = acc + b.cpu().numpy()
        want_sum = want_sum + acc
    np.testing.assert_array_equal(got_sum, want_sum)
    v, g = want_sum.astype(np.float64), f64(gamma)
    want = R.norm(v, g, None if be is None else f64(be), 1e-5, kind == _lib.RMS_NORM)
    c = v if kind == _lib.RMS_NORM else v - v.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + 1e-5)
    bound = U * (np.abs(g) * inv * (48 * np.abs(v).mean(-1, keepdims=True) * (kind == _lib.LAYER_NORM) + 2 * np.abs(v))
                 + 64 * np.abs(c * inv * g) + 2 * np.abs(want))
    assert (np.abs(got - want) <= bound).all()
    want_codes, want_scales = R.encode(got.astype(np.float64))
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)


@pytest.mark.parametrize("kind", [_lib.LAYER_NORM, _lib.RMS_NORM])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 768), (3, 33), (17, 255), (9, 1000), (300, 768), (5, 1024), (6, 1088),
                                        (2, 2048), (3, 2049), (4, 4096), (2, 6000), (3, 8191), (2, 8192), (4100, 260)])
def test_norm_against_64_bits(gpu, kind, rows, width):
    rng = np.random.default_rng(rows + width)
    run_norm(gpu, rng, rows, width, kind, "f32", 2, True, kind == _lib.LAYER_NORM)


@pytest.mark.parametrize("kind", [_lib.LAYER_NORM, _lib.RMS_NORM])
@pytest.mark.parametrize("branch,splits,bias,beta,alias,shift", [
    (None, 1, False, False, None, 0), (None, 1, False, True, "sum", 0), ("f16", 1, True, True, "sum", 0),
    ("bf16", 1, False, False, "out32", 0), ("f32", 1, True, True, "out32", 0), ("f32", 3, False, True, None, 0),
    ("f32", 9, True, False, "sum", 0), ("bf16", 4, True, True, None, 0), ("f16", 2, False, True, None, 1),
    ("f32", 2, True, True, "sum", 1), ("bf16", 1, True, False, "out32", 3)])
def test_norm_branches_aliases_and_alignments(gpu, kind, branch, splits, bias, beta, alias, shift):
    rng = np.random.default_rng(splits * 100 + shift)
    for rows, width in ((21, 768), (2, 2500)):
        run_norm(gpu, rng, rows, width, kind, branch, splits, bias, beta, alias, shift)


@pytest.mark.parametrize("scale", [1e-18, 1e15])
def test_norm_of_tiny_and_huge_rows(gpu, scale):
    run_norm(gpu, np.random.default_rng(4), 8, 512, _lib.RMS_NORM, None, 1, False, False, scale=scale)


def test_norm_rows_with_nan_and_zeros_stay_apart(gpu):
    """A NaN spoils its own row alone; a row of zeros is zeros (eps keeps the root finite)."""
    t, lib = torch(), _lib.load()
    x = np.random.default_rng(5).normal(0, 1, (5, 300)).astype(np.float32)
    x[1, 7], x[3] = np.nan, 0
    out, y = Rows8(gpu, 5, 300), t.zeros(5, 300, device=gpu)
    held, ones = up(x, gpu), t.ones(300, device=gpu)
    check(lib.laya_op_norm8(p(held), None, _lib.F32, 1, 0, None, p(ones), None, 1e-5,
                            _lib.RMS_NORM, None, p(y), p(out.codes), p(out.scales), 5, 300, stream()))
    codes, scales = out.host()
    np.testing.assert_array_equal(np.isnan(f64(y)).all(-1), [False, True, False, False, False])
    assert (scales[1, :10] == 255).all() and not (scales[[0, 2, 3, 4]] == 255).any()
    assert (codes[3] == 0).all() and (scales[3] == 0).all()


# ---------------- product ----------------

def linear(gpu, x, w, *, act="none", bias=None, residual=None, rtype="f32", out="f32", tile=-1, inplace=False):
    """(values, bound) of laya_op_linear8 beside the 64-bit product: returns got, want, tolerance."""
    t, lib = torch(), _lib.load()
    M, K, N = x.rows, x.width, w.rows
    cols = N // 2 if act in ("geglu", "swiglu") else N
    res = None if residual is None else t.cat([up(residual, gpu).to(dtype(rtype)), t.full((1, cols), 9.0, device=gpu, dtype=dtype(rtype))])
    kept = None if res is None else f64(res)[:M]
    b = None if bias is None else up(bias, gpu)
    if out == "e4m3":
        o = Rows8(gpu, M, cols)
        outs = p(o.codes), p(o.scales)
    else:
        o = res if inplace else t.full((M + 1, cols), 9.0, dtype=dtype(out), device=gpu)
        outs = p(o), None
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), p(b), p(res), CODE[rtype], *outs, CODE[out],
                              ACT[act], M, N, K, tile, stream()))
    with np.errstate(invalid="ignore", over="ignore"):
        v = x.values @ w.values.T
        mag = np.abs(x.values) @ np.abs(w.values).T
        sq = np.sqrt((x.values ** 2) @ (w.values ** 2).T)
        if bias is not None:
            v, mag = v + bias.astype(np.float64), mag + np.abs(bias)
        steps = R.width8(K) // 32
        tol = (steps + 6) * 2 * U * mag + (0 if out == "f32" else 2.0 ** -11 * sq)
        want = R.activate(v, act)
        if act in ("geglu", "swiglu"):  # |act'| <= 1.13 and |act(g)| <= |g|
            g = v.reshape(M, -1, 2, 16)
            e = tol.reshape(M, -1, 2, 16)
            tol = (1.13 * e[:, :, 0] * np.abs(g[:, :, 1]) + e[:, :, 1] * (np.abs(g[:, :, 0]) + e[:, :, 0])).reshape(M, -1)
            tol += 1e-6 * np.abs(g[:, :, 1]).reshape(M, -1) + 4 * U * np.abs(want)
        elif act != "none":
            tol = 1.13 * tol + 1e-6
        if residual is not None:
            want = want + kept
            tol = tol + U * np.abs(want)
    if out == "e4m3":
        codes, scales = o.host()
        assert (codes[:, cols:] == 0).all()
        top = np.repeat(np.abs(np.pad(want, ((0, 0), (0, R.width8(cols) - cols)))).reshape(M, -1, 32).max(-1), 32, 1)[:, :cols]
        # Half a step of a code, or of the smallest code at the block's scale (at most top / 448 * 2).
        return R.decode(codes, scales, cols), want, tol + 2.0 ** -4 * (np.abs(want) + tol) + 2.0 ** -10 * (top + tol.max()) / 224
    assert (o[M:] == 9).all()
    return f64(o)[:M], want, tol + HALF[out] * (np.abs(want) + tol)


def close(got, want, tol):
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    off = np.abs(got - want)[~nan] - np.broadcast_to(tol, want.shape)[~nan]
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} beyond, worst by {off.max()}"


def operands(gpu, rng, M, N, K):
    return (Rows8.of(gpu, rng.normal(0, 1, (M, K)) * np.exp(rng.normal(0, .5, K))), Rows8.of(gpu, rng.normal(0, K ** -.5, (N, K))))


def tiles(M, N, K, act="none", out="f32"):
    """Tiles that take this output (refused ones are skipped), and the planner's."""
    return [-1, *range(64)]


def every_tile(gpu, x, w, **kw):
    ran = 0
    for tile in tiles(0, 0, 0):
        try:
            got = linear(gpu, x, w, tile=tile, **kw)
        except RuntimeError as e:
            assert "no such tile" in str(e) and tile >= 0
            continue
        close(*got)
        ran += 1
    assert ran >= 2  # the planner's choice and at least one tile by name


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (1, 1, 1), (2, 33, 31), (17, 100, 129), (16, 256, 512), (33, 130, 300),
                                   (129, 513, 1088), (64, 128, 4096), (300, 96, 640), (257, 300, 2100)])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
def test_linear_sizes_on_every_tile(gpu, M, N, K, out):
    rng = np.random.default_rng(M * 7 + N)
    x, w = operands(gpu, rng, M, N, K)
    every_tile(gpu, x, w, out=out, bias=rng.normal(0, .5, N).astype(np.float32))


@pytest.mark.parametrize("act", ["none", "gelu", "relu", "geglu", "swiglu"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("rtype", ["", "f32", "f16", "bf16"])
def test_linear_epilogues(gpu, act, out, rtype):
    rng = np.random.default_rng(len(act) + len(out))
    for M, N, K in ((19, 192, 256), (150, 1056, 384)):
        x, w = operands(gpu, rng, M, N, K)
        cols = N // 2 if act in ("geglu", "swiglu") else N
        every_tile(gpu, x, w, act=act, out=out, bias=rng.normal(0, .5, N).astype(np.float32),
                   residual=rng.normal(0, 1, (M, cols)).astype(np.float32) if rtype else None, rtype=rtype or "f32")


@pytest.mark.parametrize("M,N,K", [(4200, 4352, 256), (4333, 4416, 384), (65, 66048, 640)])
@pytest.mark.parametrize("out,act,rtype", [("bf16", "none", "bf16"), ("f16", "gelu", ""), ("e4m3", "relu", ""), ("f32", "none", "f32"),
                                           ("f32", "swiglu", ""), ("e4m3", "geglu", ""), ("bf16", "swiglu", "f32")])
def test_linear_more_tiles_than_compute_units(gpu, M, N, K, out, act, rtype):
    """The tile with the highest number (the persistent one) walks several tiles a workgroup: every output against 64 bits."""
    t, lib = torch(), _lib.load()
    gen = t.Generator(device=gpu).manual_seed(M)
    normal = lambda *s: t.randn(*s, device=gpu, generator=gen)  # noqa: E731

    def rows8(n, k, std):
        held = Rows8(gpu, n, k)
        v = normal(n, k) * std
        check(lib.laya_op_quantize8(p(v), _lib.F32, k, p(held.codes), p(held.scales), n, k, stream()))
        back = t.empty(n, k, device=gpu)
        check(lib.laya_op_dequantize8(p(held.codes), p(held.scales), p(back), _lib.F32, k, n, k, stream()))
        return held, back.double()

    (x, xv), (w, wv) = rows8(M, K, 1.0), rows8(N, K, K ** -.5)
    gated = act in ("geglu", "swiglu")
    cols = N // 2 if gated else N
    bias = normal(N) * .5
    res = normal(M, cols).to(dtype(rtype)) if rtype else None
    o = Rows8(gpu, M, cols) if out == "e4m3" else t.full((M + 1, cols), 9.0, dtype=dtype(out), device=gpu)
    args = (p(x.codes), p(x.scales), p(w.codes), p(w.scales), p(bias), p(res), CODE[rtype or "f32"],
            *((p(o.codes), p(o.scales)) if out == "e4m3" else (p(o), None)), CODE[out], ACT[act], M, N, K)
    for tile in range(63, -1, -1):
        if lib.laya_op_linear8(*args, tile, stream()) == _lib.OK:
            break
    assert tile > 0
    wt = wv.t().contiguous()
    v = xv @ wt + bias.double()
    # As the small cases': (steps + 6) 2 u of the magnitudes, and 2^-11 of the products' root sum of squares on the 8-bit unit.
    tol = (R.width8(K) // 32 + 6) * 2 * U * (xv.abs() @ wt.abs() + bias.abs().double())
    if out != "f32":
        tol += 2.0 ** -11 * ((xv ** 2) @ (wt ** 2)).sqrt()
    gelu = lambda g: g * t.special.ndtr(g)  # noqa: E731
    if gated:
        g, e = v.view(M, -1, 2, 16), tol.view(M, -1, 2, 16)
        a = gelu(g[:, :, 0]) if act == "geglu" else g[:, :, 0] * t.sigmoid(g[:, :, 0])
        want = (a * g[:, :, 1]).reshape(M, -1)
        tol = (1.13 * e[:, :, 0] * g[:, :, 1].abs() + e[:, :, 1] * (g[:, :, 0].abs() + e[:, :, 0]) + 1e-6 * g[:, :, 1].abs()).reshape(M, -1)
        tol += 4 * U * want.abs()
    else:
        want = gelu(v) if act == "gelu" else v.clamp(min=0) if act == "relu" else v
        if act != "none":
            tol = 1.13 * tol + 1e-6
    if res is not None:
        want = want + res.double()
        tol += U * want.abs()
    if out == "e4m3":
        assert (o.codes[-1] == GUARD).all() and (o.scales[-1] == GUARD).all()
        back = t.empty(M, cols, device=gpu)
        check(lib.laya_op_dequantize8(p(o.codes), p(o.scales), p(back), _lib.F32, cols, M, cols, stream()))
        pad = R.width8(cols) - cols
        assert not pad or not o.codes[:-1, cols:].any()
        top = t.nn.functional.pad(want.abs(), (0, pad)).view(M, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :cols]
        got, tol = back.double(), tol + 2.0 ** -4 * (want.abs() + tol) + 2.0 ** -10 * (top + tol.max()) / 224
    else:
        assert (o[M:] == 9).all()
        got, tol = o[:M].double(), tol + HALF[out] * (want.abs() + tol)
    off = (got - want).abs() - tol
    assert (off <= 0).all(), f"{int((off > 0).sum())} beyond, worst by {float(off.max())}"


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N", [(7, 64), (7, 67), (400, 640)])
def test_linear_onto_its_own_residual(gpu, out, M, N):
    rng = np.random.default_rng(M + N)
    x, w = operands(gpu, rng, M, N, 768)
    close(*linear(gpu, x, w, out=out, rtype=out, residual=rng.normal(0, 1, (M, N)).astype(np.float32), inplace=True))


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_linear_onto_its_own_residual_on_every_tile(gpu, out, act):
    """Rows and columns that end inside every tile: each reads a residual place before any lane writes it."""
    rng = np.random.default_rng(31)
    x, w = operands(gpu, rng, 300, 1184, 384)
    every_tile(gpu, x, w, act=act, out=out, rtype=out, inplace=True, bias=rng.normal(0, .5, 1184).astype(np.float32),
               residual=rng.normal(0, 1, (300, 592 if act == "swiglu" else 1184)).astype(np.float32))


def test_linear_nan_blocks_and_the_largest_codes(gpu):
    """A NaN block spoils its row (of x) or column (of w) alone, on every tile and in 8-bit outputs its whole block."""
    rng = np.random.default_rng(9)
    a, b = rng.normal(0, 1, (40, 384)), rng.normal(0, 1, (160, 384))
    a[3, 200], b[77, 0] = np.nan, np.inf
    a[5], b[9] = 448.0, -448.0
    x, w = Rows8.of(gpu, a), Rows8.of(gpu, b)
    for out in ("f32", "bf16"):
        every_tile(gpu, x, w, out=out)
    t, lib = torch(), _lib.load()
    o = Rows8(gpu, 40, 160)
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, None, 0, p(o.codes), p(o.scales),
                              _lib.E4M3, 0, 40, 160, 384, -1, stream()))
    nan = np.isnan(R.decode(*o.host(), 160))
    want = np.zeros((40, 160), bool)
    want[3], want[:, 64:96] = True, True
    np.testing.assert_array_equal(nan, want)


def test_linear_scales_far_apart(gpu):
    """Scales from 2^-60 to 2^60 whose products meet in the middle."""
    rng = np.random.default_rng(11)
    e = rng.integers(-60, 60, 12).repeat(32)
    x = Rows8.of(gpu, rng.normal(0, 1, (20, 384)) * np.exp2(e))
    w = Rows8.of(gpu, rng.normal(0, 1, (64, 384)) * np.exp2(-e))
    for out in ("f32", "f16"):
        every_tile(gpu, x, w, out=out)


def test_linear_repeats_bit_for_bit(gpu):
    t, lib = torch(), _lib.load()
    rng = np.random.default_rng(12)
    x, w = operands(gpu, rng, 200, 256, 1024)
    outs = []
    for _ in range(3):
        o = t.empty(200, 256, device=gpu)
        check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, None, 0, p(o), None, _lib.F32, 0,
                                  200, 256, 1024, -1, stream()))
        outs.append(o)
    assert t.equal(outs[0], outs[1]) and t.equal(outs[0], outs[2])


def test_linear_offsets_past_32_bits(gpu):
    """Codes and output past 2^32 bytes: rows at both ends of 4.3 GB of x and of an 8.6 GB output are right."""
    t, lib = torch(), _lib.load()
    M, N, K = 1 << 22, 1024, 1088  # 4,194,304 x 1,152 codes
    rng = np.random.default_rng(13)
    ends = np.r_[0:40, M - 40:M]
    x, w = operands(gpu, rng, 80, N, K)
    codes = t.zeros(M, 1152, dtype=t.uint8, device=gpu)
    scales = t.zeros(M, 36, dtype=t.uint8, device=gpu)
    at = t.from_numpy(ends).to(gpu)
    codes[at], scales[at] = x.codes[:80], x.scales[:80]
    out = t.full((M, N), 5.0, dtype=t.bfloat16, device=gpu)
    check(lib.laya_op_linear8(p(codes), p(scales), p(w.codes), p(w.scales), None, None, 0, p(out), None, _lib.BF16, 0, M, N, K,
                              -1, stream()))
    want = x.values @ w.values.T
    sq = np.sqrt((x.values ** 2) @ (w.values ** 2).T)
    close(f64(out[at]), want, 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * sq)
    assert int((out[40:M - 40] != 0).sum()) == 0


# ---------------- together ----------------

def ffn(lib, gpu, s, buffers):
    """A pre-norm block's FFN on 8-bit rows: norm, gated up projection into 8 bits, down projection onto the residual."""
    h, u = buffers["h"], buffers["u"]
    rows, d, f = s["rows"], s["d"], s["f"]
    check(lib.laya_op_norm8(p(s["res"]), p(s["branch"]), _lib.BF16, 1, 0, None, p(s["gamma"]), None, 1e-5, _lib.RMS_NORM,
                            p(buffers["sum"]), None, p(h.codes), p(h.scales), rows, d, stream()))
    check(lib.laya_op_linear8(p(h.codes), p(h.scales), p(s["up"].codes), p(s["up"].scales), None, None, 0, p(u.codes),
                              p(u.scales), _lib.E4M3, _lib.ACT_SWIGLU, rows, 2 * f, d, -1, stream()))
    check(lib.laya_op_linear8(p(u.codes), p(u.scales), p(s["down"].codes), p(s["down"].scales), None, p(buffers["sum"]),
                              _lib.F32, p(buffers["out"]), None, _lib.F32, 0, rows, d, f, -1, stream()))


def block(gpu, rng, rows, d=256, f=384):
    t = torch()
    s = {"rows": rows, "d": d, "f": f, "res": up(rng.normal(0, 1, (rows, d)).astype(np.float32), gpu),
         "branch": up(rng.normal(0, 1, (rows, d)).astype(np.float32), gpu).bfloat16(),
         "gamma": up(1 + .1 * rng.normal(0, 1, d).astype(np.float32), gpu)}
    for name, n, k in (("up", 2 * f, d), ("down", d, f)):
        wt = up(rng.normal(0, k ** -.5, (n, k)).astype(np.float32), gpu)
        held = Rows8(gpu, n, k)
        check(_lib.load().laya_op_quantize8(p(wt), _lib.F32, k, p(held.codes), p(held.scales), n, k, stream()))
        s[name] = held
    buffers = {"h": Rows8(gpu, rows, d), "u": Rows8(gpu, rows, f), "sum": t.empty(rows, d, device=gpu),
               "out": t.empty(rows, d, device=gpu)}
    return s, buffers


def ffn_reference(s, buffers):
    """Step by step from what the step before left on the device, so that each step's own tolerance holds."""
    total = f64(s["res"]) + f64(s["branch"])
    np.testing.assert_allclose(f64(buffers["sum"]), total, rtol=0, atol=8 * 2 * U)  # |v| < 16: one rounding
    y = R.norm(total, f64(s["gamma"]), None, 1e-5, True)
    h = R.decode(*buffers["h"].host(), s["d"])
    assert (np.abs(h - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -9 * np.abs(y).max() / 224 + 1e-6).all()
    up_w, down_w = (R.decode(*s[k].host(), k2) for k, k2 in (("up", s["d"]), ("down", s["f"])))
    mid = R.activate(h @ up_w.T, "swiglu")
    u = R.decode(*buffers["u"].host(), s["f"])
    g = (h @ up_w.T).reshape(len(h), -1, 2, 16)
    e = 2.0 ** -11 * np.sqrt((h ** 2) @ (up_w ** 2).T).reshape(len(h), -1, 2, 16)
    tol = ((1.13 * np.abs(g[:, :, 1]) + 1) * e[:, :, 0] + (np.abs(g[:, :, 0]) + 1) * e[:, :, 1]).reshape(mid.shape)
    assert (np.abs(u - mid) <= tol + 2.0 ** -4 * (np.abs(mid) + tol) + 2.0 ** -9 * np.abs(mid).max() / 224 + 1e-6).all()
    out = u @ down_w.T + f64(buffers["sum"])
    mag = np.abs(u) @ np.abs(down_w).T + np.abs(f64(buffers["sum"]))
    assert (np.abs(f64(buffers["out"]) - out) <= (R.width8(s["f"]) // 32 + 8) * 2 * U * mag).all()


@pytest.mark.parametrize("rows", [1, 37, 300])
def test_an_ffn_block_on_8_bit_rows(gpu, rows):
    lib = _lib.load()
    s, buffers = block(gpu, np.random.default_rng(rows), rows)
    ffn(lib, gpu, s, buffers)
    ffn_reference(s, buffers)


def test_two_captured_blocks_replay_side_by_side(gpu):
    """Two blocks captured on their own streams, replayed in turn and together with new inputs: bit-equal to the
    eager run every time."""
    t, lib = torch(), _lib.load()
    made = [block(gpu, np.random.default_rng(20 + i), rows) for i, rows in enumerate((300, 45))]
    for s, buffers in made:
        ffn(lib, gpu, s, buffers)
    t.cuda.synchronize()
    graphs = []
    for s, buffers in made:
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            ffn(lib, gpu, s, buffers)
        graphs.append((g, t.cuda.Stream()))
    for turn in range(4):
        want = []
        for s, buffers in made:
            s["res"].copy_(t.randn(s["rows"], s["d"], generator=t.Generator().manual_seed(turn)).to(gpu))
            ffn(lib, gpu, s, buffers)
            want.append(buffers["out"].clone())
            buffers["out"].zero_()
        t.cuda.synchronize()
        for g, st in graphs:
            with t.cuda.stream(st):
                g.replay()
        t.cuda.synchronize()
        for (s, buffers), w in zip(made, want):
            assert t.equal(buffers["out"], w)


def test_calls_follow_the_given_stream(gpu):
    """Work queued behind a slow producer on a side stream waits for it: the stream argument orders the call."""
    t, lib = torch(), _lib.load()
    side = t.cuda.Stream()
    x = t.zeros(4096, 768, device=gpu)
    out = Rows8(gpu, 4096, 768)
    t.cuda.synchronize()
    with t.cuda.stream(side):
        a = t.randn(4096, 4096, device=gpu)
        for _ in range(10):
            a = a @ a * 1e-3
        x.fill_(2.0)
        check(lib.laya_op_quantize8(p(x), _lib.F32, 768, p(out.codes), p(out.scales), 4096, 768, stream()))
    side.synchronize()
    codes, scales = out.host()
    assert (scales[:, :24] == 120).all() and (codes[:, :768] == 0x78).all()
