"""8-bit rows at the edges of what they hold: the largest finite values."""
import numpy as np
import pytest

import rows8_reference as R
from laya_cuda import _lib
from test_rows8_gpu import CODE, Rows8, check, dtype, f64, p, stream, torch, up

pytestmark = pytest.mark.gpu

TOP = 240 * 2.0 ** 120  # the largest value of 8-bit rows below 2^128
LARGE = np.array([2.0 ** 127, 232 * 2.0 ** 120, 247 * 2.0 ** 120, np.nextafter(np.float32(248 * 2.0 ** 120), np.float32(0)),
                  248 * 2.0 ** 120, 3.35e38, 255 * 2.0 ** 120, np.finfo(np.float32).max])


def large(rows, width):
    """Values of both signs up to the largest float, beside ordinary and small ones of the same blocks."""
    rng = np.random.default_rng(rows * width)
    x = rng.normal(0, 1, (rows, width)) * np.exp2(rng.integers(90, 126, (rows, width)))
    at = rng.random((rows, width)) < .3
    x[at] = rng.choice(LARGE, at.sum()) * rng.choice([-1, 1], at.sum())
    return x.astype(np.float32)


def expected(x):
    """To nearest, ties to even, as everywhere; what rounds to 2^128 is the largest value below it."""
    want = R.decode(*R.encode(x.astype(np.float64)), x.shape[1])
    return np.clip(want, -TOP, TOP)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width", [(3, 33), (64, 1024), (700, 4096)])
def test_finite_values_stay_finite(gpu, kind, rows, width):
    t, lib = torch(), _lib.load()
    x = up(large(rows, width), gpu).to(dtype(kind))
    x = t.where(t.isfinite(x), x, t.sign(x) * 255 * 2.0 ** 120)  # the largest bf16
    out = Rows8(gpu, rows, width)
    check(lib.laya_op_quantize8(p(x), CODE[kind], width, p(out.codes), p(out.scales), rows, width, stream()))
    back = t.empty(rows, width, device=gpu)
    check(lib.laya_op_dequantize8(p(out.codes), p(out.scales), p(back), _lib.F32, width, rows, width, stream()))
    out.host()
    np.testing.assert_array_equal(f64(back), expected(f64(x)))
    half = t.empty(rows, width, dtype=t.bfloat16, device=gpu)
    check(lib.laya_op_dequantize8(p(out.codes), p(out.scales), p(half), _lib.BF16, width, rows, width, stream()))
    np.testing.assert_array_equal(f64(half), expected(f64(x)))


def test_norm_outputs_stay_finite(gpu):
    """Rows of ones and minus ones have a root mean square of one: out32 is gamma (1 + 1e-5)^-1/2, up to the largest floats, and the
    codes are those of out32."""
    t, lib = torch(), _lib.load()
    x = up(np.random.default_rng(2).choice([-1.0, 1.0], (9, 300)).astype(np.float32), gpu)
    gamma = up(np.linspace(1e38, 3.4e38, 300).astype(np.float32), gpu)
    out, y = Rows8(gpu, 9, 300), t.empty(9, 300, device=gpu)
    check(lib.laya_op_norm8(p(x), None, _lib.F32, 1, 0, None, p(gamma), None, 1e-5, _lib.RMS_NORM, None, p(y), p(out.codes),
                            p(out.scales), 9, 300, stream()))
    got = f64(y)
    assert np.isfinite(got).all() and np.abs(got).max() > 3.39e38
    np.testing.assert_array_equal(R.decode(*out.host(), 300), expected(got))


@pytest.mark.parametrize("act,tile", [("none", tile) for tile in (-1, -2, 3, 4, 6, 8, 10, 12, 13, 14)] + [("swiglu", -1), ("swiglu", 13), ("swiglu", 14)])
def test_product_outputs_stay_finite(gpu, act, tile):
    """Products of zeros onto a residual of the largest floats, into 8-bit rows."""
    t, lib = torch(), _lib.load()
    M, cols, K = 300, 592, 384
    N = 2 * cols if act == "swiglu" else cols
    res = up(large(M, cols), gpu)
    x, w, out = Rows8.of(gpu, np.zeros((M, K))), Rows8.of(gpu, np.zeros((N, K))), Rows8(gpu, M, cols)
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, p(res), _lib.F32, p(out.codes), p(out.scales),
                              _lib.E4M3, 4 if act == "swiglu" else 0, M, N, K, tile, stream()))
    np.testing.assert_array_equal(R.decode(*out.host(), cols), expected(f64(res)))


@pytest.mark.parametrize("tile", [-1, 0, 3, 4, 6, 11, 12, 14])
def test_products_of_the_largest_values(gpu, tile):
    """The largest value is a product's factor like any other; a code of 2^128, which no writer makes, is an infinity."""
    t, lib = torch(), _lib.load()
    M, N, K = 40, 64, 384
    x, w = Rows8.of(gpu, np.zeros((M, K))), Rows8.of(gpu, np.zeros((N, K)))
    x.scales[:-1, 5], w.scales[:-1, 5] = 247, 127
    w.codes[:-1, 170] = 0x30  # 0.5
    x.codes[:20, 170], x.codes[20:M, 170] = 0x77, 0x78
    x.codes[10:20, 170] |= 0x80
    out = t.empty(M, N, device=gpu)
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, None, 0, p(out), None, _lib.F32, 0, M, N, K,
                              tile, stream()))
    got = f64(out)
    assert (got[:10] == TOP / 2).all() and (got[10:20] == -TOP / 2).all() and (got[20:] == np.inf).all()
