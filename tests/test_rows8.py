"""8-bit rows without a GPU: the reference against torch's float8 cast, widths, and what the entry points refuse."""
import ctypes as ct

import numpy as np
import pytest

import rows8_reference as R
from laya_cuda import _lib


def test_reference_rounds_as_the_float8_cast_does():
    import torch
    rng = np.random.default_rng(1)
    grid = R.code_values()[:127]
    middles = (grid[1:] + grid[:-1]) / 2  # the ties
    x = np.concatenate([grid, middles, np.nextafter(middles, 0), np.nextafter(middles, 500), rng.normal(0, 100, 5000).clip(-448, 448),
                        rng.normal(0, .01, 5000)])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(R._round_e4m3(x.astype(np.float64)), want)


def test_reference_round_trip_keeps_every_code():
    codes = np.tile(np.delete(np.arange(256), [0x7f, 0xff, 0x80]).astype(np.uint8), 4)[:992].reshape(31, 32)
    codes[:, 0] = 0x7e  # 448 in every block, so the scale is the block's own
    x = R.decode(codes.reshape(1, -1), np.full((1, 31), 130, np.uint8), 992)
    back, scales = R.encode(x)
    np.testing.assert_array_equal(back[:, :992].reshape(31, 32), codes)
    assert (scales[0, :31] == 130).all() and (scales[0, 31:] == 0).all()


@pytest.mark.parametrize("top,byte", [(448, 127), (448.1, 128), (896, 128), (1, 119), (1.75, 119), (1.7500001, 120), (0, 0),
                                      (3.4e38, 247), (1e-45, 0), (np.inf, 255), (np.nan, 255)])
def test_reference_scales(top, byte):
    _, scales = R.encode(np.array([[top] + [0.0] * 31], np.float32))
    assert scales[0, 0] == byte


def test_width8():
    lib = _lib.load()
    assert [lib.laya_width8(w) for w in (1, 127, 128, 129, 1000, 1 << 30)] == [128, 128, 128, 256, 1024, 1 << 30]
    assert [lib.laya_width8(w) for w in (0, -5, (1 << 30) + 1)] == [-1, -1, -1]


# Addresses that the refusals below never follow: every call fails its checks, or has no rows.
P, ODD = 0x10000, 0x10001


def refused(call, *args, match):
    lib = _lib.load()
    assert getattr(lib, call)(*args) == _lib.EINVAL
    assert match in _lib.error(None), _lib.error(None)


def test_quantize_refusals():
    ok = dict(x=P, dtype=_lib.F32, stride=100, codes=P, scales=P, rows=3, width=100, stream=None)

    def call(match, **change):
        refused("laya_op_quantize8", *{**ok, **change}.values(), match=match)

    call("dtype", dtype=_lib.E4M3)
    call("dtype", dtype=-1)
    for bad in (dict(rows=-1), dict(width=0), dict(width=(1 << 30) + 1, stride=1 << 40), dict(stride=99), dict(stride=-100)):
        call("rows, width or stride", **bad)
    call("x must", x=None)
    call("x must", x=P + 2)
    call("x must", x=ODD, dtype=_lib.BF16)
    call("required", codes=None)
    call("required", scales=None)
    call("aligned", codes=P + 8)
    call("aligned", scales=P + 2)
    assert _lib.load().laya_op_quantize8(None, _lib.F32, 100, None, None, 0, 100, None) == _lib.OK


def test_dequantize_refusals():
    ok = dict(codes=P, scales=P, out=P, dtype=_lib.F32, stride=100, rows=3, width=100, stream=None)

    def call(match, **change):
        refused("laya_op_dequantize8", *{**ok, **change}.values(), match=match)

    call("dtype", dtype=_lib.E4M3)
    for bad in (dict(rows=-1), dict(width=0), dict(stride=99)):
        call("rows, width or stride", **bad)
    call("out must", out=None)
    call("out must", out=ODD, dtype=_lib.F16)
    call("required", codes=None)
    call("aligned", codes=P + 4)
    assert _lib.load().laya_op_dequantize8(None, None, None, _lib.F32, 100, 0, 100, None) == _lib.OK


def test_norm_refusals():
    ok = dict(residual=P, branch=P, branch_dtype=_lib.F32, splits=2, part_stride=300, bias=P, gamma=P, beta=P, eps=1e-5,
              kind=_lib.RMS_NORM, sum_out=P, out32=None, codes=P, scales=P, rows=3, width=100, stream=None)

    def call(match, **change):
        refused("laya_op_norm8", *{**ok, **change}.values(), match=match)

    call("kind", kind=2)
    for bad in (dict(rows=-1), dict(width=0), dict(width=8193, part_stride=1 << 30)):
        call("width 1 to 8192", **bad)
    call("eps", eps=-1.0)
    call("eps", eps=float("nan"))
    call("branch_dtype", branch_dtype=_lib.E4M3)
    call("partial", splits=0)
    call("partial", part_stride=299)
    call("bias needs", branch=None)
    call("residual and gamma", residual=None)
    call("residual and gamma", gamma=None)
    call("aligned to their", beta=P + 2)
    call("aligned to their", branch=ODD, branch_dtype=_lib.F16, splits=1)
    call("different arrays", out32=P)
    call("required", codes=None)
    assert _lib.load().laya_op_norm8(*{**ok, "rows": 0, "codes": None}.values()) == _lib.OK


def test_linear_refusals():
    ok = dict(x=P, xs=P, w=P, ws=P, bias=P, residual=P, residual_dtype=_lib.F32, out=P, out_scales=None, out_dtype=_lib.F32,
              act=_lib.ACT_NONE, M=3, N=64, K=100, tile=-1, stream=None)

    def call(match, **change):
        refused("laya_op_linear8", *{**ok, **change}.values(), match=match)

    call("activation", act=5)
    call("activation", act=-1)
    call("out_dtype", out_dtype=4)
    call("residual_dtype", residual_dtype=_lib.E4M3)
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(K=(1 << 20) + 1), dict(N=(1 << 20) + 1)):
        call("N and K", **bad)
    call("groups of 32", act=_lib.ACT_GEGLU, N=48)
    call("x: codes", x=None)
    call("x: codes", xs=P + 1)
    call("w: codes", ws=None)
    call("w: codes", w=P + 8)
    call("out_scales", out=None)
    call("out_scales", out_scales=P)
    call("out_scales", out_dtype=_lib.E4M3)
    call("output: codes", out_dtype=_lib.E4M3, out=P + 4, out_scales=P)
    call("aligned to their", out=P + 2)
    call("aligned to their", bias=ODD)
    call("aligned to their", residual=P + 2)
    assert _lib.load().laya_op_linear8(*{**ok, "M": 0, "x": None, "out": None}.values()) == _lib.OK


def test_nothing_is_wrapped_in_ctypes_structures():
    """The new operators add no structure: the binding's ABI version stays."""
    assert _lib.load().laya_abi_version() == _lib.ABI_VERSION == 2
    assert _lib.SIGNATURES["laya_op_linear8"][1] is ct.c_int


def test_extents_past_a_launch_are_refused():
    """Codes and spans that no launch covers, and offsets that would not fit 64 bits."""
    refused("laya_op_quantize8", P, _lib.F32, 1, P, P, 1 << 29, 1, None, match="2^36 codes")
    refused("laya_op_quantize8", P, _lib.F32, 1 << 62, P, P, 2, 100, None, match="2^50 elements")
    refused("laya_op_quantize8", P, _lib.F32, 100, P, P, (1 << 63) - 1, 100, None, match="2^36 codes")
    refused("laya_op_dequantize8", P, P, P, _lib.F32, 1 << 62, 2, 100, None, match="2^50 elements")
    refused("laya_op_dequantize8", P, P, P, _lib.F32, 1 << 20, 1 << 17, 1 << 20, None, match="2^36 codes")
    norm = dict(residual=P, branch=None, branch_dtype=0, splits=1, part_stride=0, bias=None, gamma=P, beta=None, eps=1e-5,
                kind=_lib.RMS_NORM, sum_out=None, out32=None, codes=P, scales=P, rows=1 << 26, width=4, stream=None)
    refused("laya_op_norm8", *norm.values(), match="fewer than 2^26")
    refused("laya_op_norm8", *{**norm, "rows": 1 << 24, "width": 2052}.values(), match="fewer than 2^26")
