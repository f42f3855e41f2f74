"""laya_op_rotary on the GPU against 64 bits.

Tolerance: an angle is exact to 2^-27 of a turn (5e-8 radians), sine, cosine and amplitude add four roundings of fp32, the two
products and their sum three more: (5e-8 + 7 u) (|a| + |b|) amplitude with u = 2^-24, then half a step of the type.
"""
import ctypes as ct

import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
CODE = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}


def setup(gpu, kind, rows, heads, dim, rotated, far, row=None, head=None, offset=0, seed=0):
    """x in its strides with NaNs around it, positions and frequencies on both sides."""
    import torch as t
    dtype = {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[kind]
    rng = np.random.default_rng(seed)
    head = head or dim
    row = row or heads * head
    held = t.full((offset + rows * max(row, heads * head) + 64,), float("nan"), dtype=dtype, device=gpu)
    x = held[offset:].as_strided((rows, heads, dim), (row, head, 1))
    x.copy_(t.from_numpy(rng.normal(0, 2, (rows, heads, dim))).to(gpu))
    positions = rng.integers(-far, far, rows).astype(np.int32)
    positions[0] = far - 1
    turns = 10000.0 ** (-np.arange(0, rotated, 2) / rotated) / (2 * np.pi)
    return held, x, positions, turns


def run(lib, x, out, kind, positions, turns, rotated, amplitude=1.0, layout=0, direction=1):
    import torch as t
    rows, heads, dim = x.shape
    at = lambda v: ct.c_void_p(v.data_ptr())  # noqa: E731
    p, f = t.from_numpy(positions).to(x.device), t.from_numpy(np.asarray(turns)).to(x.device)
    _lib.check(lib.laya_op_rotary(at(x), x.stride(0), x.stride(1), at(out), out.stride(0), out.stride(1), CODE[kind], at(p), at(f),
                                  amplitude, layout, direction, rows, heads, dim, rotated,
                                  ct.c_void_p(t.cuda.current_stream().cuda_stream)))
    t.cuda.synchronize()


def compare(got, x64, positions, turns, kind, amplitude, layout, direction):
    want = A.rotate(x64, positions, turns, amplitude, layout == 1, direction)
    r = 2 * len(turns)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout else (slice(0, r // 2), slice(r // 2, r))
    size = np.zeros_like(want)
    size[..., a] = size[..., b] = (np.abs(x64[..., a]) + np.abs(x64[..., b])) * abs(amplitude)
    bound = (5e-8 + 7 * 2.0 ** -24) * size + HALF[kind] * np.abs(want) + 2.0 ** -25
    bound[..., r:] = 0
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / np.maximum(bound, 1e-30))


CASES = [  # rows, heads, dim, rotated, far, row, head, offset
    (1, 1, 2, 2, 10, None, None, 0),
    (1, 24, 64, 64, 1024, None, None, 0),
    (3, 5, 80, 32, 1 << 20, None, None, 0),
    (257, 12, 64, 64, 8192, 3 * 12 * 64, None, 0),     # within a projection's rows
    (33, 7, 128, 96, 2 ** 31 - 1, None, 136, 0),       # the farthest positions, gaps between heads
    (19, 3, 64, 34, 1000, None, None, 0),              # halves off whole 16 bytes
    (19, 3, 66, 64, 1000, None, None, 0),              # heads off whole 16 bytes
    (19, 3, 64, 64, 1000, 201, 67, 1),                 # odd strides, an odd address
    (1000, 2, 256, 250, 100, None, None, 0),
    (5, 1, 8192, 8192, 100, None, None, 0),
    (2, 300, 96, 96, 70000, None, None, 0),            # more units a row than a workgroup takes at once
    (2000, 40, 64, 64, 70000, None, None, 0),
    (300, 17, 72, 72, 1000, None, None, 0),            # halves of 36: a narrower unit for each power of two that divides
    (300, 12, 100, 100, 1000, None, None, 0),          # of 50
    (300, 13, 98, 98, 1000, None, None, 0),            # of 49
    (300, 16, 80, 20, 1000, None, None, 2),            # of 10, at an address off 8 bytes
    (3, 4, 200, 104, 1000, 812, 204, 4),               # strides of whole 4 values only
    (3, 128, 8192, 8192, 1000, None, None, 1),         # a row of 2^20 values, one by one
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,rotated,far,row,head,offset", CASES)
def test_rotary(gpu, kind, layout, rows, heads, dim, rotated, far, row, head, offset):
    lib = _lib.load()
    held, x, positions, turns = setup(gpu, kind, rows, heads, dim, rotated, far, row, head, offset)
    import torch as t
    x64 = x.double().cpu().numpy()
    for direction, amplitude in ((1, 1.0), (-1, 1.25)):
        out = t.full_like(x, 7.0, memory_format=t.contiguous_format)
        run(lib, x, out, kind, positions, turns, rotated, amplitude, layout, direction)
        compare(out.double().cpu().numpy(), x64, positions, turns, kind, amplitude, layout, direction)
    before = held.clone()
    run(lib, x, x, kind, positions, turns, rotated, 1.0, layout, 1)  # in place
    compare(x.double().cpu().numpy(), x64, positions, turns, kind, 1.0, layout, 1)
    x.copy_(before[offset:].as_strided(x.shape, x.stride()))
    same = (held == before) | (held.isnan() & before.isnan())
    assert same.all()  # nothing between rows and heads was written


@pytest.mark.parametrize("layout", [0, 1])
def test_turning_back_is_the_gradient(gpu, layout):
    """<R x, y> = <x, R^T y>, and the derivative of <R x, y> along e is its difference quotient, R being linear: each side an
    fp32 rotation, off by at most (5e-8 + 8 u) of the summed magnitudes (test_rotary's bound and the fp32 output)."""
    import torch as t
    lib = _lib.load()
    _, x, positions, turns = setup(gpu, "f32", 100, 3, 48, 40, 5000, seed=1)
    _, y, *_ = setup(gpu, "f32", 100, 3, 48, 40, 5000, seed=2)
    rx, ry, r2 = t.empty_like(x), t.empty_like(x), t.empty_like(x)
    run(lib, x, rx, "f32", positions, turns, 40, 1.5, layout, 1)
    run(lib, y, ry, "f32", positions, turns, 40, 1.5, layout, -1)
    left, right = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    size = 1.5 * 4 * (x.double().abs().sum() * y.double().abs().max())
    assert abs(left - right) <= (5e-8 + 8 * 2.0 ** -24) * size
    e = t.zeros_like(x)
    e[17, 1, 5] = 1.0  # a step of 1: the function is linear, so the quotient is the derivative
    run(lib, x + e, r2, "f32", positions, turns, 40, 1.5, layout, 1)
    quotient = ((r2.double() - rx.double()) * y.double()).sum()
    near = 4 * (5e-8 + 8 * 2.0 ** -24) * 1.5 * (x[17, 1].abs().max().double() + 1) * y[17, 1].abs().max().double() * 4
    assert abs(quotient - ry[17, 1, 5].double()) <= near


def test_rows_on_another_stream_and_in_a_graph(gpu):
    import torch as t
    lib = _lib.load()
    _, x, positions, turns = setup(gpu, "bf16", 300, 8, 64, 64, 9000)
    p, f = t.from_numpy(positions).to(gpu), t.from_numpy(turns).to(gpu)
    out = t.zeros_like(x, memory_format=t.contiguous_format)

    def call(stream):
        at = lambda v: ct.c_void_p(v.data_ptr())  # noqa: E731
        _lib.check(lib.laya_op_rotary(at(x), x.stride(0), x.stride(1), at(out), out.stride(0), out.stride(1), _lib.BF16, at(p), at(f), 1.0, 0,
                                      1, 300, 8, 64, 64, ct.c_void_p(stream.cuda_stream)))

    t.cuda.synchronize()
    side = t.cuda.Stream()
    call(side)
    side.synchronize()
    eager = out.clone()
    compare(eager.double().cpu().numpy(), x.double().cpu().numpy(), positions, turns, "bf16", 1.0, 0, 1)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        call(t.cuda.current_stream())
    for turn in range(3):
        x.copy_(t.randn(x.shape, device=gpu))
        p.copy_(t.randint(0, 5000, (300,), device=gpu, dtype=t.int32))
        out.zero_()
        graph.replay()
        t.cuda.synchronize()
        got = out.clone()
        call(t.cuda.current_stream())
        t.cuda.synchronize()
        assert t.equal(got, out)
