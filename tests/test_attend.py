"""Rotary frequencies, workspaces and refusals of the rotary and attention entry points, without a GPU."""
import ctypes as ct
import math

import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib

P, ODD = 0x10000, 0x10001  # addresses that no refused call follows


def frequencies(kind, theta, rotated, factor=1.0, original=0.0, low=0.0, high=0.0):
    out = (ct.c_double * (rotated // 2))()
    _lib.check(_lib.load().laya_rotary_frequencies(kind, theta, rotated, factor, original, low, high, out))
    return np.array(out) * 2 * math.pi


def plain(theta, rotated):
    return theta ** (-np.arange(0, rotated, 2) / rotated)


@pytest.mark.parametrize("theta,rotated", [(10000.0, 64), (160000.0, 32), (500000.0, 128), (10000.0, 2), (3.0, 250)])
def test_frequencies(theta, rotated):
    # pow and a division or two: a few units of 2^-53
    np.testing.assert_allclose(frequencies(_lib.FREQ_PLAIN, theta, rotated), plain(theta, rotated), rtol=1e-14)
    np.testing.assert_allclose(frequencies(_lib.FREQ_LINEAR, theta, rotated, 8.0), plain(theta, rotated) / 8, rtol=1e-14)


def test_base_scaling_slows_the_slowest_pair_by_the_factor():
    got, was = frequencies(_lib.FREQ_BASE, 10000.0, 64, 4.0), plain(10000.0, 64)
    assert got[0] == was[0]
    np.testing.assert_allclose(got[-1], was[-1] / 4, rtol=1e-13)
    assert (np.diff(got / was) < 0).all()
    np.testing.assert_allclose(frequencies(_lib.FREQ_BASE, 10000.0, 2, 4.0), [1.0], rtol=1e-14)


def test_scaling_by_parts():
    got, was = frequencies(_lib.FREQ_PARTS, 10000.0, 128, 8.0, 8192.0, 1.0, 32.0), plain(10000.0, 128)
    turns = 8192 * was / (2 * math.pi)
    np.testing.assert_allclose(got[turns >= 32], was[turns >= 32], rtol=1e-14)
    np.testing.assert_allclose(got[turns <= 1], was[turns <= 1] / 8, rtol=1e-14)
    kept = (turns - 1) / 31
    between = (turns > 1) & (turns < 32)
    assert between.any()
    np.testing.assert_allclose(got[between], (was * kept + was / 8 * (1 - kept))[between], rtol=1e-13)


def refused(call, *args, match):
    lib = _lib.load()
    assert getattr(lib, call)(*args) == _lib.EINVAL
    assert match in _lib.error(None), _lib.error(None)


def test_frequency_refusals():
    out = (ct.c_double * 4)()
    ok = dict(kind=_lib.FREQ_PARTS, theta=10000.0, rotated=8, factor=2.0, original=100.0, low=1.0, high=4.0, out=out)

    def call(match, **change):
        refused("laya_rotary_frequencies", *{**ok, **change}.values(), match=match)

    call("kind", kind=4)
    call("kind", kind=-1)
    for bad in (0, 1, 7, -2, 8194):
        call("rotated", rotated=bad)
    for bad in (0.0, -1.0, math.nan, math.inf):
        call("theta", theta=bad)
    for bad in (0.5, math.nan, math.inf):
        call("factor", factor=bad)
    for bad in (dict(original=0.0), dict(low=4.0), dict(low=-1.0), dict(high=math.nan)):
        call("original", **bad)
    call("host_turns", out=None)


def test_rotary_refusals():
    ok = dict(x=P, x_row=256, x_head=64, out=P + 0x8000, out_row=256, out_head=64, dtype=_lib.F16, positions=P, turns=P, amplitude=1.0,
              layout=0, direction=1, rows=3, heads=4, dim=64, rotated=32, stream=None)

    def call(match, **change):
        refused("laya_op_rotary", *{**ok, **change}.values(), match=match)

    call("dtype", dtype=_lib.E4M3)
    call("layout", layout=2)
    call("direction", direction=0)
    call("amplitude", amplitude=math.inf)
    for bad in (dict(dim=1), dict(dim=8194), dict(heads=0), dict(heads=1 << 15)):
        call("dim must be", **bad)
    for bad in (0, 33, 66, -2):
        call("rotated", rotated=bad)
    for bad in (-1, (1 << 23) + 1):
        call("rows", rows=bad)
    for bad in (dict(x_row=-1), dict(x_head=1 << 40), dict(out_row=-64)):
        call("strides", **bad)
    call("2^50", x_row=1 << 39, rows=1 << 20)
    call("2^50", x_head=(1 << 40) - 64, heads=1 << 14)
    for bad in (dict(out_head=63), dict(out_row=63), dict(out_row=255), dict(out_row=64), dict(out_row=64, out_head=191)):
        call("must not overlap", **bad)
    for name in ("x", "out", "positions", "turns"):
        call("are required", **{name: None})
    call("aligned to their", x=ODD)
    call("aligned to their", out=P + 2, dtype=_lib.F32)
    call("aligned to their", turns=P + 4)
    call("aligned to their", positions=P + 2)
    call("in place", out=P, x_row=512)
    assert _lib.load().laya_op_rotary(*{**ok, "rows": 0, "x": None, "out": None}.values()) == _lib.OK


def test_bounds_refusals():
    ok = dict(documents=P, starts=P, lengths=P, n_seq=2, rows=100, max_length=50, bounds=P, stream=None)

    def call(match, **change):
        refused("laya_op_document_bounds", *{**ok, **change}.values(), match=match)

    for bad in (dict(n_seq=-1), dict(rows=-1), dict(rows=1 << 30), dict(max_length=-1), dict(max_length=1 << 30)):
        call("must not be negative", **bad)
    call("too large", n_seq=1 << 20, max_length=1 << 20)
    for name in ("documents", "starts", "lengths", "bounds"):
        call("are required", **{name: None})
    call("aligned", bounds=P + 4)
    call("aligned", documents=P + 2)
    for nothing in (dict(n_seq=0), dict(rows=0), dict(max_length=0)):
        assert _lib.load().laya_op_document_bounds(*{**ok, **nothing, "documents": None}.values()) == _lib.OK


def description(**change):
    values = dict(struct_bytes=ct.sizeof(_lib.LayaAttend), dtype=_lib.F16, q=P, k=P, v=P, out=P, q_row=256, q_head=64, k_row=128, k_head=64,
                  v_row=128, v_head=64, out_row=256, out_head=64, heads=4, kv_heads=2, dim=64, q_rows=100, k_rows=100, n_seq=2, max_q=50,
                  max_k=50, q_starts=P, q_lengths=P, k_starts=P, k_lengths=P, scale=0.125, cap=0.0, slopes=None, table=None, span=0,
                  before=-1, after=-1, kernel=0, prefix=None, bounds=None)
    return _lib.LayaAttend(**{**values, **change})


def test_attend_refusals():
    def call(match, workspace=None, size=0, **change):
        refused("laya_op_attend", ct.byref(description(**change)), workspace, size, None, match=match)

    refused("laya_op_attend", None, None, 0, None, match="struct_bytes")
    call("struct_bytes", struct_bytes=200)
    for bad in (_lib.F32, _lib.E4M3, -1):
        call("dtype", dtype=bad)
    for bad in (0, 4, 65, 264, -8):
        call("dim", dim=bad)
    for bad in (dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(heads=1 << 17, kv_heads=1 << 16), dict(kv_heads=-2)):
        call("multiple of kv_heads", **bad)
    for name in ("q_rows", "k_rows", "n_seq", "max_q", "max_k"):
        call("must not be negative", **{name: -1})
    for name in ("q_rows", "k_rows", "max_q", "max_k"):
        call("below 2^30", **{name: 1 << 30})
    for name in ("before", "after"):
        call("no limit", **{name: -2})
        call("no limit", **{name: 1 << 30})
    for bad in (-1, 3):
        call("kernel", kernel=bad)
    call("not both", slopes=P, table=P)
    call("span", table=P, span=-1)
    call("span", table=P, span=1025)
    call("too large", n_seq=1 << 23)
    call("too large", n_seq=1 << 12, max_q=1 << 20)
    call("too large", n_seq=1 << 21, heads=4, kv_heads=4, dim=96, max_q=1, kernel=_lib.ATTEND_MANY)  # 2^23 workgroups of 512 threads
    for bad in (dict(scale=-0.1), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.inf),
                dict(cap=math.nan), dict(cap=1e-11), dict(cap=1025.0)):
        call("scale must be", **bad)
    for name in ("q_row", "k_head", "v_row", "out_head"):
        call("strides", **{name: 132})
        call("strides", **{name: -64})
        call("strides", **{name: 1 << 40})
    call("rows of k and v", k_row=56)
    call("rows of k and v", v_row=1 << 23)
    call("2^50", q_row=(1 << 40) - 64, q_rows=1 << 20)
    call("2^50", k_head=(1 << 40) - 64, heads=1 << 14, kv_heads=1 << 13, n_seq=1)
    for bad in (dict(out_head=56), dict(out_row=56), dict(out_row=248), dict(out_row=64), dict(out_row=64, out_head=64 * 99)):
        call("must not overlap", **bad)
    for name in ("q", "k", "v", "out", "q_starts", "q_lengths", "k_starts", "k_lengths"):
        call("are required", **{name: None})
    for name in ("q", "k", "v", "out"):
        call("16-byte", **{name: P + 8})
    call("8-byte", bounds=P + 4)
    for name in ("q_starts", "k_lengths", "prefix", "slopes"):
        call("4-byte", **{name: P + 2})
    long = dict(max_q=1, max_k=100000)
    need = _lib.load().laya_attend_workspace(ct.byref(description(**long)))
    assert need > 0 and need % 4 == 0
    call("workspace", **long)
    call("workspace", workspace=P, size=need - 1, **long)
    call("workspace", workspace=P + 8, size=need, **long)
    for nothing in (dict(n_seq=0), dict(max_q=0), dict(q_rows=0)):
        assert _lib.load().laya_op_attend(ct.byref(description(**nothing, q=None, out=None)), None, 0, None) == _lib.OK


def test_workspaces():
    lib = _lib.load()

    def need(**change):
        return lib.laya_attend_workspace(ct.byref(description(**change)))

    assert need() == 0
    assert need(dim=7) == -1 and lib.laya_attend_workspace(None) == -1
    assert need(n_seq=64, max_q=1024, max_k=1024) == 0  # a workgroup for each 128 queries
    one = need(n_seq=1, max_q=1, max_k=1 << 17)
    assert one == 2 * 64 * 32 * (64 + 2) * 4  # two key heads, 64 splits, 32 rows
    assert need(n_seq=1, max_q=1, max_k=1 << 17, before=100, after=0) == 0  # the window leaves little to share
    assert need(n_seq=1, max_q=1, max_k=1 << 17, before=100, after=0, prefix=P) == one
    assert need(n_seq=1, max_q=1, max_k=1 << 17, kernel=_lib.ATTEND_FEW) == one
    assert need(n_seq=1, max_q=1, max_k=1 << 17, kernel=_lib.ATTEND_MANY) == 0


def test_reference_against_torch():
    import torch
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(0, 1, (20, 4, 16)), rng.normal(0, 1, (33, 2, 16)), rng.normal(0, 1, (33, 2, 16))
    out, bound = A.attend(q, k, v, 0.25, after=0, before=9, prefix=3)
    mask = torch.from_numpy(A.visible(20, 33, 9, 0, 3, None))
    want = torch.nn.functional.scaled_dot_product_attention(
        torch.from_numpy(q).transpose(0, 1), torch.from_numpy(k).transpose(0, 1).repeat_interleave(2, 0),
        torch.from_numpy(v).transpose(0, 1).repeat_interleave(2, 0), attn_mask=mask, scale=0.25).transpose(0, 1)
    np.testing.assert_allclose(out, want.numpy(), atol=1e-12)
    assert (bound > 0).all()
    assert not A.attend(q, k, v, 0.25, bounds=np.zeros((20, 2), int))[0].any()
    np.testing.assert_array_equal(A.document_bounds([5, 5, 1, 5, 5, 5]), [[0, 2], [0, 2], [2, 3], [3, 6], [3, 6], [3, 6]])


def test_the_structure_mirrors_the_header():
    """Field names and order of LayaAttend in the header and the binding."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "laya_hip.h").read_text()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct LayaAttend \{(.*?)\} LayaAttend;", text, re.S)[1], flags=re.S)
    names = [n.strip().lstrip("*").split()[-1].lstrip("*") for part in body.split(";") for n in part.split(",") if n.strip()]
    assert names == [f[0] for f in _lib.LayaAttend._fields_]
    assert ct.sizeof(_lib.LayaAttend) == 224
