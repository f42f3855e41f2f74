"""The sums of laya_op_linear8, seen on their own: the residual is minus the 64-bit result, so an output of any type is the
sum's error, rounded relative to itself.

Planned calls and the tiles of exact products: every 32-code step adds 32 exact products to fp32 accumulators in a tree of
at most 6 levels, so a sum is within (steps + 6) 2 u of the sum of magnitudes (u = 2^-24; the matrix unit's additions may
truncate).  The 8-bit unit's tiles: a group of 8 products is cut off, towards zero, 2^13 below its largest sum of exponents.  Seven
of them lose less than 7 2^-13 < 2^-10 of the largest product, at most that share of the sum of magnitudes.  A subnormal code's
exponent is its type's least, up to 2^3 over the code's own: where one is in the largest product, 2^-7 (in both, nothing is
lost).  Then the residual's rounding and addition, and the output's own.
"""
import numpy as np
import pytest

import rows8_reference as R
from laya_cuda import _lib
from test_rows8_gpu import CODE, HALF, U, Rows8, check, dtype, f64, p, stream, torch, up

pytestmark = pytest.mark.gpu

FAST_TILES = (5, 7, 8, 9, 10, 13)


def made(gpu, kind, M, N, K):
    """Two sets of 8-bit rows with their values in 64 bits."""
    t, lib = torch(), _lib.load()
    gen = t.Generator(device=gpu).manual_seed(M + N + K)
    normal = lambda *s: t.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, w = normal(M, K), normal(N, K) * K ** -.5
    if kind != "normal":  # a channel in 128 a thousand times the others
        many = t.ones(K, device=gpu)
        many[3::128] = 1000.0
        x = x * many
    if kind == "one sign":
        x, w = x.abs(), w.abs() * K ** -.5
    if kind == "wide":
        x, w = t.exp(2 * normal(M, K)), t.exp(2 * normal(N, K)) / K

    def rows8(v):
        n, k = v.shape
        held = Rows8(gpu, n, k)
        check(lib.laya_op_quantize8(p(v), _lib.F32, k, p(held.codes), p(held.scales), n, k, stream()))
        back = t.empty(n, k, device=gpu)
        check(lib.laya_op_dequantize8(p(held.codes), p(held.scales), p(back), _lib.F32, k, n, k, stream()))
        return held, back.double()

    return rows8(x), rows8(w)


def error_of(gpu, a, b, out, tile):
    """(error of the sums, sum of magnitudes, what the residual and the output may add) of x w^T, in 64 bits."""
    t, lib = torch(), _lib.load()
    (x, xv), (w, wv) = a, b
    (M, K), N = xv.shape, wv.shape[0]
    wt = wv.t().contiguous()
    want, mag = xv @ wt, xv.abs() @ wt.abs()
    res = (-want).float()
    o = Rows8(gpu, M, N) if out == "e4m3" else t.full((M + 1, N), 9.0, dtype=dtype(out), device=gpu)
    outs = (p(o.codes), p(o.scales)) if out == "e4m3" else (p(o), None)
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, p(res), _lib.F32, *outs, CODE[out], 0,
                              M, N, K, tile, stream()))
    own = 2 * U * want.abs()
    if out == "e4m3":
        got = t.from_numpy(R.decode(*o.host(), N)).to(gpu)
        # Half a step of a code, or of the smallest one at the block's scale (the top is over 224 of them, read at 2^-4).
        top = t.nn.functional.pad(got.abs(), (0, -N % 32)).view(M, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :N]
        own = own + 2.0 ** -4 * got.abs() + 2.0 ** -10 * top / 208
    else:
        assert (o[M:] == 9).all()
        got = o[:M].double()
        own = own + 2 * HALF[out] * got.abs() + (2.0 ** -25 if out == "f16" else 0)
    return (got - (want + res.double())).abs(), mag, own


def exact_bound(K):
    return (R.width8(K) // 32 + 6) * 2 * U


# Few rows, one round of tiles, odd sizes, and more 256 x 256 tiles than compute units.
SIZES = [(1, 256, 1024), (7, 67, 129), (96, 2304, 768), (300, 640, 512), (512, 1024, 384), (1571, 1088, 256), (5000, 1024, 1024),
         (4333, 4416, 384)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
def test_planned_sums_are_held_in_32_bits(gpu, out, M, N, K):
    """Outputs of every type, large channels and sums of one sign among them, at row counts that take different tiles."""
    for kind in ("normal", "channels", "one sign", "wide"):
        off, mag, own = error_of(gpu, *made(gpu, kind, M, N, K), out, -1)
        worst = ((off - own) / mag).max().item()
        assert worst <= exact_bound(K), f"{kind}: {worst:.3g} of the sum of magnitudes, {exact_bound(K):.3g} allowed"


@pytest.mark.parametrize("M,N,K", [(96, 256, 128), (300, 640, 512), (150, 1056, 4096), (260, 256, 65536), (4333, 4416, 384)])
@pytest.mark.parametrize("out", ["f16", "bf16", "e4m3"])
def test_the_8_bit_unit_s_bound(gpu, out, M, N, K):
    """Calls that ask for the 8-bit unit, and each of its tiles by name, with the largest products normal ones: within 2^-10 of the
    sum of magnitudes."""
    for kind in ("normal", "channels", "one sign", "wide"):
        a, b = made(gpu, kind, M, N, K)
        for tile in (_lib.TILE_FAST, *FAST_TILES):
            if M * N * K > 1 << 31 and tile in FAST_TILES[:-1]:
                continue  # the planner's and the ring
            try:
                off, mag, own = error_of(gpu, a, b, out, tile)
            except RuntimeError as e:
                assert "no such tile" in str(e) and tile == 13 and K <= 128  # the ring takes two slabs at least
                continue
            worst = ((off - own) / mag).max().item()
            assert worst <= 2.0 ** -10 + exact_bound(K), f"{kind}, tile {tile}: {worst:.3g}"


@pytest.mark.parametrize("tile,share", [(_lib.TILE_EXACT, 0.0), (_lib.TILE_FAST, 2.0 ** -7), (5, 2.0 ** -7), (9, 2.0 ** -7), (13, 2.0 ** -7)])
@pytest.mark.parametrize("subnormal", [False, True])
def test_small_products_beside_a_large_one(gpu, tile, share, subnormal):
    """A group's large product and seven that lie just below the 8-bit unit's cut, in every group of a row: exact tiles keep
    them all, the unit's lose them, and no more."""
    t, lib = torch(), _lib.load()
    M, N, K = 300, 256, 256
    x, w = (Rows8.of(gpu, np.ones((n, K))) for n in (M, N))
    # Codes by hand at scale 1: x is 2^-9 (subnormal) or 1 everywhere, w 256 once a group and 1.875 2^-3 or 2^-6 beside it.
    x.codes[:-1] = 0x01 if subnormal else 0x38
    w.codes[:-1] = 0x27 if subnormal else 0x0f
    w.codes[:-1, ::8] = 0x78
    x.scales[:-1], w.scales[:-1] = 127, 127
    xv, wv = (R.decode(*r.host(), K) for r in (x, w))
    want = xv @ wv.T
    res = up((-want).astype(np.float32), gpu)
    out = t.empty(M, N, dtype=t.bfloat16, device=gpu)
    check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), None, p(res), _lib.F32, p(out), None, _lib.BF16, 0,
                              M, N, K, tile, stream()))
    off = np.abs(f64(out) - (want + f64(res)))
    assert (off <= (share if subnormal else share / 8) * want + exact_bound(K) * want + 2 * U * want + 2 * HALF["bf16"] * off).all()


def test_fp32_outputs_ignore_the_8_bit_unit(gpu):
    """An fp32 output is exact whatever its caller allows, and refuses the unit's tiles by name."""
    a, b = made(gpu, "one sign", 300, 640, 512)
    off, mag, own = error_of(gpu, a, b, "f32", _lib.TILE_FAST)
    assert (off <= own + exact_bound(512) * mag).all()
    for tile in FAST_TILES:
        with pytest.raises(RuntimeError, match="no such tile"):
            error_of(gpu, a, b, "f32", tile)


@pytest.mark.parametrize("out,act,rtype", [("f16", "none", ""), ("bf16", "gelu", "bf16"), ("bf16", "swiglu", "f32"), ("e4m3", "relu", "f16"),
                                           ("e4m3", "geglu", ""), ("f16", "swiglu", "")])
@pytest.mark.parametrize("M,N,K", [(4200, 4352, 256), (4333, 4416, 384), (65, 66048, 640)])
def test_both_rings_over_more_tiles_than_compute_units(gpu, M, N, K, out, act, rtype):
    rings(gpu, M, N, K, out, act, rtype)


@pytest.mark.parametrize("out,act,rtype,rest", [
    ("f32", "none", "", 4), ("f32", "gelu", "f32", 8), ("f32", "none", "bf16", 12), ("f32", "relu", "f16", 4), ("bf16", "none", "", 8),
    ("f16", "gelu", "f32", 8), ("bf16", "relu", "bf16", 8), ("e4m3", "none", "", 1), ("e4m3", "gelu", "", 7), ("e4m3", "relu", "", 14),
    ("e4m3", "none", "f32", 4), ("e4m3", "gelu", "bf16", 12), ("e4m3", "relu", "f16", 8)])
@pytest.mark.parametrize("M,N,K", [(4333, 4400, 384), (300, 512, 256), (70, 66048, 640)])
def test_rings_of_columns_that_end_inside_a_block(gpu, M, N, K, out, act, rtype, rest):
    """Columns past a multiple of 16: the persistent kernels take every number whose stores and residual quads are whole."""
    rings(gpu, M, N + rest, K, out, act, rtype)


@pytest.mark.parametrize("out,rtype,N", [("f32", "", 1001), ("f32", "", 1002), ("bf16", "", 1004), ("f16", "", 1003), ("e4m3", "f32", 1002),
                                         ("e4m3", "bf16", 1001)])
def test_rings_refuse_columns_that_end_inside_a_store(gpu, out, rtype, N):
    """Such calls take the other tiles, by the planner's choice, and get the same sums."""
    rings(gpu, 700, N, 256, out, "none", rtype, refused=True)


def rings(gpu, M, N, K, out, act, rtype, refused=False):
    """Every output of both persistent kernels beside the exact tile of 128 x 128."""
    t, lib = torch(), _lib.load()
    (x, xv), (w, wv) = made(gpu, "normal", M, N, K)
    gen = t.Generator(device=gpu).manual_seed(5)
    cols = N // 2 if act in ("geglu", "swiglu") else N
    bias = t.randn(N, device=gpu, generator=gen) * .5
    res = t.randn(M, cols, device=gpu, generator=gen).to(dtype(rtype)) if rtype else None

    def run(tile):
        o = Rows8(gpu, M, cols) if out == "e4m3" else t.full((M + 1, cols), 9.0, dtype=dtype(out), device=gpu)
        outs = (p(o.codes), p(o.scales)) if out == "e4m3" else (p(o), None)
        check(lib.laya_op_linear8(p(x.codes), p(x.scales), p(w.codes), p(w.scales), p(bias), p(res), CODE[rtype or "f32"], *outs,
                                  CODE[out], ["none", "gelu", "relu", "geglu", "swiglu"].index(act), M, N, K, tile, stream()))
        if out != "e4m3":
            assert (o[M:] == 9).all()
            return o[:M].double()
        assert (o.codes[-1] == 0x5a).all() and (o.scales[-1] == 0x5a).all()
        back = t.empty(M, cols, device=gpu)
        check(lib.laya_op_dequantize8(p(o.codes), p(o.scales), p(back), _lib.F32, cols, M, cols, stream()))
        return back.double()

    want, mag = run(11), xv.abs() @ wv.abs().t().contiguous() + bias.abs()
    step = 2.0 ** -4 if out == "e4m3" else HALF[out]
    for tile, share in ((14, 2 * exact_bound(K)), (13, 2.0 ** -10 + 2 * exact_bound(K))):
        if refused or (tile == 13 and out == "f32"):
            with pytest.raises(RuntimeError, match="no such tile"):
                run(tile)
            tile, share = -1, 2 * exact_bound(K)
        got = run(tile)
        if act in ("geglu", "swiglu"):  # |act'| <= 1.13 and |act(g)| <= |g|
            m = mag.view(M, -1, 2, 16)
            e = share * m
            tol = (1.13 * e[:, :, 0] * m[:, :, 1] + e[:, :, 1] * m[:, :, 0] + 2e-6 * m[:, :, 1]).reshape(M, -1)
        else:
            tol = 1.13 * share * mag + (2e-6 if act == "gelu" else 0)
        tol = tol + 2 * U * (want.abs() + 8) + 2 * step * want.abs()  # a step apart where the sums lie about a rounding's border
        if out == "e4m3":
            tol = tol + 2.0 ** -9 * t.nn.functional.pad(want.abs(), (0, -cols % 32)).view(M, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :cols] / 200
        assert ((got - want).abs() <= tol).all(), f"tile {tile}: {((got - want).abs() - tol).max().item():.3g} beyond"
        if tile == 14:  # the same exact sums in the same order of steps: few of them round apart
            assert (got != want).double().mean().item() < .01
