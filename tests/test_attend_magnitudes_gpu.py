"""laya_op_attend where scores are as large as biases and scales allow: what counts is their difference, whatever their size.

Scores of one size are made equal to the last bit (zero queries, or products of small whole numbers), so that a softmax over n of
them is 1 / n each.  Equal scores get equal weights, whose roundings to 16 bits cancel in the normaliser; what is left are the sums
in fp32, 2 u a key (u = 2^-24) of sum w |v|, the division's and the sum's last roundings (2 u), and half a step of the output.
With a cap, a step past a table's span has its exponents off by two more roundings of the cap, so that its weights may round to the
other neighbour: a step of the type, 2 h, of sum w |v|.
"""
import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib
from test_attend_gpu import KERNELS, ODD, Call, torch

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128), ("bf16", 256)])


def compare(c, table=None):
    """Against 64 bits, with the bound above.  table: in the place of the call's."""
    torch().cuda.synchronize()
    q, kv, got = (x.double().cpu().numpy()[..., :c.dim] for x in (c.q, c.kv, c.out))
    for s in range(len(c.nq)):
        rows, keys = slice(c.q0[s], c.q0[s] + c.nq[s]), slice(c.k0[s], c.k0[s] + c.nk[s])
        given = (c.scale, c.cap, c.slopes, c.table if table is None else table, c.before, c.after)
        want, _ = A.attend(q[rows], kv[keys, :c.kv_heads], kv[keys, c.kv_heads:], *given, kind=c.kind)
        size, _ = A.attend(q[rows], kv[keys, :c.kv_heads], np.abs(kv[keys, c.kv_heads:]), *given, kind=c.kind)
        bound = (2 * A.U * (c.nk[s] + 1) + (2 * A.HALF[c.kind] if c.cap else 0)) * size + A.HALF[c.kind] * np.abs(want) + 2.0 ** -25
        off = np.abs(got[rows] - want)
        assert (off <= bound).all(), (s, off.max(initial=0), np.argwhere(~(off <= bound))[:3])


@KINDS
@pytest.mark.parametrize("bias", [1e3, -1e6, 1.7e7, -1e9, 1.1e9, -7.3e9, -1e12, 3e20, -5e29])
@pytest.mark.parametrize("cap", [0.0, 9.0])
@pytest.mark.parametrize("masks", [dict(), dict(after=0), dict(before=9, after=40)], ids=["all", "causal", "window"])
@KERNELS
def test_one_bias_for_every_key_is_none(gpu, kind, dim, bias, cap, masks, kernel):
    """Keys within the table's span and past it, a whole step and single ones."""
    c = Call(gpu, kind, ODD + [300], 4, 2, dim, cap=cap, bias="table", span=20, **masks)
    c.q[..., :dim] = 0
    c.table[:] = bias
    c.describe(kernel=kernel).run()
    compare(c, np.zeros_like(c.table))


@KINDS
@pytest.mark.parametrize("bias", [-1e4, -1e9, -3.4e38])
@KERNELS
def test_masks_by_bias_beside_keys_that_are_seen(gpu, kind, dim, bias, kernel):
    """The usual lowest values as masks: keys behind the query, and far before it, weigh nothing beside those that are left."""
    c = Call(gpu, kind, ODD + [300], 4, 2, dim, bias="table", span=20)
    hidden = np.r_[:9, 21:41]  # distances below -11, and above 0
    c.table[:, hidden] = bias
    c.describe(kernel=kernel).run()
    c.table[:, hidden] = -np.inf
    c.check()


@KINDS
@pytest.mark.parametrize("scale", [1.0, 1e4, 1e7, 1e10])
@pytest.mark.parametrize("cap", [0.0, 1024.0])
@KERNELS
def test_scales_that_leave_the_largest_scores(gpu, kind, dim, scale, cap, kernel):
    """Scores are whole multiples of the scale, and those that tie share the weight; with a cap all positive ones tie, but for
    scale 1, which is left out."""
    if cap and scale == 1.0:
        scale = 3e6
    c = Call(gpu, kind, ODD, 4, 2, dim, scale=scale, cap=cap)
    c.q[..., :dim] = (c.q[..., :dim] * 0.3).round()
    c.kv[:, :c.kv_heads, :dim] = (c.kv[:, :c.kv_heads, :dim] * 0.4).round()
    if scale == 1.0:  # neighbouring scores 32 apart: a weight of e^-32 beside the largest one's 1
        c.q[..., :dim] *= 32
    c.describe(kernel=kernel).run()
    compare(c)


@KINDS
@pytest.mark.parametrize("slope", [1e3, 1e6, 1e9, 1e20, 1e30])
@KERNELS
def test_steep_slopes_leave_the_nearest_key(gpu, kind, dim, slope, kernel):
    c = Call(gpu, kind, ODD + [300], 4, 2, dim, bias="slopes", before=200, after=70)
    c.slopes[:] = slope
    c.describe(kernel=kernel).run()
    torch().cuda.synchronize()
    for s in range(len(c.nq)):
        got = c.out[c.q0[s]:c.q0[s] + c.nq[s], :, :dim]
        want = c.kv[c.k0[s]:c.k0[s] + c.nk[s], 2:, :dim].repeat_interleave(2, 1)
        assert torch().equal(got, want)


@KINDS
@KERNELS
def test_scores_below_1e30_hide_and_others_do_not(gpu, kind, dim, kernel):
    for bias, hides in ((-0.99e30, False), (-1.01e30, True)):
        c = Call(gpu, kind, ODD, 4, 2, dim, bias="table", span=20)
        c.q[..., :dim] = 0
        c.table[:] = bias
        c.describe(kernel=kernel).run()
        compare(c, np.full_like(c.table, -np.inf) if hides else np.zeros_like(c.table))


@KINDS
@pytest.mark.parametrize("slope", [4e37, 3.4e38])
@pytest.mark.parametrize("scale,cap", [(None, 0.0), (1e-6, 0.0), (None, 30.0)])
@KERNELS
def test_slopes_of_the_largest_values(gpu, kind, dim, slope, scale, cap, kernel):
    """Slopes past the type's range in units of a raw score: 0 at the query's own key, and every other key hidden."""
    c = Call(gpu, kind, ODD + [300], 4, 2, dim, bias="slopes", before=200, after=70, scale=scale, cap=cap)
    c.slopes[:] = slope
    c.describe(kernel=kernel).run()
    torch().cuda.synchronize()
    for s in range(len(c.nq)):
        got = c.out[c.q0[s]:c.q0[s] + c.nq[s], :, :dim]
        assert torch().equal(got, c.kv[c.k0[s]:c.k0[s] + c.nk[s], 2:, :dim].repeat_interleave(2, 1))


@KINDS
@pytest.mark.parametrize("bias", [-1e6, -1e9, -7.3e9, -1e12])
@pytest.mark.parametrize("cap", [0.0, 9.0])
def test_biases_of_long_keys_shared_by_workgroups(gpu, kind, dim, bias, cap):
    """A mask by bias over all but the nearest keys, and one bias for every key, of contexts that several workgroups share."""
    for everywhere in (False, True):
        c = Call(gpu, kind, [1, 3, 40], 4, 2, dim, key_lengths=[9001, 4500, 70], bias="table", span=20, after=0, cap=cap)
        if everywhere:
            c.q[..., :dim] = 0
            c.table[:] = bias
        else:
            c.table[:, :9] = bias
        c.describe(kernel=_lib.ATTEND_FEW).run()
        assert c.workspace is not None
        if everywhere:
            compare(c, np.zeros_like(c.table))
        else:
            c.table[:, :9] = -np.inf
            c.check()


@KINDS
@pytest.mark.parametrize("slope", [40.0, 1e3, 3.3e6, 1e9, 1.7e12, 1e30])
@pytest.mark.parametrize("ahead", [1, 17, 31, 100])
@KERNELS
def test_steep_slopes_at_any_place_of_a_step(gpu, kind, dim, slope, ahead, kernel):
    """Queries behind a cache: their own keys lie anywhere in a step of 32.  The next key weighs e^-40 or less."""
    lengths = [1, 33, 130, 64]
    c = Call(gpu, kind, lengths, 4, 2, dim, key_lengths=[n + ahead for n in lengths], bias="slopes", after=0)
    c.slopes[:] = slope
    c.describe(kernel=kernel).run()
    torch().cuda.synchronize()
    for s, n in enumerate(lengths):
        got = c.out[c.q0[s]:c.q0[s] + n, :, :dim].double()
        want = c.kv[c.k0[s] + ahead:c.k0[s] + ahead + n, 2:, :dim].repeat_interleave(2, 1).double()
        # A score is at most 30 here: e^-10 of a value of at most 6, a hundred of them, where the slope is 40; else nothing.
        assert ((got - want).abs() <= (0.03 if slope == 40.0 else 0.0)).all()
