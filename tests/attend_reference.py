"""Attention with masks, capped scores and distance biases, and rotary positions, in 64 bits (NumPy), with error bounds.

Bounds of laya_op_attend's outputs, in roundings (u = 2^-24, h = half a step of the 16-bit type relative to the value):
  * a score is a sum of dim exact products in fp32, in any order (2 u: additions inside the matrix unit may truncate), then
    a few roundings of itself and its bias; a cap adds 2^-20 of itself (exponential and reciprocal of 1 ulp, each twice 2 cap);
  * a weight is off by its score's error and h, and the normaliser sums the rounded weights: 2 (h + e) of sum w |v|;
  * fp16 weights below 2^-14 are off by up to 2^-25, of a total that is at least 1: keys * 2^-25 * max |v|;
  * sums of weights and values are fp32: 2 u * keys of sum w |v|;
  * then h of the output, or half the smallest fp16 step.
"""
import numpy as np

U = 2.0 ** -24
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def visible(nq, nk, before, after, prefix, bounds):
    p, j = np.arange(nk - nq, nk)[:, None], np.arange(nk)[None, :]
    see = np.ones((nq, nk), bool)
    if before >= 0:
        see &= j >= p - before
    if after >= 0:
        see &= j <= p + after
    if bounds is not None:
        see &= (j >= bounds[:, :1]) & (j < bounds[:, 1:])
    return see | (j < prefix)


def attend(q, k, v, scale, cap=0.0, slopes=None, table=None, before=-1, after=-1, prefix=0, bounds=None, kind="f16"):
    """One sequence: q [nq][heads][dim], k and v [nk][kv_heads][dim] in 64 bits; (out, bound) [nq][heads][dim]."""
    (nq, heads, dim), (nk, kv_heads, _) = q.shape, k.shape
    out, bound = np.zeros_like(q), np.zeros_like(q)
    see = visible(nq, nk, before, after, prefix, bounds)
    h = HALF[kind]
    distance = np.arange(nk)[None, :] - np.arange(nk - nq, nk)[:, None]
    for i in range(heads):
        ki, vi = k[:, i // (heads // kv_heads)], v[:, i // (heads // kv_heads)]
        with np.errstate(invalid="ignore", over="ignore"):
            t = q[:, i] @ ki.T * scale
            magnitude = np.abs(q[:, i]) @ np.abs(ki).T * scale
            if cap:
                t = cap * np.tanh(t / cap)
            bias = np.zeros_like(t)
            if slopes is not None:
                bias = -float(slopes[i]) * np.abs(distance)
            if table is not None:
                span = table.shape[1] // 2
                bias = table[i].astype(np.float64)[np.clip(distance, -span, span) + span]
            t = np.where(see, t + bias, -np.inf)
            t = np.where(t > -1e30, t, np.where(np.isnan(t), t, -np.inf))
            top = np.where(np.isneginf(t.max(1, initial=-np.inf)), 0.0, t.max(1, initial=-np.inf))[:, None]
            w = np.exp(t - top)
            total = w.sum(1, keepdims=True)
            w = w / np.where(total == 0, 1.0, total)
            # Hidden keys are not there: a product of a weight of 0 and what lies in their values is none.
            finite = np.isfinite(vi).all(1)
            out[:, i] = w[:, finite] @ vi[finite]
            for j in np.flatnonzero(~finite):
                out[:, i] += np.where(see[:, j:j + 1], w[:, j:j + 1] * vi[j], 0.0)
            clean = np.where(np.isfinite(vi), np.abs(vi), 0.0)
            seen_bias = np.where(see & (np.abs(bias) < 1e30), np.abs(bias), 0.0).max(1, initial=0.0)
            seen_size = np.where(see & np.isfinite(magnitude), magnitude, 0.0).max(1, initial=0.0)
            e = (dim + 8) * 2 * U * seen_size + cap * 2.0 ** -20 + 8 * U * (seen_size + seen_bias) + 4 * U
            sums = w @ clean
            bound[:, i] = (2 * (h + e)[:, None] + 2 * U * nk) * sums + h * np.abs(out[:, i]) + 2.0 ** -25
            if kind == "f16":
                bound[:, i] += nk * 2.0 ** -25 * clean.max(initial=0.0)
    return out, bound


def rotate(x, positions, turns, amplitude=1.0, interleaved=False, direction=1):
    """x [rows][heads][dim] in 64 bits, turned; a position times a frequency in 64 bits of mantissa before whole turns go."""
    r = 2 * len(turns)
    turn = np.asarray(positions, np.longdouble)[:, None] * np.asarray(turns, np.longdouble)
    angle = 2 * np.pi * (turn - np.rint(turn)).astype(np.float64)[:, None]
    c, s = np.cos(angle) * amplitude, np.sin(angle) * amplitude * direction
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out = np.array(x, np.float64)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return out


def document_bounds(ids):
    ids = np.asarray(ids)
    edges = np.concatenate([[0], np.flatnonzero(np.diff(ids)) + 1, [len(ids)]]) if len(ids) else np.array([0])
    run = np.searchsorted(edges, np.arange(len(ids)), side="right") - 1
    return np.stack([edges[run], edges[run + 1]], 1) if len(ids) else np.zeros((0, 2), int)
