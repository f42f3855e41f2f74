"""NumPy reference of 8-bit rows (include/laya_hip.h): encoding, decoding, the norms and the product in 64 bits."""
import math

import numpy as np


def width8(width):
    return -(-width // 128) * 128


def _round_e4m3(y):
    """Codes of values of at most 448 in magnitude, ties to even (y: float64)."""
    mag = np.abs(y)
    _, p = np.frexp(mag)
    e = np.maximum(p - 1, -6)
    steps = np.rint(mag / np.exp2(e - 3.0)).astype(np.int64)  # 0..16 steps of 2^(e - 3)
    # A significand of 8..15 steps is normal; 16 carries into the next exponent by the same arithmetic.
    code = np.where(steps < 8, steps, ((e + 7) << 3) + (steps - 8))
    return np.where(np.signbit(y), code | 0x80, code).astype(np.uint8)


def encode(x):
    """(codes [rows][width8], scales [rows][width8 / 32]) of a float array; NaN codes in blocks that are not finite."""
    x = np.asarray(x, np.float64)
    rows, width = x.shape
    blocks = np.zeros((rows, width8(width)))
    blocks[:, :width] = x
    blocks = blocks.reshape(rows, -1, 32)
    finite = np.isfinite(blocks).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(blocks), blocks, 0)).max(-1), 0)
    e = np.full(top.shape, -127, np.int64)
    live = top > 0
    m, p = np.frexp(top[live])  # top = m 2^p: at most 448 2^e = 0.875 2^(e + 9)
    e[live] = np.maximum(p - 9 + (m > 0.875), -127)
    codes = _round_e4m3(np.where(finite[..., None], blocks, 0) * np.exp2(-e.astype(np.float64))[..., None])
    codes[~finite] = 0x7f
    return codes.reshape(rows, -1), np.where(finite, e + 127, 255).astype(np.uint8)


def code_values():
    """The 256 codes' values."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * np.exp2(e - 7.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


def decode(codes, scales, width):
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (code_values()[codes] * np.repeat(scale, 32, axis=1))[:, :width]


def activate(v, act):
    erf = np.vectorize(math.erf, otypes=[np.float64])

    def gelu(t):
        return 0.5 * t * (1 + erf(t / math.sqrt(2)))

    if act == "gelu":
        return gelu(v)
    if act == "relu":
        return np.where(v < 0, 0, v)
    if act in ("geglu", "swiglu"):
        g = v.reshape(len(v), -1, 2, 16)
        gate = gelu(g[:, :, 0]) if act == "geglu" else g[:, :, 0] / (1 + np.exp(-g[:, :, 0]))
        return (gate * g[:, :, 1]).reshape(len(v), -1)
    return v


def norm(v, gamma, beta, eps, rms):
    c = v if rms else v - v.mean(-1, keepdims=True)
    y = c / np.sqrt((c * c).mean(-1, keepdims=True) + eps) * gamma
    return y if beta is None else y + beta
