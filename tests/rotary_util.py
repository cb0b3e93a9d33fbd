"""Rotation of new rows in 64 bits, with the error that FP32 arithmetic allows.

With gains, n = x r gain, r = 1 / sqrt(ss / D + eps): the sum of D squares, all
positive, in at most 8 fused steps and 4 additions is off by 12 2^-24 of itself,
its division by D is exact, the addition, the root (2 2^-24) and the division
(3 2^-24) add 6 2^-24 to half of 13 2^-24, and the two products 2 2^-24: less than
2^-19 of n. A rotated value adds the roundings of two products and a sum, 3 2^-24
of |n_i cos| + |n_j sin|. So |error| <= 2^-18 (|n_i cos| + |n_j sin|), and half a
step of the stored type more."""
import numpy as np

import xpu_playground_amd as xpu
from cache_util import HALF_STEP, TINY


def tables(positions, dims, theta=1e4):
    angle = np.arange(positions)[:, None] * theta ** -(np.arange(dims // 2) / (dims // 2))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def turned(x, at, cos, sin, adjacent=False, gain=None, eps=0.0):
    """x: [rows, heads, d] as float64; (result, |n_i cos| + |n_j sin|)."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * gain
    half = cos.shape[1]
    i = np.arange(half) * (2 if adjacent else 1)
    j = i + (1 if adjacent else half)
    c, s = (t[at][:, None].astype(np.float64) for t in (cos, sin))
    y, size = x.copy(), np.abs(x)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    size[..., i] = np.abs(x[..., i] * c) + np.abs(x[..., j] * s)
    size[..., j] = np.abs(x[..., j] * c) + np.abs(x[..., i] * s)
    return y, size


def bound(y, size, dtype):
    return 2.0 ** -18 * size + HALF_STEP[dtype] * (np.abs(y) + 2.0 ** -18 * size) + TINY[dtype]
