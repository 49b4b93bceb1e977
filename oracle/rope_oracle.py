"""Normalised and rotated rows from their definition, in 64 bits on the CPU
(numpy), with what a rounding bound is made of."""
from __future__ import annotations

import numpy as np


def turned(x, weight, eps, row, interleaved):
    """x [heads, D] of one token, row [r] its cosines and sines.  Returns
    (y, size): size is the sum of the magnitudes of the terms of each y."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    r = len(row)
    c, s = np.asarray(row[:r // 2], np.float64), np.asarray(row[r // 2:], np.float64)
    j = np.arange(r // 2)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + r // 2)
    y, size = x.copy(), np.abs(x)
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    size[:, a], size[:, b] = (np.abs(x[:, a] * c) + np.abs(x[:, b] * s), np.abs(x[:, b] * c) + np.abs(x[:, a] * s))
    return y, size


def bound(y, size, D, dtype_eps, subnormal):
    """How far float32 arithmetic, rounded once, may be off: half a step of the
    result; in float32 the sum of squares (D roundings, half of which reach its
    root), a root, a quotient, and up to five products and sums of each term."""
    e = (D / 2 + 10) * 2.0 ** -24 * size
    return dtype_eps / 2 * (np.abs(y) + e) + e + subnormal
