"""Attention over a paged cache from its definition, query by query in 64 bits
on the CPU (numpy): the tokens a query sees are picked first, so what the
others hold cannot matter."""
from __future__ import annotations

import numpy as np


def attend(q, keys, values, scale, cap, sees):
    """One request.  q [T, Hq, D], keys and values [n, H, D] (its tokens in
    order), sees [T, n] bool.  Returns out, lse, and what a rounding bound is
    made of: per output the weighted mean of |v|, and per row the largest
    sum |q k| * scale, the sum of |v| over the row's weight total, and the
    tokens seen."""
    T, Hq, D = q.shape
    H = keys.shape[1]
    out, lse = np.zeros((T, Hq, D)), np.full((T, Hq), -np.inf)
    mean, dots, spread = np.zeros((T, Hq, D)), np.zeros((T, Hq)), np.zeros((T, Hq, D))
    for i in range(T):
        at = np.flatnonzero(sees[i])
        if not len(at):
            continue
        for h in range(Hq):
            k, v = keys[at, h // (Hq // H)], values[at, h // (Hq // H)]
            with np.errstate(invalid="ignore", over="ignore"):
                s = (k @ q[i, h]) * scale
                if cap > 0:
                    s = cap * np.tanh(s / cap)
                m = s.max()
                p = np.exp(s - m)
                out[i, h] = p @ v / p.sum()
                lse[i, h] = m + np.log(p.sum())
                mean[i, h] = p @ np.abs(v) / p.sum()
                dots[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() * scale
                spread[i, h] = np.abs(v).sum(0) / p.sum()
    return out, lse, mean, dots, spread


def visible(n, T, mask):
    """sees [T, n] of a request of n tokens whose last T are queries; mask: rows
    of 64-bit words, or None for each seeing itself and those before."""
    d = np.arange(n)[None, :] - (n - T)
    if mask is None:
        return d <= np.arange(T)[:, None]
    sees = np.broadcast_to(d < 0, (T, n)).copy()
    for i in range(T):
        for j in range(T):
            if 0 <= n - T + j < n and (int(mask[i, j // 64]) >> (j % 64)) & 1:
                sees[i, n - T + j] = True
    return sees


def bounds(D, dtype_eps, out, lse, mean, dots, spread, cap, n, subnormal):
    """How far a result in float32 sums with weights rounded to the values' type
    may be off: (out, lse).
    scores   D + 4 float32 roundings of sum |q k|, then cap's tanh (2^-21 of it)
    weights  half a step of the type each (eps / 2), or of its subnormals
             against a row's largest weight of 1; twice the scores' error, the
             exponential's 2^-21
    out      half a step of the result; sums of n / 32 partial float32 results"""
    u = dtype_eps / 2
    e_s = ((D + 4) * 2.0 ** -24 * dots + 2.0 ** -21 * cap)
    rel = 2 * e_s + 2.0 ** -21 + (n / 32 + 64) * 2.0 ** -24
    with np.errstate(invalid="ignore", over="ignore"):
        o = u * (mean + np.abs(out)) * (1 + u) + rel[..., None] * mean * 1.01 + subnormal * (spread + 1)
        s = 2 * e_s + 2.0 ** -21 + (n + 64) * 2.0 ** -24 + 2.0 ** -21 * np.abs(np.where(np.isfinite(lse), lse, 0))
    return o, s
