"""Quantised pages from their definition, in 64 bits on the CPU (numpy): blocks
of 32 elements share the smallest power of two 2^e, -117 <= e <= 127, that
brings the block's largest magnitude within 448 (mxfp8) or 6 (mxfp4); elements
are the nearest representable values, ties to the even code; a block with a
non-finite value has scale byte 255 and zero elements."""
from __future__ import annotations

import numpy as np

BLOCK = 32
TOP = {"mxfp8": 448.0, "mxfp4": 6.0}
_E4M3 = np.array([(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)])
_E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = {"mxfp8": _E4M3, "mxfp4": _E2M1}


def quantize(x: np.ndarray, fmt: str):
    """(codes [..., D], scale bytes [..., D / 32]) of x [..., D] (float64)."""
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    finite = np.isfinite(b).all(-1)
    amax = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0)).max(-1), 0)
    e = np.full(amax.shape, -117)
    while (bad := (amax > TOP[fmt] * 2.0 ** e)).any():
        e = e + bad
    y = np.where(finite[..., None], np.where(np.isfinite(b), b, 0) * 2.0 ** (-e.astype(np.float64))[..., None], 0)
    v = VALUES[fmt]
    mid = (v[1:] + v[:-1]) / 2
    a = np.abs(y)
    code = np.searchsorted(mid, a, side="left")
    tie = (code < len(mid)) & (a == mid[np.minimum(code, len(mid) - 1)])
    code = code + (tie & (code % 2 == 1))
    code = code + np.where(np.signbit(y), 128 if fmt == "mxfp8" else 8, 0)
    byte = np.where(finite, e + 127, 255)
    return code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def pack(codes: np.ndarray, fmt: str) -> np.ndarray:
    """Element bytes: one each, or two to a byte with the even one low."""
    return codes if fmt == "mxfp8" else codes[..., 0::2] | (codes[..., 1::2] << 4)


def values(data: np.ndarray, byte: np.ndarray, fmt: str) -> np.ndarray:
    """float64 values of element bytes and scale bytes."""
    if fmt == "mxfp8":
        code, sign = data & 127, data >> 7
        v = np.append(_E4M3, np.nan)[code]
    else:
        code = np.stack([data & 15, data >> 4], -1).reshape(data.shape[:-1] + (2 * data.shape[-1],))
        code, sign = code & 7, code >> 3
        v = _E2M1[code]
    v = np.where(sign == 1, -v, v)
    scale = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    b = v.reshape(v.shape[:-1] + (v.shape[-1] // BLOCK, BLOCK)) * scale[..., None]
    return b.reshape(v.shape)


def page_half(x: np.ndarray, fmt: str) -> np.ndarray:
    """The bytes of half a page from its values [P, H, D]."""
    codes, byte = quantize(x, fmt)
    return np.concatenate([pack(codes, fmt).ravel(), byte.ravel()])


def split(cache: np.ndarray, head_dim: int):
    """Views (element bytes, scale bytes) of caches [..., P, H, R]."""
    P, H, R = cache.shape[-3:]
    width = R - head_dim // BLOCK
    flat = cache.reshape(cache.shape[:-3] + (-1,))
    cut = P * H * width
    return (flat[..., :cut].reshape(cache.shape[:-1] + (width,)),
            flat[..., cut:].reshape(cache.shape[:-1] + (head_dim // BLOCK,)))
