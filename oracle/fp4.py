"""The 4-bit cache's format in numpy, from its definition: the codes and scale bytes of
rows of values, and the values that they stand for, in float64."""
from __future__ import annotations

import numpy as np

BLOCK = 32
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_bytes(x):
    """x [..., d] float64 -> scale bytes [..., d / 32]."""
    top = np.abs(x).reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK).max(-1)
    finite = np.isfinite(top)
    mantissa, e = np.frexp(np.where(finite & (top > 0), top, 1.0))  # top = mantissa 2^e, mantissa in [1/2, 1)
    e = e - 1 + (mantissa >= 1.75 / 2)
    e = np.where(top > 0, e, -1000)
    return np.where(finite, np.clip(e - 2 + 127, 2, 252), 255).astype(np.uint8)


def codes(x, scales):
    """The codes [..., d] of x by its scale bytes: the nearest, ties to the even code."""
    s = 2.0 ** (scales.astype(np.float64) - 127)
    with np.errstate(invalid="ignore"):
        y = np.abs(x).reshape(*scales.shape, BLOCK) / s[..., None]
        off = np.abs(y[..., None] - VALUES)
    best = np.where(np.isnan(off), np.inf, off).min(-1, keepdims=True)
    hits = off == best
    even = hits & (np.arange(8) % 2 == 0)
    at = np.where(even.any(-1), even.argmax(-1), hits.argmax(-1))
    return (at.reshape(x.shape) + 8 * (x < 0)).astype(np.uint8)


def pack(c):
    """Codes [..., d] as bytes [..., d / 2]."""
    return (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)


def quantise(x):
    """x [..., d] -> (bytes [..., d / 2], scale bytes [..., d / 32])."""
    x = np.asarray(x, np.float64)
    scales = scale_bytes(x)
    return pack(codes(x, scales)), scales


def values(data, scales):
    """What bytes and scale bytes stand for, float64."""
    c = np.stack((data & 15, data >> 4), -1).reshape(*data.shape[:-1], 2 * data.shape[-1])
    x = VALUES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (x.reshape(*scales.shape, BLOCK) * s[..., None]).reshape(x.shape)
