"""Norms of heads and their rotation by position in float64 numpy, from the definition,
with elementwise bounds of what float32 arithmetic and one rounding of the results may
change.

A row x of D values: r = (mean x^2 + eps)^(-1/2), y = x r w; pairs of the first R
values turned. A sum of n terms in float32, in any order, is off by at most n f of the
sum of their magnitudes (f = 2^-24); r, whose sum is of squares, by (D / 2 + 4) f of
itself (the square root halves it; the division by D, eps, the root and the quotient
round once each)."""
from __future__ import annotations

import numpy as np

from .attention import TINY, UNIT

F = 2.0 ** -24


def pairs(d, rotary, interleaved):
    """(index of the other value of each pair, sign of its sine, column of the angle), for the first `rotary` values."""
    i = np.arange(rotary)
    half = rotary // 2
    if interleaved:
        return i ^ 1, np.where(i % 2, 1.0, -1.0), i // 2
    return np.where(i < half, i + half, i - half), np.where(i < half, -1.0, 1.0), i % max(half, 1)


def turn(y, cos, sin, interleaved, back=False):
    """y [..., H, D] by the angles [..., R / 2] of its tokens, and the sum of magnitudes each result is made of."""
    other, sign, col = pairs(y.shape[-1], 2 * cos.shape[-1], interleaved)
    r = len(other)
    c, s = cos[..., None, col], sin[..., None, col] * (-sign if back else sign)
    z, size = y.copy(), np.abs(y)
    z[..., :r] = y[..., :r] * c + y[..., other] * s
    size[..., :r] = np.abs(y[..., :r] * c) + np.abs(y[..., other] * s)
    return z, size


def rows(x, w, cos, sin, positions, eps, interleaved, dtype, grad=None, weight_dtype="float32"):
    """One of q and k: x [B,T,H,D], w [D] (the offset in it), positions [B,T]. Returns a dict of y and, with
    grad, dx and dw, and bounds under the same names with "_tol"."""
    u, tiny = UNIT[dtype], TINY[dtype]
    d = x.shape[-1]
    known = (positions >= 0) & (positions < cos.shape[0])
    at = np.where(known, positions, 0)
    c, s = (t[at] if t.shape[0] else np.zeros((*at.shape, t.shape[1])) for t in (cos, sin))
    m = known[..., None, None]
    x = np.where(m, x, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        n = x * r * w
    z, size = turn(n, c, s, interleaved)
    of_r = (d / 2 + 4) * F
    out = {"y": np.where(m, z, 0.0), "y_tol": np.where(m, 1.1 * (u * np.abs(z) + (of_r + 6 * F) * size) + tiny, 0.0)}
    if grad is None:
        return out
    g = np.where(m, grad, 0.0)
    h, h_size = turn(g, c, s, interleaved, back=True)
    h_err = 4 * F * h_size
    t = h * w
    t_err = h_err * np.abs(w) + 3 * F * np.abs(t)
    mean = (t * x).mean(-1, keepdims=True)
    mean_err = (np.abs(x) * t_err).mean(-1, keepdims=True) + (d + 4) * F * np.abs(t * x).mean(-1, keepdims=True)
    dx = r * (t - x * r * r * mean)
    err = r * (t_err + np.abs(x) * r * r * (mean_err + (2 * of_r + 6 * F) * np.abs(mean)))
    err += (of_r + 4 * F) * r * (np.abs(t) + np.abs(x * r * r * mean))
    out["dx"] = np.where(m, dx, 0.0)
    out["dx_tol"] = np.where(m, 1.1 * (u * np.abs(dx) + err) + tiny, 0.0)
    hx = np.where(m, h * x * r, 0.0)
    axes = tuple(range(x.ndim - 1))
    terms = known.sum() * x.shape[-2]
    out["dw"] = hx.sum(axes)
    err = np.where(m, h_err * np.abs(x) * r + (of_r + 4 * F) * np.abs(hx), 0.0).sum(axes) + (terms + 4) * F * np.abs(hx).sum(axes)
    out["dw_tol"] = 1.1 * (UNIT[weight_dtype] * np.abs(out["dw"]) + err) + TINY[weight_dtype]
    return out
