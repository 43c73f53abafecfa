"""Windowed attention in float64 numpy, from its definition: what the device
kernels are checked against, with bounds of their rounding errors.

A query at position p sees key j when j <= p and (j > p - window or j < sinks);
the queries are the last Tq positions of Tk keys. One head at a time, dense
scores."""
from __future__ import annotations

import numpy as np

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # rounding to nearest
TINY = {"float32": 2.0 ** -126, "bfloat16": 2.0 ** -126, "float16": 2.0 ** -24}  # spacing at zero, or flushed


def visible(tq, tk, window, sinks):
    pos = tk - tq + np.arange(tq)[:, None]
    key = np.arange(tk)[None, :]
    seen = key <= pos
    if window is not None:
        seen &= (key > pos - window) | (key < sinks)
    return seen


def head(q, k, v, scale, window, sinks, seen=None):
    """(o [Tq,D], lse [Tq], p [Tq,Tk]) of one head."""
    if seen is None:
        seen = visible(len(q), len(k), window, sinks)
    s = np.where(seen, scale * (q @ k.T), -np.inf)
    top = s.max(axis=1, initial=-np.inf, keepdims=True)
    w = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = w.sum(1, keepdims=True)
    some = total[:, 0] > 0
    p = np.where(some[:, None], w / np.where(total > 0, total, 1.0), 0.0)
    lse = np.full(len(q), -np.inf)
    lse[some] = top[some, 0] + np.log(total[some, 0])
    return p @ v, lse, p


def head_grad(q, k, v, scale, o, p, go, glse=None):
    """(dq, dk, dv, ds) of one head."""
    delta = (go * o).sum(1) - (0.0 if glse is None else np.where(p.sum(1) > 0, glse, 0.0))
    ds = p * (go @ v.T - delta[:, None])
    return scale * ds @ k, scale * ds.T @ q, p.T @ go, ds


def attention(q, k, v, scale, window=None, sinks=0, go=None, glse=None, dtype="float32"):
    """One sequence, all heads: q [Tq,Hq,D], k, v [Tk,Hk,D]. Returns a dict of
    o, lse and (with go) dq, dk, dv, and under the same names with "_tol" an
    elementwise bound of a kernel's error that reads inputs exactly, forms
    scores, softmax and sums in float32, rounds p and ds to `dtype` as product
    operands and its results once:
      scores     relative error of p: e = 2 (D 2^-24 scale |q|.|k| + 2^-21)
                 (the products' sums, log2(e) folded in, the exponential)
      sums       every sum of n terms: (n + 8) 2^-24 of the absolute sum
      rounding   u of each operand and of the result, u the type's unit
      delta      u of |do|.|o| (o is read back rounded)
    """
    u, tiny, f = UNIT[dtype], TINY[dtype], 2.0 ** -24
    ub = 0.0 if dtype == "float32" else u  # operands p and ds: float32 ones are not rounded
    tq, hq, d = q.shape
    tk, hk, _ = k.shape
    group = hq // hk
    out = {n: np.zeros(x.shape) for n, x in (("o", q), ("o_tol", q))}
    out["lse"], out["lse_tol"] = np.full((tq, hq), -np.inf), np.zeros((tq, hq))
    if go is not None:
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            out[n], out[n + "_tol"] = np.zeros(x.shape), np.zeros(x.shape)
    acc = (tk + d + 8) * f
    for h in range(hq):
        qh, kh, vh = q[:, h], k[:, h // group], v[:, h // group]
        seen = visible(tq, tk, window, sinks)
        kz, vz = (np.where(seen.any(0)[:, None], x, 0.0) for x in (kh, vh))  # what no query sees is never read
        o, lse, p = head(qh, kz, vz, scale, window, sinks, seen)
        e = 2 * (d * f * abs(scale) * np.abs(qh) @ np.abs(kz).T + 2.0 ** -21) * seen
        e = e + e.max(axis=1, initial=0.0, keepdims=True)  # of p: the score's own, and the sum's
        dp_ = p * e
        out["o"][:, h], out["lse"][:, h] = o, lse
        out["o_tol"][:, h] = u * np.abs(o) + ((ub + acc) * p + dp_) @ np.abs(vz) * 1.1 + tiny
        out["lse_tol"][:, h] = np.where(np.isfinite(lse), e.max(1, initial=0.0) + acc + 4 * f * np.abs(
            np.where(np.isfinite(lse), lse, 0.0)), 0.0)
        if go is None:
            continue
        g = go[:, h]
        dq, dk, dv, ds = head_grad(qh, kz, vz, scale, o, p, g, None if glse is None else glse[:, h])
        out["dq"][:, h] += dq
        out["dk"][:, h // group] += dk
        out["dv"][:, h // group] += dv
        absg, absdp = np.abs(g), np.abs(g) @ np.abs(vz).T
        delta_err = (u * np.abs(o) * absg).sum(1) + (out["o_tol"][:, h] * absg).sum(1) + acc * (np.abs(o) * absg).sum(1)
        if glse is not None:
            delta_err = delta_err + 4 * f * np.abs(glse[:, h])
        ds_err = ((ub + acc) * np.abs(ds) + dp_ * (absdp + np.abs(g * o).sum(1)[:, None]
                                                   + (0 if glse is None else np.abs(glse[:, h])[:, None]))
                  + p * (delta_err[:, None] + acc * absdp))
        p_err = (ub + (tq * group + 8) * f) * p + dp_ + (tiny if ub else 0.0) * seen
        out["dq_tol"][:, h] = u * np.abs(dq) + 1.1 * abs(scale) * (ds_err + acc * np.abs(ds)) @ np.abs(kz) + tiny
        sums = (tq * group + 8) * f
        out["dk_tol"][:, h // group] += u * np.abs(dk) + 1.1 * abs(scale) * (ds_err + sums * np.abs(ds)).T @ np.abs(qh) + tiny
        out["dv_tol"][:, h // group] += u * np.abs(dv) + 1.1 * p_err.T @ absg + tiny
    return out


def packed(q, k, v, scale, window, sinks, cu_q, cu_k, go=None, glse=None, dtype="float32"):
    """Packed sequences: attention of each, rows of none left at zero (lse -inf)."""
    total = None
    for b in range(len(cu_q) - 1):
        a, z, c, y = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        one = attention(q[a:z], k[c:y], v[c:y], scale, window, sinks, None if go is None else go[a:z],
                        None if glse is None else glse[a:z], dtype)
        if total is None:
            total = {n: np.zeros((k.shape[0] if n.startswith(("dk", "dv")) else q.shape[0],) + x.shape[1:])
                     for n, x in one.items()}
            total["lse"][:] = -np.inf
        for n, x in one.items():
            total[n][(slice(c, y) if n.startswith(("dk", "dv")) else slice(a, z))] = x
    return total
