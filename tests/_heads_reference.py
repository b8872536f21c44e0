"""The batched attention operators from their formulas, in 64 bits on the CPU, one sequence and head at a time -- with bounds on how far
the kernels may be off, counted from the roundings they make:

* u = half a step of the output type (bf16 2^-8, fp32 2^-24): the one rounding of an output, relative to its value;
* w = half a step of the operand type: softmax weights (and dS) are rounded to it before a product, relative to each term;
* a score is a sum of dk products in fp32: off by (dk + 4) 2^-24 sum |q k| scale, and what a score is off by, its weight is off by
  relatively (the exponential's own error and the running rescale: 2^-20 in all);
* sums over n keys or rows in fp32: n 2^-24 of the sum of magnitudes.
"""
import math

import numpy as np

F32 = 2.0 ** -24
EXP = 2.0 ** -20


def half_step(dtype):
    return {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}[dtype]


def visible(nq, nk, window, sinks):
    pos = nk - nq + np.arange(nq)[:, None]
    key = np.arange(nk)[None, :]
    return (key <= pos) & ((pos - key < window) | (key < sinks))


def attention(q, k, v, see, scale, dtype):
    """one head: q [nq, dk], k [nk, dk], v [nk, dv] -> out, lse, weights P, and the bounds of out, lse, P's relative error"""
    s = scale * (q @ k.T)
    nq, nk = s.shape
    ds = (q.shape[1] + 4) * F32 * abs(scale) * (np.abs(q) @ np.abs(k).T)
    p = np.zeros_like(s)
    lse = np.full(nq, -np.inf)
    err = np.zeros(nq)                                     # a row's relative error of any weight
    for i in range(nq):
        at = see[i]
        if at.any():
            m = s[i, at].max()
            e = np.exp(s[i, at] - m)
            lse[i] = m + math.log(e.sum())
            p[i, at] = e / e.sum()
            err[i] = 2 * ds[i, at].max() + EXP + nk * F32 + abs(m) * 4 * F32
    seen_v = np.where(see.any(0)[:, None], v, 0.0)
    out = p @ seen_v
    mag = p @ np.abs(seen_v)
    u = half_step(dtype)
    tol_out = u * np.abs(out) + mag * ((u if dtype == "bf16" else 0) + err[:, None] + nk * F32) + 1e-30
    tol_lse = err + np.where(np.isfinite(lse), np.abs(lse), 0.0) * 4 * F32
    return out, lse, p, tol_out, tol_lse, err


def gradients(q, k, v, dout, p, out, err, scale, dtype):
    """-> dq, dk, dv of one query head and their bounds"""
    u = half_step(dtype)
    w = u if dtype == "bf16" else 0.0
    n = max(q.shape[0], k.shape[0])
    dp = dout @ v.T
    delta = (dout * out).sum(1, keepdims=True)
    ds = p * (dp - delta)
    # what the pair's dS is off by: its own rounding, the weight's error, the two sums', and `out` as it was stored
    e = np.abs(ds) * (w + err[:, None]) + p * ((v.shape[1] + 4) * F32 * (np.abs(dout) @ np.abs(v).T) +
                                               (u + w + err[:, None] + n * F32) * (np.abs(dout) * np.abs(out)).sum(1, keepdims=True) +
                                               w * (p @ np.abs(v) * np.abs(dout)).sum(1, keepdims=True))
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ dout
    a = np.abs
    tq = u * a(dq) + abs(scale) * (e + n * F32 * a(ds)) @ a(k) + 1e-30
    tk = abs(scale) * (e + n * F32 * a(ds)).T @ a(q) + 1e-30          # (the group's sum is rounded once: the caller adds u |dk|)
    tv = (p * (w + err[:, None] + n * F32)).T @ a(dout) + 1e-30
    return dq, dk, dv, tq, tk, tv


def kept(weights, n, budget, sinks, recent):
    """old indices that stay, for one row of weights"""
    if n <= budget:
        return list(range(n))
    order = sorted(range(sinks, n - recent), key=lambda j: (0 if weights[j] != weights[j] else 1, 0.0 if weights[j] != weights[j] else weights[j]), reverse=True)
    # (sorted(reverse=True) keeps the order of equal elements: ties stay at the lowest index)
    return sorted(list(range(sinks)) + order[:budget - sinks - recent] + list(range(n - recent, n)))
