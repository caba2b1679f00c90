"""fp64 restatement of the operators around a recurrent mixer, each with a bound of what fp32
arithmetic may be off by, element by element, before the output's own rounding.

Sequences are lists of token ranges, so packed and batched calls share one code. The bounds
count roundings: ``U`` is half a unit in the last place of fp32 relative to the value.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import numpy as np

U = 2.0 ** -24
# exp2, reciprocal and what is built on them (sigmoid, softplus): a few units in the last
# place each; 2^-20 (16 half units) covers the longest chain, softplus
APPROX = 2.0 ** -20
# Exponentials below the smallest normal fp32 value are zero. A sigmoid(v) = e / (1 + e) with
# e = exp(v) < 2^-126 is then off by e itself, so by less than 2^-126, and w * v * sigmoid(v)
# by less than 2^-126 |w v|.
FLUSH = 2.0 ** -126


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1.0 + np.exp(-v))


def softplus(v):
    return np.maximum(v, 0.0) + np.log1p(np.exp(-np.abs(v)))


def short_conv(x, weight, bias, ranges: List[Tuple[int, int]], initial=None, activation="silu"):
    """x [T, D] -> (y, bound of y, final [N, W - 1, D]); tokens of no range are zero."""
    T, D = x.shape
    W = weight.shape[1]
    y, mag = np.zeros((T, D)), np.zeros((T, D))
    final = np.zeros((len(ranges), W - 1, D))
    b = np.zeros(D) if bias is None else bias
    for n, (s, e) in enumerate(ranges):
        past = np.zeros((W - 1, D)) if initial is None else initial[n]
        line = np.concatenate([past, x[s:e]])
        for t in range(s, e):
            win = line[t - s:t - s + W]                    # [W, D], oldest first
            y[t] = b + (weight.T * win).sum(0)
            mag[t] = np.abs(b) + np.abs(weight.T * win).sum(0)
        final[n] = line[e - s:]
    tol = (W + 1) * U * mag
    if activation == "silu":
        # |silu'| <= 1.1; exp's argument is rounded (|v| U log2 e), which its factor damps
        tol = 1.1 * tol + (APPROX + 2 * U * np.abs(y)) * np.abs(silu(y)) + FLUSH * np.abs(y)
        y = silu(y)
    return y, tol, final


def ssm_scan(x, dt, A, B, C, ranges, D=None, z=None, dt_bias=None, dt_softplus=True, initial=None,
             chunked=True):
    """x, dt, z [T, D], B, C [T, G, n] -> (y, bound of y, final [N, D, n], bound of final).

    The state's bound follows the recurrence: e[t] = a e[t-1] + |a h[t-1]| da + |dx B| db
    with da the relative error of a decay: its approximation and its argument's roundings: 4 U of
    one step's, and where a chunk's decay is formed from a compensated sum of its steps 10 U
    (of the sum 7, of A log2(e) 2, of their product 1), taken as 16.
    """
    T, ch = x.shape
    n, G = A.shape[1], B.shape[1]
    per = ch // G
    d = dt if dt_bias is None else dt + dt_bias
    # the sum dt + bias is rounded, then the activation is
    d_err = np.abs(d) * U
    if dt_softplus:
        slope = 1.0 / (1.0 + np.exp(-d))
        d = softplus(d)
        d_err = slope * d_err + APPROX * d
    y, ytol = np.zeros((T, ch)), np.zeros((T, ch))
    final, ftol = np.zeros((len(ranges), ch, n)), np.zeros((len(ranges), ch, n))
    for i, (s, e) in enumerate(ranges):
        h = np.zeros((ch, n)) if initial is None else initial[i].astype(np.float64)
        err = np.zeros((ch, n))
        for t in range(s, e):
            Bt, Ct = np.repeat(B[t], per, 0), np.repeat(C[t], per, 0)
            arg = d[t][:, None] * A
            a = np.exp(arg)
            add = (d[t] * x[t])[:, None] * Bt
            da = APPROX + np.abs(arg) * (16 * U if chunked else 4 * U) + np.abs(A) * d_err[t][:, None]
            db = 4 * U + d_err[t][:, None] / np.maximum(np.abs(d[t][:, None]), 1e-300)
            err = a * err + np.abs(a * h) * da + np.abs(add) * db
            h = a * h + add
            err = err + np.abs(h) * U
            skip = 0.0 if D is None else D * x[t]
            y[t] = (Ct * h).sum(1) + skip
            ytol[t] = ((np.abs(Ct) * err).sum(1) + (n + 8) * U * (np.abs(Ct * h).sum(1) + np.abs(skip)))
        final[i], ftol[i] = h, err
    if z is not None:
        g = silu(z)
        ytol = ytol * np.abs(g) + np.abs(y * g) * (APPROX + 2 * U * np.abs(z)) + FLUSH * np.abs(y * z)
        y = y * g
    return y, ytol, final, ftol


def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """(y, relative bound of y, h): a sum of D squares in pieces of at most 64 that meet in a
    tree of at most 16 levels, halved by the root, and a few roundings; the addition of x and
    residual, which are exact, is one of them (half a unit of h, whatever cancels)."""
    h = x if residual is None else x + residual
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight
    serial = 64 + max(0, x.shape[-1] // 256)
    return y, (serial + 16 + 16) * U, h


def e4m3_scale(y, group: Optional[int]):
    """[M, D] -> scales [M, groups]"""
    M, D = y.shape
    g = group or D
    out = [np.abs(y[:, c:c + g]).max(1) / 448.0 for c in range(0, D, g)]
    return np.maximum(np.stack(out, 1), 2.0 ** -126)
