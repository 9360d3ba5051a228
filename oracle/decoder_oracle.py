"""Oracle of the 8-bit decoder operators: their definitions in 64 bits, in numpy.

Inputs are arrays that hold the operators' inputs exactly (fp16 / bf16 / fp32 values as float64,
int8 codes); nothing here knows tiles, splits or matrix instructions.
"""
from __future__ import annotations

import math

import numpy as np

FLOOR = 2.0 ** -112


def quantize_rows(u):
    """(u / scale before rounding, scale) of the rows of u [rows, cols]; NaN for a row that is not
    finite."""
    u = np.asarray(u, np.float64)
    with np.errstate(all="ignore"):
        top = np.maximum(np.abs(u).max(-1), FLOOR)
        top = np.where(np.isfinite(u).all(-1), top, np.nan)
        return u * (127 / top)[:, None], top / 127


def rms_quantize(h, weight, eps):
    """(normalised / scale before rounding, scale, rstd) of rows h."""
    h, w = np.asarray(h, np.float64), np.asarray(weight, np.float64)
    rstd = 1 / np.sqrt((h * h).mean(-1) + eps)
    q, scale = quantize_rows(h * w)
    return q, scale * rstd, rstd


def rms_smooth(h, weight, eps):
    """The normalised rows without the rounding, whose derivative the training form takes."""
    h = np.asarray(h, np.float64)
    return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight


def rms_backward(h, weight, eps, dy, dh):
    """(dx, d_weight) with the rounding's gradient straight through."""
    h, w, dy = (np.asarray(v, np.float64) for v in (h, weight, dy))
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, dn = h * rstd, dy * w
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdims=True))
    return (dx if dh is None else dx + dh), (dy * n).sum(0)


def activation(v, act):
    if act == "relu":
        return np.where(v < 0, 0.0, v)
    if act == "silu":
        with np.errstate(over="ignore"):
            return v / (1 + np.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + np.vectorize(math.erf)(v / math.sqrt(2)))
    return v


def linear(codes, scales, weight, weight_scales, bias, act, residual):
    """(y, magnitude of what was added up for it)."""
    acc = codes.astype(np.float64) @ weight.astype(np.float64).T  # whole numbers below 2^53: exact
    v = acc * np.asarray(scales, np.float64)[:, None] * np.asarray(weight_scales, np.float64)
    size = np.abs(v)
    if bias is not None:
        v, size = v + bias, size + np.abs(bias)
    v = activation(v, act)
    if residual is not None:
        v, size = v + residual, size + np.abs(residual)
    return v, size


def append_page(old, old_scale, new):
    """One page and head: old codes [s0, dim] on old_scale, new values [n, dim].  (codes before
    rounding [s0 + n, dim], scale)."""
    new = np.asarray(new, np.float64)
    with np.errstate(all="ignore"):
        scale = max(np.abs(new).max(initial=0.0), FLOOR) / 127
        if len(old):
            scale = max(scale, float(old_scale))
        if not np.isfinite(new).all() or (len(old) and not np.isfinite(old_scale)):
            scale = np.nan
        moved = old.astype(np.float64) * (old_scale / scale) if len(old) else np.zeros((0, new.shape[1]))
        return np.concatenate([moved, new / scale]), scale


def attention(q, keys, k_scale, values, v_scale, count, scale, causal, window):
    """One sequence and cache head.  q [n, group, dim] are the last n of `count` tokens; keys, values
    [count, dim] codes with a scale for each token.  (out [n, group, dim], error that rounding
    the weights to 11 bits, relative to a reference up to 8 times the largest value scale, may make).
    """
    n, G, D = q.shape
    out, off = np.zeros((n, G, D)), np.zeros((n, G, D))
    for i in range(n):
        pos = count - n + i
        hi = min(count, pos + 1) if causal else count
        lo = max(0, pos - window + 1) if window else 0
        if lo >= hi:
            continue
        k = keys[lo:hi] * k_scale[lo:hi, None]
        v, vs = values[lo:hi].astype(np.float64), v_scale[lo:hi, None]
        for g in range(G):
            with np.errstate(all="ignore"):
                s = k @ q[i, g] * scale
                e = np.exp(s - s.max())
                out[i, g] = e @ (v * vs) / e.sum()
                w = np.maximum(2.0 ** -11 * e[:, None] * vs, 2.0 ** -25 * 8 * np.nanmax(v_scale))
                off[i, g] = (w * np.abs(v)).sum(0) / e.sum()
                off[i, g] += 2.0 ** -17 * (e @ (np.abs(v) * vs)) / e.sum()
    return out, off
