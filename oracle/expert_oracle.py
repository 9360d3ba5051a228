"""Oracle of the expert layers' operators: their definitions in 64 bits, in numpy.

Inputs are arrays that hold the operators' inputs exactly (fp16 / bf16 / fp32 values as float64,
int8 codes); nothing here knows lanes, tiles or chunks.
"""
from __future__ import annotations

import numpy as np

import decoder_oracle as D


def scores(logits, score):
    x = np.asarray(logits, np.float64)
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-x))
        top = x.max(-1, keepdims=True)
        e = np.exp(x - np.where(top == -np.inf, 0, top))
        total = e.sum(-1, keepdims=True)
        return np.where(total == 0, 0.0, e / np.where(total == 0, 1, total))


def choose(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, group_best=1):
    """int32 [tokens, top_k], best first."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    clean = lambda v: np.where(np.isnan(v), -np.inf, v) + 0.0
    rounded = scores(x, score).astype(np.float32)
    with np.errstate(all="ignore"):
        c = rounded if bias is None else rounded + np.asarray(bias, np.float32)
    order = clean(x if bias is None else c)
    out = np.zeros((T, top_k), np.int32)
    for t in range(T):
        among = np.arange(E)
        if groups > 1:
            by = clean(x[t].astype(np.float32) if bias is None and group_best == 1 else c[t])
            members = -np.sort(-by.reshape(groups, -1), axis=-1)
            n = min(group_best, E // groups)
            with np.errstate(all="ignore"):
                value = members[:, 0] if n == 1 else members[:, 0] + members[:, 1]
            best = sorted(range(groups), key=lambda g: (-clean(value)[g], g))
            among = np.sort(np.concatenate([np.arange(g * (E // groups), (g + 1) * (E // groups))
                                            for g in best[:top_groups or groups]]))
        out[t] = sorted(among, key=lambda e: (-order[t, e], e))[:top_k]
    return out


def weights(logits, experts, score="softmax", renormalize=True, scale=1.0):
    x = np.asarray(logits, np.float64)
    s = np.take_along_axis(scores(x, score), experts.astype(np.int64), 1)
    if renormalize:
        picked = np.take_along_axis(x, experts.astype(np.int64), 1)
        top = picked.max(-1, keepdims=True)
        with np.errstate(all="ignore"):
            if score == "softmax":  # the sum over all experts goes out
                s = np.exp(picked - top)
            else:  # relative to the largest, so that none underflows
                s = np.exp(np.minimum(picked, 0) - np.minimum(top, 0)) / (1 + np.exp(-np.abs(picked)))
            s = np.where(top == -np.inf, 0.0, s / s.sum(-1, keepdims=True))
    if score == "softmax":
        s = np.where((np.isnan(x) | (x == np.inf)).any(-1, keepdims=True), np.nan, s)
    return s * scale


def route_backward(logits, experts, d_weights, score="softmax", renormalize=True, scale=1.0):
    """Gradient of sum(weights * d_weights) for fixed experts."""
    x, g = np.asarray(logits, np.float64), np.asarray(d_weights, np.float64) * scale
    ids = experts.astype(np.int64)
    s = scores(x, score)
    w = weights(x, experts, score, renormalize)
    out = np.zeros_like(x)
    if renormalize:
        part = w * (g - (g * w).sum(-1, keepdims=True))
        if score == "sigmoid":
            part = part * (1 - np.take_along_axis(s, ids, 1))
        np.put_along_axis(out, ids, part, 1)
    elif score == "sigmoid":
        np.put_along_axis(out, ids, g * w * (1 - w), 1)
    else:
        np.put_along_axis(out, ids, g, 1)
        out = s * (out - (g * w).sum(-1, keepdims=True))
    return out


def group(experts, num_experts):
    """(offsets, entries, places)."""
    flat = experts.reshape(-1)
    ids = np.where((flat < 0) | (flat >= num_experts), num_experts, flat)
    entries = np.concatenate([np.nonzero(ids == e)[0] for e in range(num_experts + 1)]).astype(np.int32)
    offsets = np.array([(ids < e).sum() for e in range(num_experts + 1)], np.int32)
    places = np.empty(len(flat), np.int32)
    places[entries] = np.arange(len(flat), dtype=np.int32)
    places[ids == num_experts] = -1
    return offsets, entries, places.reshape(experts.shape)


def linear(codes, scales, weight, weight_scales, offsets, entries, top_k, bias, act, gated, grouped):
    """(y of the experts' places, magnitude of what was added up, slope of the last factor)."""
    rows, sizes = [], []
    for e in range(len(offsets) - 1):
        at = np.arange(offsets[e], offsets[e + 1])
        r = at if grouped else entries[at] // top_k
        b = None if bias is None else bias[e]
        if not gated:
            y, size = D.linear(codes[r], scales[r], weight[e], weight_scales[e], b, act, None)
        else:
            n = weight.shape[1] // 2
            up, us = D.linear(codes[r], scales[r], weight[e, n:], weight_scales[e, n:],
                              None if b is None else b[n:], None, None)
            y, size = D.linear(codes[r], scales[r], weight[e, :n], weight_scales[e, :n],
                               None if b is None else b[:n], act, None)
            y, size = y * up, size * np.abs(up) + np.abs(y) * us
        rows.append(y)
        sizes.append(size)
    return np.concatenate(rows), np.concatenate(sizes)


def combine(y, weights, places, residual):
    """(out, magnitude of what was added up)."""
    held = (places >= 0)[..., None]
    rows = np.where(held, y[np.maximum(places, 0)], 0.0) * weights[..., None]
    out, size = rows.sum(1), np.abs(rows).sum(1)
    if residual is not None:
        out, size = out + residual, size + np.abs(residual)
    return out, size


def combine_backward(y, weights, places, d_out):
    """(d_y, d_weights, magnitude of what was added up for d_weights)."""
    dy, dw, size = np.zeros_like(y), np.zeros_like(weights), np.zeros_like(weights)
    for t, row in enumerate(places):
        for j, p in enumerate(row):
            if p >= 0:
                dy[p] = weights[t, j] * d_out[t]
                dw[t, j] = d_out[t] @ y[p]
                size[t, j] = np.abs(d_out[t]) @ np.abs(y[p])
    return dy, dw, size
