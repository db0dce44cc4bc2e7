"""Plain 64-bit definitions of the sparse MLP block's operators (numpy, loops over
tokens) that their GPU tests compare against."""
from __future__ import annotations

import math

import numpy as np

GROUP = 128


def block_norm(x, residual, post, gate, scale, pre, eps):
    """(y, h) float64; None where the operator takes NULL."""
    with np.errstate(all="ignore"):
        def unit(v):
            return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)

        y = 0.0 if residual is None else residual.astype(np.float64)
        if x is not None:
            u = x.astype(np.float64)
            if post is not None:
                u = unit(u) * post
            y = y + scale * (u if gate is None else u * gate)
        h = unit(y)
        return y, h if pre is None else h * pre


def _sigmoid(x):
    return 1.0 / (1.0 + math.exp(-x)) if x > -700 else 0.0


def route(logits, bias, score, groups, top_groups, group_top, top_k, renormalize, scale):
    """(ids, weights) of rows of logits (float64)."""
    T, E = logits.shape
    ids, weights = np.full((T, top_k), -1, np.int64), np.zeros((T, top_k))
    n = E // groups
    for t in range(T):
        x = logits[t]
        here = [e for e in range(E) if x[e] > -math.inf and (bias is None or bias[e] > -math.inf)]
        if score == "sigmoid":
            s = {e: _sigmoid(x[e]) for e in here}
        else:
            top = max((x[e] for e in here), default=0.0)
            s = {e: 1.0 if x[e] == top else math.exp(x[e] - top) for e in here}
            total = math.fsum(s.values())
            s = {e: v / total for e, v in s.items()}
        c = {e: s[e] + bias[e] for e in here} if bias is not None else s
        if groups > 1:
            value = {}
            for g in range(groups):
                v = sorted((c[e] for e in here if e // n == g), reverse=True)[:group_top]
                if v:
                    value[g] = v[0] + v[1] if len(v) > 1 else v[0]
            left = sorted(value, key=lambda g: (-value[g], g))[:top_groups]
            here = [e for e in here if e // n in left]
        took = sorted(here, key=lambda e: (-(x[e] if bias is None else c[e]), e))[:top_k]
        w = [s[e] for e in took]
        if renormalize and math.fsum(w) > 0:
            total = math.fsum(w)
            w = [v / total for v in w]
        ids[t, :len(took)] = took
        weights[t, :len(took)] = np.array(w) * scale
    return ids, weights


def dequantized(q, scale, zero, K):
    """[..., R, K] of packed rows q [..., R, K / 2]: even k in the high nibble."""
    w = np.stack((q >> 4, q & 15), -1).reshape(*q.shape[:-1], K).astype(np.float64)
    z = np.rint(zero.astype(np.float64)).repeat(GROUP, -1)[..., :K]
    return (w - z) * scale.astype(np.float64).repeat(GROUP, -1)[..., :K]


def swiglu_up(x, ids, w, h):
    """H after the call (float64): w [E, 2 I, K] dequantized, h [T top_k, I] before it.
    Also the size of the terms that each element's sums are made of."""
    T, k = ids.shape
    I = w.shape[1] // 2
    out, size = h.copy(), np.zeros_like(h)
    with np.errstate(all="ignore"):
        for p, e in enumerate(ids.reshape(-1)):
            if not 0 <= e < w.shape[0]:
                continue
            xt = x[p // k]
            g, u = w[e, :I] @ xt, w[e, I:] @ xt
            a = np.abs(xt)
            gs, us = np.abs(w[e, :I]) @ a, np.abs(w[e, I:]) @ a
            s = 1.0 / (1.0 + np.exp(-g))
            out[p] = g * s * u
            # |d silu| <= 1.1 |dg|
            size[p] = 1.1 * gs * np.abs(u) + np.abs(g * s) * us + np.abs(out[p])
    return out, size


def down(h, ids, weights, w, y, alpha, beta):
    """Y after the call (float64) and the size of its terms; w [E, O, K] dequantized."""
    T, k = ids.shape
    out, size = np.zeros(y.shape), np.zeros(y.shape)
    with np.errstate(all="ignore"):
        for p, e in enumerate(ids.reshape(-1)):
            if not 0 <= e < w.shape[0]:
                continue
            c = 1.0 if weights is None else float(weights.reshape(-1)[p])
            out[p // k] += c * (w[e] @ h[p])
            size[p // k] += abs(c) * (np.abs(w[e]) @ np.abs(h[p]))
        out, size = alpha * out, abs(alpha) * size
        if beta:
            out, size = out + beta * y, size + np.abs(beta * y)
    return out, size
