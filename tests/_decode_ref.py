"""Plain 64-bit definitions of the decode-step operators (numpy, loops over
sequences) that their GPU tests compare against."""
from __future__ import annotations

import numpy as np


def rotate(y, cos, sin, R, interleaved):
    """y [..., D] float64, cos / sin [R / 2]."""
    out = y.copy()
    a = np.arange(0, R, 2) if interleaved else np.arange(R // 2)
    b = a + 1 if interleaved else a + R // 2
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., b] * cos + y[..., a] * sin
    return out


def qk_norm_rope(qkv, wq, wk, cos, sin, positions, Hq, Hk, D, R, eps, interleaved):
    """(q, k, v) [T, heads, D] float64."""
    x = qkv.reshape(qkv.shape[0], Hq + 2 * Hk, D).astype(np.float64)
    q, k, v = x[:, :Hq].copy(), x[:, Hq:Hq + Hk].copy(), x[:, Hq + Hk:].copy()
    for t in range(x.shape[0]):
        for y, w in ((q, wq), (k, wk)):
            if w is not None:
                y[t] = y[t] / np.sqrt((y[t] ** 2).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
            if R:
                p = positions[t]
                if 0 <= p < cos.shape[0]:
                    y[t] = rotate(y[t], cos[p].astype(np.float64), sin[p].astype(np.float64), R, interleaved)
                else:
                    y[t] = np.nan
    return q, k, v


def attention(q, k, v, table, lens, scale, softcap=0.0, window=0):
    """q [B, Hq, D]; k, v [pages, Hk, P, D].  Returns out [B, Hq, D] and the
    softmax weights summed over the heads [B, pages in the table * P]."""
    B, Hq, D = q.shape
    pages, Hk, P, _ = k.shape
    out = np.zeros((B, Hq, D))
    added = np.zeros((B, table.shape[1] * P))
    for b in range(B):
        n = max(0, int(lens[b]))
        seen = [j for j in range(max(0, n - window) if window else 0, n) if 0 <= table[b, j // P] < pages]
        if not seen:
            continue
        j = np.array(seen)
        page = table[b, j // P]
        for h in range(Hq):
            kh = h // (Hq // Hk)
            s = k[page, kh, j % P].astype(np.float64) @ q[b, h].astype(np.float64) * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            top = s.max()
            p = np.exp(s - (top if np.isfinite(top) else 0.0 if top == -np.inf else top))
            if p.sum() == 0:
                continue
            p = p / p.sum()
            out[b, h] = p @ v[page, kh, j % P].astype(np.float64)
            added[b, j] += p
    return out, added


def evict(k, v, table, lens, weights, positions, max_context, budget, sinks, recent):
    """The cache, weights, positions and lengths afterwards (copies)."""
    k, v, weights, positions = k.copy(), v.copy(), weights.copy(), positions.copy()
    P = k.shape[2]
    after_lens = []
    for b in range(len(lens)):
        n = min(max(0, int(lens[b])), max_context)
        after = min(n, budget)
        if n > after and after:
            w = weights[b, :n].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w) + 0.0
            lowest = np.isnan(weights[b, :n])
            pos = positions[b, :n].astype(np.int64)
            safe = (pos < sinks) | (pos > pos.max() - recent)
            best = sorted(range(n), key=lambda i: (not safe[i], -w[i], lowest[i], i))[:after]
            stays = set(best)
            src = [i for i in range(after, n) if i in stays]
            dst = [i for i in range(after) if i not in stays]
            for i, j in zip(src, dst):
                a, c = table[b, i // P], table[b, j // P]
                if 0 <= a < len(k) and 0 <= c < len(k):
                    k[c, :, j % P], v[c, :, j % P] = k[a, :, i % P], v[a, :, i % P]
                weights[b, j], positions[b, j] = weights[b, i], positions[b, i]
        weights[b, after:max_context], positions[b, after:max_context] = 0.0, -1
        after_lens.append(after)
    return k, v, weights, positions, np.array(after_lens, np.int32)


def penalties(logits, history=None, history_lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
              bias_ids=None, bias_values=None, bias_counts=None, allowed=None):
    x = logits.astype(np.float64)
    B, V = x.shape
    for b in range(B):
        if history is not None:
            n = min(max(0, int(history_lens[b])), history.shape[1])
            m = int(prompt_lens[b]) if prompt_lens is not None else 0
            count, seen = np.zeros(V), np.zeros(V, bool)
            for i, t in enumerate(history[b, :n]):
                if 0 <= t < V:
                    seen[t] = True
                    count[t] += i >= m
            if repetition is not None:
                r = float(repetition[b])
                x[b] = np.where(seen, np.where(x[b] > 0, x[b] / r, x[b] * r), x[b])
            if frequency is not None:
                x[b] -= np.where(count > 0, float(frequency[b]) * count, 0.0)
            if presence is not None:
                x[b] -= np.where(count > 0, float(presence[b]), 0.0)
        if bias_ids is not None:
            m = bias_ids.shape[1] if bias_counts is None else min(max(0, int(bias_counts[b])), bias_ids.shape[1])
            last = {int(t): float(w) for t, w in zip(bias_ids[b, :m], bias_values[b, :m])}
            for t, w in last.items():
                if 0 <= t < V:
                    x[b, t] += w
        if allowed is not None:
            for t in range(V):
                if not (int(allowed[b, t // 32]) >> (t % 32)) & 1:
                    x[b, t] = -np.inf
    return x
