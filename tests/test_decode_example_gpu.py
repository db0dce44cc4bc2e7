"""The decode loop of examples/decode_step.py against a plain forward pass in 64
bits while its cache holds everything, and what the cache holds once it does not."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decode_step
    finally:
        sys.path.pop(0)
    return decode_step


def _decoder(ex, budget, batch=2):
    cfg = ex.Config(hidden=256, q_heads=4, kv_heads=2, head_dim=64, inter=512, layers=2, vocab=500, page=8, budget=budget, sinks=2, recent=6,
                    longest=100)
    return ex.Decoder(cfg, batch, seed=3)


def _weight(w):
    q, s, z = (t.cpu().numpy() for t in w)
    nib = np.stack((q >> 4, q & 15), -1).reshape(q.shape[0], -1).astype(np.float64)
    return (nib - np.repeat(z.astype(np.float64), 128, 1)) * np.repeat(s.astype(np.float64), 128, 1)


def _rms(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)


def _forward(dec, tokens):
    """Logits [T, vocab] of one sequence, every token attending to all before it."""
    from tests._decode_ref import rotate
    c, T = dec.cfg, len(tokens)
    h = dec.embed.double().cpu().numpy()[tokens]
    cos, sin = dec.cos.double().cpu().numpy(), dec.sin.double().cpu().numpy()
    D, Hq, Hk = c.head_dim, c.q_heads, c.kv_heads
    for L in dec.layers:
        x = (_rms(h) @ _weight(L["qkv"]).T).reshape(T, Hq + 2 * Hk, D)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
        q, k = _rms(q) * L["qn"].double().cpu().numpy(), _rms(k) * L["kn"].double().cpu().numpy()
        q, k = (np.stack([rotate(y[t], cos[t], sin[t], D, False) for t in range(T)]) for y in (q, k))
        out = np.zeros((T, Hq, D))
        for hd in range(Hq):
            s = q[:, hd] @ k[:, hd // (Hq // Hk)].T / np.sqrt(D)
            s = np.where(np.tril(np.ones((T, T), bool)), s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            out[:, hd] = p / p.sum(-1, keepdims=True) @ v[:, hd // (Hq // Hk)]
        h = h + out.reshape(T, -1) @ _weight(L["o"]).T
        gu = _rms(h) @ _weight(L["up"]).T
        gate, up = gu[:, :c.inter], gu[:, c.inter:]
        h = h + gate / (1 + np.exp(-gate)) * up @ _weight(L["down"]).T
    return _rms(h) @ dec.head.double().cpu().numpy()


def test_steps_are_the_forward_pass():
    """fp16 activations through two layers: every stage rounds to 2^-11, some twenty of
    them in a row, whose errors the layers pass on about once each: 2 % of the
    largest logit is more than all of them together."""
    import torch
    ex = _example()
    dec = _decoder(ex, budget=40)
    tokens = torch.randint(0, 500, (2, 20), generator=dec.g, device="cuda")
    got = torch.stack([dec.step(tokens[:, t]).clone() for t in range(20)], 1).double().cpu().numpy()
    for b in range(2):
        want = _forward(dec, tokens[b].cpu().numpy())
        assert np.abs(got[b] - want).max() <= 0.02 * np.abs(want).max()
    assert dec.lens.tolist() == [20, 20]


def test_bounded_cache_holds_what_its_positions_say():
    import torch
    ex = _example()
    c = _decoder(ex, budget=20)
    cfg = c.cfg
    allowed = torch.full((2, -(-cfg.vocab // 32)), 0x55555555, dtype=torch.int32, device="cuda")
    seen = []  # layer -> position -> (k, v) rows of every head as they were written
    step = c.step

    def recording(tokens, **kw):
        pos = int(c.position[0])
        scores = step(tokens, **kw)
        seen.append(pos)
        for li, L in enumerate(c.layers):
            at = (L["positions"] == pos).nonzero()
            for b, i in at.tolist():
                page, row = int(c.table[b, i // cfg.page]), i % cfg.page
                rows[li][b][pos] = (L["cache"].k[page, :, row].clone(), L["cache"].v[page, :, row].clone())
        return scores

    rows = [[{}, {}] for _ in c.layers]
    c.step = recording
    prompt = torch.randint(0, cfg.vocab, (2, 6), generator=c.g, device="cuda")
    made = ex.generate(c, prompt, 50, allowed)
    assert bool((made % 2 == 0).all())
    assert c.lens.tolist() == [20, 20] and seen == list(range(56))
    for li, L in enumerate(c.layers):
        for b in range(2):
            pos = L["positions"][b].tolist()
            kept = pos[:20]
            assert pos[20:] == [-1] and len(set(kept)) == 20
            assert {0, 1} <= set(kept) and set(range(50, 56)) <= set(kept)  # the sinks and the newest
            assert bool((L["weights"][b, :20] > 0).all()) and float(L["weights"][b, 20]) == 0.0
            for i, p in enumerate(kept):
                page, row = int(c.table[b, i // cfg.page]), i % cfg.page
                k, v = rows[li][b][p]
                assert torch.equal(L["cache"].k[page, :, row], k) and torch.equal(L["cache"].v[page, :, row], v)
