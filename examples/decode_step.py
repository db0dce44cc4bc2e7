#!/usr/bin/env python3
"""A decode loop on the library: INT4 linear layers, the operators around them and
a key-value cache of bounded size.

Each step takes one token per sequence through a Llama-style decoder -- fused QKV
projection, norms and rotation of queries and keys with the cache write, attention
over the pages (which also adds up what each cached token is attended with), output
projection into the residual stream, SwiGLU MLP, or with --experts a sparse one: a
router and the products of the experts it chose -- and through the logits'
penalties and grammar mask to the next token.  A sequence that outgrows the budget
loses the token of the least accumulated attention weight in every layer, so the
cache never holds more than `budget` tokens a sequence however long the answer is.

Weights are random: the point is the calls and what they share.

    python examples/decode_step.py --steps 64 --batch 4 --budget 48
    python examples/decode_step.py --experts 32 --top-k 4 --inter 1024
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import clove_compute_amd as cg  # noqa: E402

GROUP = cg.INT4_GROUP_SIZE


class Config:
    def __init__(self, hidden=2048, q_heads=32, kv_heads=8, head_dim=64, inter=8192, layers=2, vocab=32000, page=16, budget=48,
                 sinks=4, recent=16, longest=4096, experts=0, top_k=2):
        self.hidden, self.q_heads, self.kv_heads, self.head_dim, self.inter = hidden, q_heads, kv_heads, head_dim, inter
        self.layers, self.vocab, self.page, self.budget, self.sinks, self.recent = layers, vocab, page, budget, sinks, recent
        self.longest = longest
        self.experts, self.top_k = experts, top_k  # 0 experts: a dense MLP


class Decoder:
    def __init__(self, cfg: Config, batch: int, seed: int = 0):
        self.cfg, self.batch = cfg, batch
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        c, half = cfg, torch.float16
        qkv = (c.q_heads + 2 * c.kv_heads) * c.head_dim
        self.embed = self._normal(c.vocab, c.hidden)
        self.head = self._normal(c.hidden, c.vocab, std=c.hidden ** -0.5)
        # one page table for all layers: each has its own pages of the same numbers
        self.capacity = c.budget + 1  # the new token is there before one leaves
        per = -(-self.capacity // c.page)
        self.table = torch.randperm(batch * per, generator=self.g, device="cuda").to(torch.int32).view(batch, per)
        self.layers = []
        for _ in range(c.layers):
            k, v = (torch.zeros(batch * per, c.kv_heads, c.page, c.head_dim, dtype=half, device="cuda") for _ in range(2))
            self.layers.append(dict(
                qkv=self._int4(qkv, c.hidden), o=self._int4(c.hidden, c.q_heads * c.head_dim), **self._mlp(), qn=1.0 + self._normal(c.head_dim, std=0.1), kn=1.0 + self._normal(c.head_dim, std=0.1),
                cache=cg.KVCache(k, v), weights=torch.zeros(batch, self.capacity, device="cuda"),
                positions=torch.full((batch, self.capacity), -1, dtype=torch.int32, device="cuda")))
        angle = torch.arange(c.longest, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, c.head_dim, 2, dtype=torch.float64, device="cuda") / c.head_dim)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")       # tokens in the cache
        self.lens_out = torch.zeros_like(self.lens)
        self.position = torch.zeros(batch, dtype=torch.int32, device="cuda")   # of the next token
        self.history = torch.zeros(batch, c.longest, dtype=torch.int32, device="cuda")
        self.rows = torch.arange(batch, device="cuda")

        def buffer(*shape):
            return torch.empty(*shape, dtype=half, device="cuda")

        self.hidden, self.x = buffer(batch, c.hidden), buffer(batch, c.hidden)
        self.proj, self.q = buffer(batch, qkv), buffer(batch, c.q_heads, c.head_dim)
        self.attn, self.act = buffer(batch, c.q_heads, c.head_dim), buffer(batch * (c.top_k if c.experts else 1), c.inter)
        if c.experts:
            self.route = buffer(batch, c.experts)
            self.chosen = torch.empty(batch, c.top_k, dtype=torch.int32, device="cuda")
            self.share = torch.empty(batch, c.top_k, device="cuda")
        self.logits, self.scores = buffer(batch, c.vocab), torch.empty(batch, c.vocab, device="cuda")

    def _normal(self, *shape, std=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * std).half()

    def _int4(self, out, k):
        """Random 4-bit weights whose product has about unit variance."""
        q = torch.randint(0, 256, (out, k // 2), generator=self.g, device="cuda", dtype=torch.uint8)
        scale = torch.full((out, k // GROUP), 1.0 / (4.6 * k ** 0.5), device="cuda").half()
        return q, scale, torch.full_like(scale, 8.0)

    def _mlp(self):
        c = self.cfg
        if not c.experts:
            return dict(up=self._int4(2 * c.inter, c.hidden), down=self._int4(c.hidden, c.inter))
        up, down = ([torch.stack(x) for x in zip(*(self._int4(r, k) for _ in range(c.experts)))]
                    for r, k in ((2 * c.inter, c.hidden), (c.hidden, c.inter)))
        return dict(up=up, down=down, router=self._normal(c.hidden, c.experts, std=c.hidden ** -0.5))

    def _norm(self, out):
        cg.block_norm(None, self.hidden, out, self.batch, self.cfg.hidden)

    def step(self, tokens, **penalties):
        """The tokens [batch] through the model: fp32 scores [batch, vocab] of the next
        ones, after the penalties (penalize_logits' arguments)."""
        c, B = self.cfg, self.batch
        self.history[self.rows, self.position.long()] = tokens.to(torch.int32)
        self.hidden.copy_(self.embed[tokens])
        # the new token's place: the slot after the last one
        at = self.lens.long()
        slots = (self.table[self.rows, at // c.page] * c.page + (at % c.page).to(torch.int32)).to(torch.int32)
        self.lens += 1
        for L in self.layers:
            L["positions"][self.rows, at], L["weights"][self.rows, at] = self.position, 0.0
            self._norm(self.x)
            cg.gemm_w4a16(self.x, *L["qkv"], self.proj, B, self.proj.shape[1], c.hidden)
            cg.qk_norm_rope(self.proj, L["qn"], L["kn"], self.cos, self.sin, self.position, self.q, B, c.q_heads, c.kv_heads, c.head_dim,
                            cache=L["cache"], slots=slots)
            cg.paged_attention(self.q, L["cache"], self.table, self.lens, self.attn, B, c.q_heads, self.capacity, weights=L["weights"])
            cg.gemm_w4a16(self.attn, *L["o"], self.hidden, B, c.hidden, c.q_heads * c.head_dim, 1.0, 1.0)
            cg.cache_evict(L["cache"], self.table, self.lens, L["weights"], L["positions"], L["weights"], L["positions"], self.lens_out, B,
                           self.capacity, c.budget, sinks=c.sinks, recent=c.recent)
            self._norm(self.x)
            if c.experts:
                cg.gemm_fp16(self.x, L["router"], self.route, B, c.experts, c.hidden)
                cg.moe_route(self.route, self.chosen, self.share, B, c.experts, c.top_k, renormalize=True)
                cg.moe_w4a16_swiglu(self.x, self.chosen, *L["up"], self.act, B, c.top_k, c.experts, c.inter, c.hidden)
                cg.moe_w4a16(self.act, self.chosen, self.share, *L["down"], self.hidden, B, c.top_k, c.experts, c.hidden, c.inter, beta=1.0)
            else:
                cg.w4a16_swiglu(self.x, *L["up"], self.act, B, c.inter, c.hidden)
                cg.gemm_w4a16(self.act, *L["down"], self.hidden, B, c.hidden, c.inter, 1.0, 1.0)
        self.lens.copy_(self.lens_out)  # every layer keeps as many
        self.position += 1
        self._norm(self.x)
        cg.gemm_fp16(self.x, self.head, self.logits, B, c.vocab, c.hidden)
        cg.penalize_logits(self.logits, self.scores, B, c.vocab, history=self.history, history_lens=self.position, **penalties)
        return self.scores


def generate(dec: Decoder, prompt, steps: int, allowed=None):
    """`prompt` [batch, n] a token at a time, then `steps` greedy tokens: [batch, steps]."""
    B = dec.batch
    told = torch.full((B,), prompt.shape[1], dtype=torch.int32, device="cuda")
    penalty = dict(prompt_lens=told, repetition=torch.full((B,), 1.1, device="cuda"), presence=torch.full((B,), 0.2, device="cuda"),
                   frequency=torch.full((B,), 0.1, device="cuda"), allowed=allowed)
    for i in range(prompt.shape[1]):
        scores = dec.step(prompt[:, i], **penalty)
    made = []
    for _ in range(steps):
        made.append(scores.argmax(-1))
        scores = dec.step(made[-1], **penalty)
    return torch.stack(made, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--budget", type=int, default=48)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--inter", type=int, default=8192, help="width of the MLP, or of one expert")
    ap.add_argument("--experts", type=int, default=0, help="of a sparse MLP (0: a dense one)")
    ap.add_argument("--top-k", type=int, default=2, help="experts a token")
    a = ap.parse_args()
    cfg = Config(budget=a.budget, layers=a.layers, inter=a.inter, experts=a.experts, top_k=a.top_k)
    dec = Decoder(cfg, a.batch)
    prompt = torch.randint(0, cfg.vocab, (a.batch, 8), generator=dec.g, device="cuda")
    # a grammar that allows even tokens only
    allowed = torch.full((a.batch, -(-cfg.vocab // 32)), 0x55555555, dtype=torch.int32, device="cuda")
    tokens = generate(dec, prompt, 4, allowed)
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens = generate(dec, tokens, a.steps, allowed)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    print(f"{a.batch} sequences, {a.layers} layers: {(a.steps + 4) / t * a.batch:.0f} tokens/s, "
          f"{int(dec.position[0])} tokens seen, {int(dec.lens[0])} in the cache (budget {cfg.budget})")
    print("first sequence:", tokens[0, :16].tolist())


if __name__ == "__main__":
    main()
