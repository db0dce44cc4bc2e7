"""Workloads of the decode-step operators: norms and rotation of queries and
keys with the cache write, attention of one new token over the paged cache,
eviction from that cache by accumulated attention weight, and the penalties,
biases and masks on the logits.

`listed` names the standing cases, `draw` gives more of the same ranges,
`prepare` builds what a serving loop holds before the call and `run` makes one
call: through the library where `own` is set, in elementary torch operations
otherwise.  `exact` is the definition in 64 bits.  Inputs come from seeded
generators.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MOST_BYTES = 1.2e9  # no drawn case moves more than the largest listed one


def listed():
    return [
        # one token of one sequence after the fused QKV projection of a 1B-class
        # layer (32 query / 8 KV heads of 64): the smallest call
        dict(name="rope_token", op="rope", T=1, Hq=32, Hk=8, D=64, R=64, page=16, dtype="fp16", norm=True, interleaved=False),
        # a decode batch of 200 sequences, partial interleaved rotation
        dict(name="rope_batch", op="rope", T=200, Hq=32, Hk=8, D=128, R=64, page=32, dtype="bf16", norm=True, interleaved=True),
        # a long prompt chunk into the cache
        dict(name="rope_prompt", op="rope", T=8192, Hq=32, Hk=8, D=128, R=128, page=64, dtype="fp16", norm=True, interleaved=False),
        # a chat turn of one sequence: a few hundred cached tokens, latency bound
        dict(name="attend_short", op="attend", B=1, longest=411, ragged=False, Hq=32, Hk=8, D=64, page=16, dtype="fp16",
             window=0, softcap=0.0, weights=False),
        # one sequence with a long document in the cache: split over its length
        dict(name="attend_long", op="attend", B=1, longest=65536, ragged=False, Hq=32, Hk=8, D=128, page=64, dtype="bf16",
             window=0, softcap=0.0, weights=False),
        # a serving batch of mixed lengths, one empty, that accumulates the
        # attention weights eviction goes by
        dict(name="attend_batch", op="attend", B=48, longest=6144, ragged=True, Hq=32, Hk=8, D=64, page=16, dtype="fp16",
             window=0, softcap=0.0, weights=True),
        # a 7B-class layer with as many KV heads as query heads: the most cache per token
        dict(name="attend_heads", op="attend", B=16, longest=4096, ragged=False, Hq=32, Hk=32, D=128, page=32, dtype="fp16",
             window=0, softcap=0.0, weights=False),
        # one token over the budget in every sequence of a batch: each step of a full cache
        dict(name="evict_step", op="evict", B=48, longest=2049, ragged=False, budget=2048, sinks=4, recent=256, Hk=8, D=64,
             page=16, dtype="fp16"),
        # prompts of mixed lengths cut down to the budget
        dict(name="evict_prompt", op="evict", B=12, longest=24576, ragged=True, budget=4096, sinks=4, recent=1024, Hk=8,
             D=128, page=64, dtype="bf16"),
        # one sequence's logits after a long answer
        dict(name="logits_one", op="logits", B=1, V=32000, dtype="fp16", out="fp16", history=1500, bias=8, mask=False),
        # a structured-output batch over an odd vocabulary, every row with a grammar mask
        dict(name="logits_grammar", op="logits", B=33, V=50001, dtype="bf16", out="fp32", history=4000, bias=300, mask=True),
        # a large batch over a large vocabulary
        dict(name="logits_batch", op="logits", B=256, V=128000, dtype="fp32", out="fp32", history=8000, bias=64, mask=True),
    ]


def _logint(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "rope", "attend", "attend", "attend", "evict", "evict", "logits", "logits"])
        dtype, page = rng.choice(["fp16", "bf16"]), rng.choice([16, 16, 32, 64, 128, 24])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256, 100])
        Hk = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
        Hq = Hk * rng.choice([1, 1, 2, 4, 4, 5, 8, 16])
        if op == "rope":
            R = rng.choice([D, D, D, D // 2 // 4 * 4])
            c = dict(op=op, T=_logint(rng, 1, 8192), Hq=Hq, Hk=Hk, D=D, R=R, page=page, dtype=dtype, norm=rng.random() < 0.8,
                     interleaved=rng.random() < 0.4)
        elif op == "attend":
            c = dict(op=op, B=_logint(rng, 1, 128), longest=_logint(rng, 1, 131072), ragged=rng.random() < 0.6, Hq=Hq, Hk=Hk,
                     D=D, page=page, dtype=dtype, window=0, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                     weights=rng.random() < 0.35)
            if rng.random() < 0.2:
                c["window"] = _logint(rng, 16, 4096)
        elif op == "evict":
            longest = _logint(rng, 64, 65536)
            budget = longest - 1 if rng.random() < 0.35 else _logint(rng, 32, longest)
            c = dict(op=op, B=_logint(rng, 1, 64), longest=longest, ragged=rng.random() < 0.6, budget=budget,
                     sinks=rng.choice([0, 4, 16]), recent=_logint(rng, 1, max(1, budget // 2)), Hk=Hk, D=D, page=page, dtype=dtype)
        else:
            dtype = rng.choice(["fp16", "bf16", "fp32"])
            c = dict(op=op, B=_logint(rng, 1, 256), V=_logint(rng, 4000, 256000), dtype=dtype, out=rng.choice([dtype, "fp32"]),
                     history=_logint(rng, 1, 32000), bias=rng.choice([0, 1, 8, 300]), mask=rng.random() < 0.6)
        if Hq <= 128 and max(work(c)["bytes"], _held(c)) <= MOST_BYTES:
            return c


# ---- inputs -----------------------------------------------------------------

def _lengths(c, seed=None):
    """Lengths of the sequences: all the longest, or from nothing up to it, the
    same ones for every seed in another order."""
    if not c["ragged"]:
        return [c["longest"]] * c["B"]
    rng = random.Random(c["longest"])
    n = [_logint(rng, max(1, c["longest"] // 64), c["longest"]) for _ in range(c["B"])]
    n[0] = c["longest"]
    if c["B"] > 2:
        n[1] = 0  # a place of the batch that no sequence has
    if seed is not None:
        random.Random(seed).shuffle(n)
    return n


def _pages(c, lengths, g):
    """A page table over shuffled pages (unused entries -1) and how many pages there are."""
    per = [-(-n // c["page"]) for n in lengths]
    total = sum(per) + 3
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    width = max(1, -(-c["longest"] // c["page"]))
    start = torch.tensor([sum(per[:b]) for b in range(len(per))], device="cuda")
    at = torch.arange(width, device="cuda")
    used = at < torch.tensor(per, device="cuda")[:, None]
    table = torch.where(used, order[(start[:, None] + at).clamp(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total


def _normal(g, dtype, *shape, std=1.0):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _table64(T, R):
    """Angles of `T` positions."""
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    return torch.arange(T, dtype=torch.float64, device="cuda")[:, None] * f


def _inputs(c, seed):
    """What a case reads, from its seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "logits":
        B, V, H = c["B"], c["V"], c["history"]
        st = dict(logits=_normal(g, DTYPES[c["dtype"]], B, V, std=3.0))
        # tokens of a text come back: squared uniform numbers crowd the low ids
        st["history"] = (torch.rand(B, H, generator=g, device="cuda") ** 2 * V).to(torch.int32).clamp_(max=V - 1)
        st["history_lens"] = torch.randint((H + 1) // 2, H + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        st["prompt_lens"] = (st["history_lens"] * torch.rand(B, generator=g, device="cuda")).to(torch.int32)
        st["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=g, device="cuda")
        st["presence"] = 0.5 * torch.rand(B, generator=g, device="cuda")
        st["frequency"] = 0.2 * torch.rand(B, generator=g, device="cuda")
        n = c["bias"]
        st["bias_ids"] = torch.randint(0, V, (B, n), generator=g, device="cuda", dtype=torch.int32) if n else None
        st["bias_values"] = 2.0 * torch.randn(B, n, generator=g, device="cuda") if n else None
        st["bias_counts"] = torch.randint(0, n + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if n else None
        st["allowed"] = None
        if c["mask"]:
            words = -(-V // 32)
            st["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g, device="cuda").to(torch.int32)
        return st
    dt, Hk, D, P = DTYPES[c["dtype"]], c["Hk"], c["D"], c["page"]
    if c["op"] == "rope":
        T, R = c["T"], c["R"]
        pages = -(-T // P) + 2
        st = dict(qkv=_normal(g, dt, T, (c["Hq"] + 2 * Hk) * D))
        st["positions"] = torch.randint(0, 8192, (T,), generator=g, device="cuda", dtype=torch.int32)
        st["slots"] = torch.randperm(pages * P, generator=g, device="cuda", dtype=torch.int32)[:T].contiguous()
        if T >= P:  # a chunk fills whole pages in order
            page = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
            t = torch.arange(T, device="cuda", dtype=torch.int32)
            st["positions"], st["slots"] = t % 8192, page[t // P] * P + t % P
        angle = _table64(8192, R)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        norm = c["norm"]
        st["wq"] = 1.0 + _normal(g, dt, D, std=0.1) if norm else None
        st["wk"] = 1.0 + _normal(g, dt, D, std=0.1) if norm else None
        st["k"], st["v"] = (torch.zeros(pages, Hk, P, D, dtype=dt, device="cuda") for _ in range(2))
        return st
    n = _lengths(c, seed)
    table, pages = _pages(c, n, g)
    st = dict(table=table, lens=torch.tensor(n, dtype=torch.int32, device="cuda"))
    st["k"], st["v"] = _normal(g, dt, pages, Hk, P, D), _normal(g, dt, pages, Hk, P, D)
    if c["op"] == "attend":
        st["q"] = _normal(g, dt, c["B"], c["Hq"], D, std=1.5)
        st["weights"] = None
        if c["weights"]:  # what a few tokens have left there
            st["weights"] = torch.rand(c["B"], c["longest"], generator=g, device="cuda") * (8.0 * c["Hq"] / c["longest"])
    else:
        B, L = c["B"], c["longest"]
        # heavy-tailed sums of attention weights; tokens nothing looked at have none
        w = torch.exp(1.5 * torch.randn(B, L, generator=g, device="cuda"))
        st["weights"] = torch.where(torch.rand(B, L, generator=g, device="cuda") < 0.01, 0.0, w)
        # slots in the order that earlier evictions left
        st["positions"] = torch.rand(B, L, generator=g, device="cuda").argsort(1).to(torch.int32) + 1000
    return st


def prepare(case, seed):
    c = dict(case)
    st = _inputs(c, seed)
    st["case"] = c
    if c["op"] == "logits":
        st["out"] = torch.empty(c["B"], c["V"], dtype=DTYPES[c["out"]], device="cuda")
    elif c["op"] == "rope":
        st["q_out"] = torch.empty(c["T"], c["Hq"], c["D"], dtype=DTYPES[c["dtype"]], device="cuda")
    elif c["op"] == "attend":
        st["out"] = torch.empty_like(st["q"])
    else:
        st["weights_out"], st["positions_out"] = torch.empty_like(st["weights"]), torch.empty_like(st["positions"])
        st["lens_out"] = torch.empty_like(st["lens"])
    return st


# ---- one pass through the library ---------------------------------------------

def _own(st):
    import clove_compute_amd as cg
    c = st["case"]
    if c["op"] == "logits":
        cg.penalize_logits(st["logits"], st["out"], c["B"], c["V"], history=st["history"], history_lens=st["history_lens"],
                           prompt_lens=st["prompt_lens"], repetition=st["repetition"], presence=st["presence"],
                           frequency=st["frequency"], bias_ids=st["bias_ids"], bias_values=st["bias_values"],
                           bias_counts=st["bias_counts"], allowed=st["allowed"])
        return st["out"]
    # the handle of the cache, which a serving loop makes once and keeps
    cache = st.get("cache") or st.setdefault("cache", cg.KVCache(st["k"], st["v"]))
    if c["op"] == "rope":
        cg.qk_norm_rope(st["qkv"], st["wq"], st["wk"], st["cos"], st["sin"], st["positions"], st["q_out"], c["T"], c["Hq"],
                        c["Hk"], c["D"], rot_dim=c["R"], eps=1e-6, interleaved=c["interleaved"], cache=cache,
                        slots=st["slots"])
        return [st["q_out"], st["k"], st["v"]]
    if c["op"] == "attend":
        cg.paged_attention(st["q"], cache, st["table"], st["lens"], st["out"], c["B"], c["Hq"], c["longest"],
                           window=c["window"], softcap=c["softcap"], weights=st["weights"])
        return [st["out"], st["weights"]] if c["weights"] else st["out"]
    cg.cache_evict(cache, st["table"], st["lens"], st["weights"], st["positions"], st["weights_out"], st["positions_out"],
                   st["lens_out"], c["B"], c["longest"], c["budget"], sinks=c["sinks"], recent=c["recent"])
    return [st["k"], st["v"], st["weights_out"], st["positions_out"], st["lens_out"]]


# ---- the plain forms ------------------------------------------------------------

def _rotate(y, cos, sin, R, interleaved):
    """y [T, H, D] in 32 bits, cos / sin [T, R/2]."""
    cos, sin = cos[:, None], sin[:, None]
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    x, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((x, z), -1).flatten(-2) if interleaved else torch.cat((x, z), -1)
    return torch.cat((turned, y[..., R:]), -1)


def _plain_rope(st):
    c = st["case"]
    T, Hq, Hk, D, P = c["T"], c["Hq"], c["Hk"], c["D"], c["page"]
    x = st["qkv"].view(T, Hq + 2 * Hk, D)
    q, k, v = x[:, :Hq].float(), x[:, Hq:Hq + Hk].float(), x[:, Hq + Hk:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * st["wq"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * st["wk"].float()
    cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
    st["q_out"].copy_(_rotate(q, cos, sin, c["R"], c["interleaved"]))
    page, at = st["slots"].long() // P, st["slots"].long() % P
    st["k"][page, :, at] = _rotate(k, cos, sin, c["R"], c["interleaved"]).to(st["k"].dtype)
    st["v"][page, :, at] = v
    return [st["q_out"], st["k"], st["v"]]


def _gathered(cache, table):
    """[B, Hk, pages * page, D] of the pages of each sequence."""
    x = cache[table.clamp(min=0).long()]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(st):
    c = st["case"]
    B, Hq, Hk, D, L = c["B"], c["Hq"], c["Hk"], c["D"], c["longest"]
    at, n = torch.arange(L, device="cuda"), st["lens"][:, None]
    seen = (at < n) & ((at >= n - c["window"]) if c["window"] else (at >= 0))
    seen = seen[:, None, None]
    k = _gathered(st["k"], st["table"])[:, :, :L].float()
    s = torch.matmul(st["q"].float().view(B, Hk, Hq // Hk, D), k.transpose(2, 3)) / math.sqrt(D)
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = _gathered(st["v"], st["table"])[:, :, :L].float().masked_fill(~seen[:, 0, :, :, None], 0.0)
    st["out"].copy_(torch.matmul(p, v).view(B, Hq, D))
    if not c["weights"]:
        return st["out"]
    st["weights"] += p.sum((1, 2))
    return [st["out"], st["weights"]]


def _plain_evict(st):
    c = st["case"]
    L, P, budget = c["longest"], c["page"], c["budget"]
    at, n = torch.arange(L, device="cuda"), st["lens"][:, None]
    here = at < n
    newest = torch.where(here, st["positions"], -1).amax(1, keepdim=True)
    safe = (st["positions"] < c["sinks"]) | (st["positions"] > newest - c["recent"])
    order = torch.where(here, st["weights"], -math.inf).argsort(dim=1, descending=True, stable=True)
    rank = (2 * here + (here & safe)).to(torch.int8).gather(1, order)
    order = order.gather(1, rank.argsort(dim=1, descending=True, stable=True))
    kept = torch.zeros_like(here).scatter_(1, order, (at < budget).expand_as(order)) & here
    after = n.clamp(max=budget)
    hole, moves = ~kept & (at < after), kept & (at >= after)
    # the j-th moving slot goes into the j-th hole
    to = torch.nonzero(hole)
    b, frm = torch.nonzero(moves).unbind(1)
    to = to[:, 1]
    src, dst = st["table"][b, frm // P].long(), st["table"][b, to // P].long()
    st["k"][dst, :, to % P] = st["k"][src, :, frm % P]
    st["v"][dst, :, to % P] = st["v"][src, :, frm % P]
    st["lens_out"].copy_(after[:, 0])
    st["weights_out"].copy_(st["weights"])
    st["weights_out"][b, to] = st["weights"][b, frm]
    st["weights_out"].masked_fill_(at >= after, 0.0)
    st["positions_out"].copy_(st["positions"])
    st["positions_out"][b, to] = st["positions"][b, frm]
    st["positions_out"].masked_fill_(at >= after, -1)
    return [st["k"], st["v"], st["weights_out"], st["positions_out"], st["lens_out"]]


def _plain_logits(st):
    c = st["case"]
    B, V = c["B"], c["V"]
    at = torch.arange(c["history"], device="cuda")
    ids = st["history"].long()
    there = at < st["history_lens"][:, None]
    made = there & (at >= st["prompt_lens"][:, None])
    zero = torch.zeros(B, V, device="cuda")
    seen = zero.scatter_add(1, ids, there.float()) > 0
    count = zero.scatter_add(1, ids, made.float())
    x = st["logits"].float()
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if c["bias"]:
        # the last entry for a token counts
        entry = torch.arange(c["bias"], device="cuda").expand(B, -1)
        entry = torch.where(entry < st["bias_counts"][:, None], entry, -1)
        last = torch.full((B, V), -1, device="cuda").scatter_reduce(1, st["bias_ids"].long(), entry, "amax")
        x = x + torch.where(last >= 0, st["bias_values"].gather(1, last.clamp(min=0)), 0.0)
    if c["mask"]:
        v = torch.arange(V, device="cuda")
        x = x.masked_fill((st["allowed"][:, v // 32] >> (v % 32)) & 1 == 0, -math.inf)
    st["out"].copy_(x)
    return st["out"]


_PLAIN = {"rope": _plain_rope, "attend": _plain_attend, "evict": _plain_evict, "logits": _plain_logits}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def _held(c):
    """Bytes of the cache a case holds."""
    return 4.0 * sum(_lengths(c)) * c["Hk"] * c["D"] if c["op"] in ("attend", "evict") else 0.0


def work(case):
    c = case
    if c["op"] == "rope":
        T, H, D = c["T"], c["Hq"] + 2 * c["Hk"], c["D"]
        return {"bytes": 4.0 * T * H * D + 4.0 * T * c["R"] + 8.0 * T, "flops": 8.0 * T * H * D}
    if c["op"] == "attend":
        n = sum(min(x, c["window"] or x) for x in _lengths(c))
        return {"bytes": 4.0 * n * c["Hk"] * c["D"] + 4.0 * c["B"] * c["Hq"] * c["D"] + (8.0 * n if c["weights"] else 0.0),
                "flops": 4.0 * n * c["Hq"] * c["D"]}
    if c["op"] == "evict":
        # with weights in no order, a kept token lies past the budget as often as any
        n = sum(_lengths(c))
        moved = sum(c["budget"] * (x - c["budget"]) / x for x in _lengths(c) if x > c["budget"])
        return {"bytes": 8.0 * n + 8.0 * c["B"] * c["longest"] + 8.0 * moved * c["Hk"] * c["D"], "flops": 4.0 * n}
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    per = size[c["dtype"]] + size[c["out"]] + (0.125 if c["mask"] else 0.0)
    return {"bytes": c["B"] * (per * c["V"] + 3.0 * c["history"] + 8.0 * c["bias"]), "flops": 8.0 * c["B"] * c["V"]}


# ---- 64-bit results -----------------------------------------------------------------

def _exact_rope(c, st):
    T, Hq, Hk, D, R, P = c["T"], c["Hq"], c["Hk"], c["D"], c["R"], c["page"]
    pos = st["positions"].long()
    z = torch.complex(st["cos"].double()[pos], st["sin"].double()[pos])[:, None]

    def turn(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        y = x.clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        u = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        y[..., first], y[..., second] = u.real, u.imag
        return y

    x = st["qkv"].view(T, Hq + 2 * Hk, D)
    k, v = st["k"].double(), st["v"].double()
    slots = st["slots"].long()
    k.transpose(1, 2)[slots // P, slots % P] = turn(x[:, Hq:Hq + Hk], st["wk"])
    v.transpose(1, 2)[slots // P, slots % P] = x[:, Hq + Hk:].double()
    return [turn(x[:, :Hq], st["wq"]), k, v]


def _exact_attend(c, st):
    B, Hq, Hk, D, P = c["B"], c["Hq"], c["Hk"], c["D"], c["page"]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    weights = st["weights"].double() if c["weights"] else None
    for b, n in enumerate(st["lens"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == first:
            continue
        j = torch.arange(first, n, device="cuda")
        page = st["table"][b, j // P].long()
        for h in range(Hk):
            q = st["q"][b, h * (Hq // Hk):(h + 1) * (Hq // Hk)].double()
            s = (q @ st["k"][page, h, j % P].double().T) / math.sqrt(D)
            if c["softcap"]:
                s = c["softcap"] * torch.tanh(s / c["softcap"])
            p = torch.softmax(s, -1)
            out[b, h * (Hq // Hk):(h + 1) * (Hq // Hk)] = p @ st["v"][page, h, j % P].double()
            if c["weights"]:
                weights[b, first:n] += p.sum(0)
    return [out, weights] if c["weights"] else out


def _exact_evict(c, st):
    P, L = c["page"], c["longest"]
    k, v = st["k"].double(), st["v"].double()
    weights, positions = st["weights"].double().cpu().numpy(), st["positions"].cpu().numpy()
    table, lens = st["table"].cpu().numpy(), st["lens"].tolist()
    for b, n in enumerate(lens):
        w, pos = weights[b, :n].copy(), positions[b, :n].copy()
        after = min(n, c["budget"])
        if n > after:
            safe = (pos < c["sinks"]) | (pos > pos.max() - c["recent"])
            best = np.lexsort((np.arange(n), -w, ~safe))[:after]
            frm = np.sort(best[best >= after])
            to = np.setdiff1d(np.arange(after), best)
            src, dst = (torch.from_numpy(table[b, x // P].astype(np.int64)).cuda() for x in (frm, to))
            at, into = torch.from_numpy(frm % P).cuda(), torch.from_numpy(to % P).cuda()
            k[dst, :, into], v[dst, :, into] = k[src, :, at], v[src, :, at]
            weights[b, to], positions[b, to] = w[frm], pos[frm]
        weights[b, after:], positions[b, after:], lens[b] = 0.0, -1, after
    return [k, v, torch.from_numpy(weights), torch.from_numpy(positions), torch.tensor(lens, dtype=torch.int32)]


def _exact_logits(c, st):
    rows = []
    for b in range(c["B"]):
        x = st["logits"][b].double()
        n, m = int(st["history_lens"][b]), int(st["prompt_lens"][b])
        told, made = (torch.bincount(st["history"][b, i:n].long(), minlength=c["V"]) for i in (0, m))
        r, f, p = (float(st[name][b]) for name in ("repetition", "frequency", "presence"))
        x = torch.where(told > 0, torch.where(x > 0, x / r, x * r), x) - f * made - p * (made > 0)
        if c["bias"]:
            m = int(st["bias_counts"][b])
            told = dict(zip(st["bias_ids"][b, :m].tolist(), st["bias_values"][b, :m].tolist()))
            if told:
                x[torch.tensor(list(told), device="cuda")] += torch.tensor(list(told.values()), dtype=torch.float64, device="cuda")
        if c["mask"]:
            bits = (st["allowed"][b][:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.flatten()[:c["V"]] == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)


_EXACT = {"rope": _exact_rope, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}


def exact(case, seed):
    return _EXACT[case["op"]](case, _inputs(dict(case), seed))
