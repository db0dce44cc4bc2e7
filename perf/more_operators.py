"""Workloads of a decoder's sparse MLP block: the norms before and after a block
with its residual, the router, and the products of the chosen experts on INT4
weights (gate and up with SwiGLU, then down with the weighted sum).

`listed` names the standing cases, `draw` gives more of the same ranges,
`prepare` builds what a program holds before the call and `run` makes one call:
through the library where `own` is set, in elementary torch operations
otherwise.  `exact` is the definition in 64 bits.  Inputs come from seeded
generators.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 128  # weights of a row that share a scale and a zero point
EPS = 1e-6


def listed():
    return [
        # the norm before a block of one token in a 1B-class decoder: the smallest call
        dict(name="norm_token", op="norm", T=1, D=2048, dtype="fp16", stream="fp16", post=False, gate="none", scale=1.0),
        # a decode batch with norms on both sides of the block and a gate per channel
        dict(name="norm_batch", op="norm", T=200, D=5120, dtype="bf16", stream="bf16", post=True, gate="row", scale=0.5),
        # a long prompt with the residual stream in fp32 and a gate for each token
        dict(name="norm_prompt", op="norm", T=8192, D=4096, dtype="fp16", stream="fp32", post=True, gate="rows", scale=1.0),
        # one token among 128 experts, renormalised softmax weights
        dict(name="route_token", op="route", T=1, E=128, k=8, dtype="fp16", score="softmax", bias=False, groups=1, top_groups=1,
             group_top=1, norm=True, masked=0.0),
        # a decode batch: sigmoid scores with a balance bias, half of the groups
        dict(name="route_batch", op="route", T=333, E=256, k=8, dtype="fp32", score="sigmoid", bias=True, groups=8, top_groups=4,
             group_top=2, norm=True, masked=0.0),
        # a long prompt over few experts' logits
        dict(name="route_prompt", op="route", T=16384, E=64, k=6, dtype="bf16", score="softmax", bias=False, groups=1, top_groups=1,
             group_top=1, norm=False, masked=0.0),
        # one token through its experts: eight narrow ones of 128
        dict(name="up_token", op="up", T=1, E=128, k=8, I=768, K=2048, absent=0.0),
        # a decode batch over 64 experts of uneven load, some places of it empty
        dict(name="up_batch", op="up", T=100, E=64, k=6, I=1408, K=2048, absent=0.1),
        # a prompt through two of eight wide experts
        dict(name="up_prompt", op="up", T=2048, E=8, k=2, I=11008, K=4096, absent=0.0),
        dict(name="down_token", op="down", T=1, E=128, k=8, O=2048, K=768, absent=0.0, beta=1.0),
        # a batch between decode and prefill: some tens of tokens for each expert
        dict(name="down_batch", op="down", T=500, E=64, k=6, O=2048, K=1408, absent=0.1, beta=1.0),
        # a prompt through narrow experts, eight for each token
        dict(name="down_prompt", op="down", T=8192, E=128, k=8, O=2048, K=768, absent=0.0, beta=0.0),
    ]


MOST_BYTES = 4.6e8  # no drawn case moves more than the largest listed one
MOST_FLOPS = 7.3e11  # ... or computes more


def _logint(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "norm", "route", "route", "up", "up", "up", "down", "down", "down"])
        if op == "norm":
            dtype = rng.choice(["fp16", "bf16"])
            c = dict(op=op, T=_logint(rng, 1, 8192), D=rng.choice([_logint(rng, 64, 16384), _logint(rng, 8, 2048) * 8]), dtype=dtype,
                     stream=rng.choice([dtype, dtype, "fp32"]), post=rng.random() < 0.6, gate=rng.choice(["none", "row", "rows"]),
                     scale=rng.choice([1.0, 0.25, 1.5]))
        elif op == "route":
            E = rng.choice([_logint(rng, 4, 512), 8, 32, 60, 64, 128, 160, 256, 384])
            groups = rng.choice([1, 1, 2, 4, 8])
            if E % groups:
                groups = 1
            c = dict(op=op, T=_logint(rng, 1, 16384), E=E, k=0, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                     score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                     top_groups=rng.randint(1, groups), group_top=rng.choice([1, 2]), norm=rng.random() < 0.6,
                     masked=rng.choice([0.0, 0.0, 0.1, 0.9]))
            c["k"] = rng.randint(1, min(12, E))
        else:
            E = rng.choice([_logint(rng, 4, 256), 8, 16, 60, 64, 128])
            c = dict(op=op, T=_logint(rng, 1, 8192), E=E, k=rng.randint(1, min(8, E)))
            # K holds whole 16-byte pieces of a row, mostly whole groups; the rows are as many as they like
            K = rng.choice([128 * _logint(rng, 2, 88), 128 * _logint(rng, 2, 32), 32 * _logint(rng, 8, 256)])
            rows = rng.choice([128 * _logint(rng, 2, 64), _logint(rng, 200, 8192)])
            c.update(dict(I=rows, K=K) if op == "up" else dict(O=rows, K=K))
            c["absent"] = rng.choice([0.0, 0.0, 0.15])
            if op == "down":
                c["beta"] = rng.choice([0.0, 1.0])
            if E * _rows(c) * K / 2 > MOST_BYTES:  # (held, whether some token hits them or not)
                continue
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


# ---- inputs -----------------------------------------------------------------

def _rows(c):
    """Weight rows of one expert."""
    return 2 * c["I"] if c["op"] == "up" else c["O"]


def _normal(g, dtype, *shape, std=1.0):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _popularity(E):
    """Log-odds of the experts: some are chosen several times as often as others."""
    return [0.6 * math.sin(2.4 * e + 1.0) + 0.4 * math.cos(1.7 * e) for e in range(E)]


def _choices(c, g):
    """Expert ids [T, k] as a router leaves them: distinct in a row, uneven over the
    experts; rows of padding tokens hold -1."""
    T, E, k = c["T"], c["E"], c["k"]
    pop = torch.tensor(_popularity(E), device="cuda")
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp(1e-7, 1.0 - 1e-7)))
    ids = (pop + noise).topk(k, dim=1).indices.to(torch.int32)
    gone = torch.rand(T, 1, generator=g, device="cuda") < c["absent"]
    return torch.where(gone, -1, ids).contiguous()


def _weights4(g, E, R, K):
    """Random 4-bit rows of E experts, with scales and zero points for each group."""
    G = -(-K // GROUP)
    q = torch.randint(0, 256, (E, R, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand(E, R, G, generator=g, device="cuda") + 0.5).mul_(1.0 / (4.6 * K ** 0.5)).half()
    zero = torch.randint(6, 11, (E, R, G), generator=g, device="cuda").half()
    return q, scale, zero


def _inputs(c, seed):
    """What a case reads, from its seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "norm":
        T, D, dt, sdt = c["T"], c["D"], DTYPES[c["dtype"]], DTYPES[c["stream"]]
        st = dict(x=_normal(g, dt, T, D), residual=_normal(g, sdt, T, D, std=3.0), pre=1.0 + _normal(g, dt, D, std=0.1))
        st["post"] = 1.0 + _normal(g, dt, D, std=0.1) if c["post"] else None
        st["gate"] = None if c["gate"] == "none" else _normal(g, dt, *((T, D) if c["gate"] == "rows" else (D,)))
        return st
    if c["op"] == "route":
        T, E = c["T"], c["E"]
        x = _normal(g, torch.float32, T, E, std=1.5)
        if c["masked"]:  # experts that are switched off for a token; with 0.9, now and then all of them
            x.masked_fill_(torch.rand(T, E, generator=g, device="cuda") < c["masked"], -math.inf)
        return dict(logits=x.to(DTYPES[c["dtype"]]), bias=_normal(g, torch.float32, E, std=0.1) if c["bias"] else None)
    ids = _choices(c, g)
    q, scale, zero = _weights4(g, c["E"], _rows(c), c["K"])
    st = dict(ids=ids, q=q, scale=scale, zero=zero)
    if c["op"] == "up":
        st["x"] = _normal(g, torch.float16, c["T"], c["K"])
    else:
        st["h"] = _normal(g, torch.float16, c["T"] * c["k"], c["K"], std=0.5)
        w = torch.rand(c["T"], c["k"], generator=g, device="cuda") + 0.05
        st["w"] = w / w.sum(1, keepdim=True)
        st["y0"] = _normal(g, torch.float16, c["T"], c["O"])
    return st


def prepare(case, seed):
    c = dict(case)
    st = _inputs(c, seed)
    st["case"] = c
    if c["op"] == "norm":
        st["y"] = torch.empty_like(st["residual"])
        st["out"] = torch.empty_like(st["x"])
    elif c["op"] == "route":
        st["ids"] = torch.empty(c["T"], c["k"], dtype=torch.int32, device="cuda")
        st["w"] = torch.empty(c["T"], c["k"], device="cuda")
    elif c["op"] == "up":
        st["h"] = torch.zeros(c["T"] * c["k"], c["I"], dtype=torch.float16, device="cuda")
    else:
        st["y"] = st.pop("y0")  # the residual stream, which the call adds to
    return st


# ---- one pass through the library ---------------------------------------------

def _own(st):
    import clove_compute_amd as cg
    c = st["case"]
    if c["op"] == "norm":
        cg.block_norm(st["x"], st["residual"], st["out"], c["T"], c["D"], y_out=st["y"], post_weight=st["post"],
                      pre_weight=st["pre"], gate=st["gate"], scale=c["scale"], eps=EPS)
        return [st["y"], st["out"]]
    if c["op"] == "route":
        score = cg.CLOVE_ROUTE_SIGMOID if c["score"] == "sigmoid" else cg.CLOVE_ROUTE_SOFTMAX
        cg.moe_route(st["logits"], st["ids"], st["w"], c["T"], c["E"], c["k"], score=score, bias=st["bias"], groups=c["groups"],
                     top_groups=c["top_groups"], group_top=c["group_top"], renormalize=c["norm"])
        return [st["ids"], st["w"]]
    if c["op"] == "up":
        cg.moe_w4a16_swiglu(st["x"], st["ids"], st["q"], st["scale"], st["zero"], st["h"], c["T"], c["k"], c["E"], c["I"], c["K"])
        return st["h"]
    cg.moe_w4a16(st["h"], st["ids"], st["w"], st["q"], st["scale"], st["zero"], st["y"], c["T"], c["k"], c["E"], c["O"], c["K"],
                 beta=c["beta"])
    return st["y"]


# ---- the plain forms ------------------------------------------------------------

def _normed(v, w):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w


def _plain_norm(st):
    c = st["case"]
    u = st["x"].float()
    if c["post"]:
        u = _normed(u, st["post"].float())
    if c["gate"] != "none":
        u = u * st["gate"].float()
    y = st["residual"].float() + c["scale"] * u
    st["y"].copy_(y)
    st["out"].copy_(_normed(y, st["pre"].float()))
    return [st["y"], st["out"]]


def _plain_route(st):
    c = st["case"]
    T, E, k = c["T"], c["E"], c["k"]
    x = st["logits"].double()  # (64 bits: experts whose values nearly agree must not change places)
    here = x > -math.inf
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        top = x.amax(1, keepdim=True)
        s = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
        total = s.sum(1, keepdim=True)
        s = s / torch.where(total > 0, total, 1.0)
    v = s + st["bias"].double() if c["bias"] else s
    order = (v if c["bias"] else x).masked_fill(~here, -math.inf)
    if c["groups"] > 1:
        n = E // c["groups"]
        of = v.masked_fill(~here, -math.inf).view(T, c["groups"], n).sort(dim=2, descending=True).values[:, :, :c["group_top"]]
        some = of[:, :, 0] > -math.inf
        value = torch.where(of > -math.inf, of, 0.0).sum(2).masked_fill(~some, -math.inf)
        best = value.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros(T, c["groups"], dtype=torch.bool, device="cuda").scatter_(1, best, True)
        order = order.masked_fill(~kept.repeat_interleave(n, 1), -math.inf)
    order, ids = order.sort(dim=1, descending=True, stable=True)
    order, ids = order[:, :k], ids[:, :k]
    found = order > -math.inf
    w = torch.where(found, s.gather(1, ids), 0.0)
    if c["norm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    st["ids"].copy_(torch.where(found, ids, -1))
    st["w"].copy_(w)
    return [st["ids"], st["w"]]


def _dequantized(st, e, dtype):
    """Rows of expert e [R, K], or of several experts [n, R, K]."""
    q = st["q"][e]
    w = torch.stack((q >> 4, q & 15), -1).flatten(-2).to(dtype)  # the even k in the high nibble
    K = w.shape[-1]
    z = st["zero"][e].to(dtype).repeat_interleave(GROUP, -1)[..., :K]
    return (w - z) * st["scale"][e].to(dtype).repeat_interleave(GROUP, -1)[..., :K]


def _gated(c, y):
    if c["op"] == "down":
        return y
    gate, up = y[:, :c["I"]], y[:, c["I"]:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _experts(st, out):
    """Products of every pair's row with its expert's, into `out`: of few pairs each with
    weights of its own, of more an expert at a time."""
    c = st["case"]
    flat = st["ids"].flatten()
    P = c["T"] * c["k"]
    if P <= c["E"] and P * _rows(c) * c["K"] <= 1 << 28:
        rows = (st["x"].repeat_interleave(c["k"], 0) if c["op"] == "up" else st["h"]).float()
        y = torch.bmm(_dequantized(st, flat.clamp(min=0).long(), torch.float32), rows[:, :, None].contiguous())[:, :, 0]
        out.copy_(torch.where(flat[:, None] >= 0, _gated(c, y), out))
        return out
    for e in range(c["E"]):
        pairs = torch.nonzero(flat == e)[:, 0]
        if pairs.numel() == 0:
            continue
        rows = st["x"][pairs // c["k"]] if c["op"] == "up" else st["h"][pairs]
        out[pairs] = _gated(c, torch.matmul(rows.float(), _dequantized(st, e, torch.float32).T)).to(out.dtype)
    return out


def _plain_up(st):
    return _experts(st, st["h"])


def _plain_down(st):
    c = st["case"]
    T, k, O = c["T"], c["k"], c["O"]
    y = _experts(st, torch.zeros(T * k, O, device="cuda"))
    total = (y.view(T, k, O) * st["w"][:, :, None]).sum(1)
    st["y"].copy_(total + c["beta"] * st["y"].float() if c["beta"] else total)
    return st["y"]


_PLAIN = {"norm": _plain_norm, "route": _plain_route, "up": _plain_up, "down": _plain_down}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def _hit(c):
    """How many experts some token of the case has chosen, about."""
    odds = [math.exp(p) for p in _popularity(c["E"])]
    T, total = c["T"] * (1.0 - c["absent"]), sum(odds)
    return sum(1.0 - (1.0 - min(1.0, c["k"] * o / total)) ** T for o in odds)


def work(case):
    c = case
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    if c["op"] == "norm":
        per = 2 * size[c["dtype"]] + 2 * size[c["stream"]] + (size[c["dtype"]] if c["gate"] == "rows" else 0)
        return {"bytes": float(per) * c["T"] * c["D"] + 4.0 * c["D"], "flops": 10.0 * c["T"] * c["D"]}
    if c["op"] == "route":
        return {"bytes": float(size[c["dtype"]]) * c["T"] * c["E"] + 8.0 * c["T"] * c["k"], "flops": 8.0 * c["T"] * c["E"]}
    R, K, P = _rows(c), c["K"], c["T"] * c["k"] * (1.0 - c["absent"])
    rows = _hit(c) * R * (K / 2 + 4.0 * -(-K // GROUP))
    if c["op"] == "up":
        return {"bytes": rows + 2.0 * c["T"] * K + 2.0 * P * c["I"], "flops": 2.0 * P * R * K}
    return {"bytes": rows + 2.0 * P * K + (4.0 if c["beta"] else 2.0) * c["T"] * c["O"], "flops": 2.0 * P * R * K}


# ---- 64-bit results -----------------------------------------------------------------

def _exact_norm(c, st):
    u = st["x"].double()

    def unit(v):
        return v / (v.pow(2).sum(-1, keepdim=True) / c["D"] + EPS).sqrt()

    if c["post"]:
        u = unit(u) * st["post"].double()
    if st["gate"] is not None:
        u = u * st["gate"].double()
    y = st["residual"].double() + c["scale"] * u
    return [y, unit(y) * st["pre"].double()]


def _exact_route(c, st):
    """A row at a time on the host, by sorting (value, index) pairs."""
    if c["T"] * c["E"] > 1 << 21:
        return None
    ids, weights = [], []
    bias = st["bias"].double().tolist() if c["bias"] else [0.0] * c["E"]
    n = c["E"] // c["groups"]
    for x in st["logits"].double().tolist():
        here = [e for e in range(c["E"]) if x[e] > -math.inf]
        if c["score"] == "sigmoid":
            s = {e: 1.0 / (1.0 + math.exp(-x[e])) for e in here}
        else:
            top = max((x[e] for e in here), default=0.0)
            total = math.fsum(math.exp(x[e] - top) for e in here)
            s = {e: math.exp(x[e] - top) / total for e in here}
        value = {e: s[e] + bias[e] for e in here}
        if c["groups"] > 1:
            per = {}
            for e in here:
                per.setdefault(e // n, []).append(value[e])
            rank = sorted(per, key=lambda q: (-sum(sorted(per[q], reverse=True)[:c["group_top"]]), q))
            here = [e for e in here if e // n in rank[:c["top_groups"]]]
        took = sorted(here, key=lambda e: (-(value[e] if c["bias"] else x[e]), e))[:c["k"]]
        w = [s[e] for e in took]
        if c["norm"] and w and sum(w) > 0:
            total = math.fsum(w)
            w = [v / total for v in w]
        ids.append(took + [-1] * (c["k"] - len(took)))
        weights.append(w + [0.0] * (c["k"] - len(w)))
    return [torch.tensor(ids, dtype=torch.int32), torch.tensor(weights, dtype=torch.float64)]


def _exact_products(c, st):
    """[T k, R] of the chosen experts: each group's whole numbers times the row, then its scale."""
    T, k, R, K = c["T"], c["k"], _rows(c), c["K"]
    x = (st["x"].double().repeat_interleave(k, 0) if c["op"] == "up" else st["h"].double())
    out = torch.zeros(T * k, R, dtype=torch.float64, device="cuda")
    ids = st["ids"].flatten().cpu().tolist()
    of = {}
    for p, e in enumerate(ids):
        if 0 <= e < c["E"]:
            of.setdefault(e, []).append(p)
    for e, pairs in of.items():
        at = torch.tensor(pairs, device="cuda")
        rows = x[at]
        w = torch.empty(R, K, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (st["q"][e] // 16).double(), (st["q"][e] % 16).double()
        for g in range(-(-K // GROUP)):
            part = slice(GROUP * g, min(K, GROUP * g + GROUP))
            w[:, part] = (w[:, part] - st["zero"][e][:, g, None].double()) * st["scale"][e][:, g, None].double()
        out[at] = rows @ w.T.contiguous()
    return out


def _exact_up(c, st):
    y = _exact_products(c, st)
    gate, up = y[:, :c["I"]], y[:, c["I"]:]
    return gate * torch.sigmoid(gate) * up


def _exact_down(c, st):
    y = _exact_products(c, st).view(c["T"], c["k"], c["O"])
    total = torch.zeros(c["T"], c["O"], dtype=torch.float64, device="cuda")
    for j in range(c["k"]):
        total += st["w"][:, j, None].double() * y[:, j]
    return total + c["beta"] * st["y0"].double()


_EXACT = {"norm": _exact_norm, "route": _exact_route, "up": _exact_up, "down": _exact_down}


def exact(case, seed):
    c = dict(case)
    return _EXACT[c["op"]](c, _inputs(c, seed))
