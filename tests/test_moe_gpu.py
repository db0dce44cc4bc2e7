"""The sparse MLP block's operators against their plain 64-bit definitions (_moe_ref).

Tolerances.  An output is rounded once: half a unit in the last place.  What fp32
leaves before that:
 * norms: a sum of D <= 32768 squares in a tree of at most 32 + 6 + 16 additions, at
   most 54 2^-24 of it, half of that in its root, and a handful of roundings more:
   below 40 2^-24 = 2.4e-6 of the terms an element is made of; 4e-6 is taken.
 * products: a group's sum adds at most 128 exact products, each addition off by at
   most 2^-23 of the partial sum (MFMA may truncate), the fold of G groups, K splits
   and places by 2^-24 each: (256 + 2 G + 64) 2^-24 of the sum of the terms' sizes,
   and 8 2^-24 for SwiGLU.  Accumulators that go on from group to group in units of
   the group's scale have 2 G 2^-24 for the units (a quotient and a product each), and
   partial sums that are no longer a group's: with terms of random sign, as here, one
   of n terms of size s is about s sqrt(n), so K / 16 additions of 2^-23 each leave
   2^-23 s K^1.5 / 24, of the terms' K s a part of 2^-23 sqrt(K) / 24: 10 2^-24 at K =
   14336, far below the 256.
 * routing: ids are equal; weights are 64-bit results rounded to fp32.
"""
import numpy as np
import pytest

from tests import _moe_ref as ref
from tests._util import rng
from tests.test_decode_gpu import HALF_ULP, TINY, _dev, _dt, _f64, _rounded

pytestmark = pytest.mark.gpu


def _cg():
    import clove_compute_amd as cg
    return cg


def _close(got, want, dtype, extra):
    got, want = _f64(got), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = np.isfinite(want)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    err = np.abs(got - np.where(ok, want, 0.0))[ok]
    bound = HALF_ULP[dtype] * np.abs(want[ok]) * 1.0001 + TINY[dtype] + np.broadcast_to(extra, want.shape)[ok]
    assert np.all(err <= bound), (float(np.max(err - bound)), float(err.max()))


# ---- block_norm ---------------------------------------------------------------

FP32 = 4e-6


def _norm_bounds(x, residual, post, gate, scale, pre, eps, y, h):
    """What fp32 may leave in y and h."""
    term = np.zeros_like(y)
    if x is not None:
        u = np.abs(x) if post is None else np.abs(x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * post)
        term = np.abs(scale) * u * (1.0 if gate is None else np.abs(gate))
    size = term + (0.0 if residual is None else np.abs(residual))
    r = 1.0 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    return FP32 * size, FP32 * (size * r * (1.0 if pre is None else np.abs(pre)) + np.abs(h))


@pytest.mark.parametrize("dtype,wide", [("fp16", False), ("bf16", False), ("fp16", True), ("bf16", True)])
@pytest.mark.parametrize("T,D,post,gate,pre", [
    (1, 2048, True, "row", True), (1, 1, True, "row", True), (3, 7, True, "rows", True), (5, 8, False, "none", True), (2, 64, True, "none", False),
    (4, 129, False, "rows", False), (3, 1000, True, "rows", True), (2, 4100, True, "row", True), (7, 5120, True, "rows", True),
    (2, 8192, False, "none", True), (2, 8195, True, "rows", True), (1, 16384, True, "row", True), (2, 32768, True, "rows", True),
    (1, 32767, True, "row", True), (300, 512, True, "none", True), (2, 16391, True, "rows", True), (70, 4096, True, "row", True)])
def test_norm_values(dtype, wide, T, D, post, gate, pre):
    import torch
    cg = _cg()
    g = rng("norm", T, D, dtype, wide)
    rt = "fp32" if wide else dtype
    x, x64 = _rounded(g, dtype, T, D, scale=2.0)
    r, r64 = _rounded(g, rt, T, D, scale=3.0)
    wo, wo64 = _rounded(g, dtype, D) if post else (None, None)
    wi, wi64 = _rounded(g, dtype, D) if pre else (None, None)
    ga, ga64 = _rounded(g, dtype, *((T, D) if gate == "rows" else (D,))) if gate != "none" else (None, None)
    y, h = torch.full((T, D), 7.0, dtype=_dt(rt), device="cuda"), torch.full((T, D), 7.0, dtype=_dt(dtype), device="cuda")
    cg.block_norm(x, r, h, T, D, y_out=y, post_weight=wo, pre_weight=wi, gate=ga, scale=0.5, eps=1e-5)
    y64, h64 = ref.block_norm(x64, r64, wo64, ga64, 0.5, wi64, 1e-5)
    by, bh = _norm_bounds(x64, r64, wo64, ga64, 0.5, wi64, 1e-5, y64, h64)
    _close(y, y64, rt, by)
    _close(h, h64, dtype, bh)
    # parts left out
    h2, y2 = torch.empty_like(h), torch.empty_like(y)
    cg.block_norm(x, r, h2, T, D, post_weight=wo, pre_weight=wi, gate=ga, scale=0.5, eps=1e-5)
    cg.block_norm(x, r, None, T, D, y_out=y2, post_weight=wo, pre_weight=wi, gate=ga, scale=0.5, eps=1e-5)
    assert torch.equal(h, h2) and torch.equal(y, y2)
    # the residual stream alone, a copy of it, in any type
    y4 = torch.empty_like(y)
    cg.block_norm(None, r, None, T, D, y_out=y4)
    assert torch.equal(y4, r)
    # in place
    x3, r3 = x.clone(), r.clone()
    cg.block_norm(x3, r3, x3, T, D, y_out=r3, post_weight=wo, pre_weight=wi, gate=ga, scale=0.5, eps=1e-5)
    assert torch.equal(h, x3) and torch.equal(y, r3)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,pad,at", [(64, 8, 0), (100, 3, 1), (2050, 1, 5), (8192, 8, 8), (333, 0, 1)])
def test_norm_strides_and_absent_inputs(dtype, D, pad, at):
    import torch
    cg = _cg()
    T = 5
    g = rng("norm-strides", D, pad)
    wide, wide64 = _rounded(g, dtype, 3, T, D + pad + at)
    x, r, ga = (w[:, at:at + D] for w in wide)
    x64, r64, ga64 = (w[:, at:at + D] for w in wide64)
    both = torch.full((T, 2 * D + 5), 3.0, dtype=_dt(dtype), device="cuda")
    y, h = both[:, 1:1 + D], both[:, D + 3:2 * D + 3]  # rows of one tensor
    for args, plain in [(dict(x=x, residual=r, gate=ga), (x64, r64, ga64)), (dict(x=None, residual=r), (None, r64, None)),
                        (dict(x=x, residual=None, gate=ga), (x64, None, ga64))]:
        both.fill_(3.0)
        cg.block_norm(args["x"], args["residual"], h, T, D, y_out=y, gate=args.get("gate"), scale=1.5)
        px, pr, pg = plain
        y64, h64 = ref.block_norm(px, pr, None, pg, 1.5, None, 1e-6)
        by, bh = _norm_bounds(px, pr, None, pg, 1.5, None, 1e-6, y64, h64)
        _close(y, y64, dtype, by)
        _close(h, h64, dtype, bh)
        rest = torch.cat((both[:, :1], both[:, 1 + D:D + 3], both[:, 2 * D + 3:]), 1)
        assert bool((rest == 3.0).all())
    assert np.array_equal(_f64(wide), wide64)


def test_norm_rows_do_not_meet():
    """A row of zeros, of infinities or NaN and of the type's largest values changes no other."""
    import torch
    cg = _cg()
    T, D = 6, 200
    g = rng("norm-odd-rows")
    x, x64 = _rounded(g, "fp16", T, D)
    x[1], x[2, 7], x[3, 199], x[4] = 0.0, float("inf"), float("nan"), 65504.0
    x64 = _f64(x)
    w, w64 = _rounded(g, "fp16", D)
    r = torch.zeros(T, D, device="cuda")
    h, y = torch.empty_like(x), torch.empty_like(r)
    cg.block_norm(x, r, h, T, D, y_out=y, pre_weight=w)
    y64, h64 = ref.block_norm(x64, np.zeros((T, D)), None, None, 1.0, w64, 1e-6)
    keep = [0, 1, 4, 5]
    _close(y[keep], y64[keep], "fp32", 0.0)
    _close(h[keep], h64[keep], "fp16", FP32 * np.abs(h64[keep]))
    assert not bool(torch.isfinite(h[3]).any())
    # an infinite scale past the end of an odd row
    cg.block_norm(x[:1, :199].contiguous(), None, None, 1, 199, y_out=y[:1, :199].contiguous(), scale=float("inf"))


@pytest.mark.parametrize("T,D", [(3, 64), (5, 101)])
def test_norm_flat_gate(T, D):
    """A gate of one dimension as long as all rows is a row for each, not the first for all."""
    import torch
    cg = _cg()
    g = rng("norm-flat-gate", T, D)
    x, x64 = _rounded(g, "fp16", T, D)
    ga, ga64 = _rounded(g, "fp16", T, D)
    y, h = torch.empty_like(x), torch.empty_like(x)
    for gate, gate64 in ((ga.flatten(), ga64), (ga[1].clone(), ga64[1])):
        cg.block_norm(x, None, h, T, D, y_out=y, gate=gate)
        y64, h64 = ref.block_norm(x64, None, None, gate64, 1.0, None, 1e-6)
        by, bh = _norm_bounds(x64, None, None, gate64, 1.0, None, 1e-6, y64, h64)
        _close(y, y64, "fp16", by)
        _close(h, h64, "fp16", bh)


@pytest.mark.parametrize("dtype,stream", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp32")])
@pytest.mark.parametrize("T,D", [(3, 1), (2, 100), (2, 2048), (2, 8195), (1, 32768)])
@pytest.mark.parametrize("size,eps", [(1e20, 1e-6), (2e38, 1e-6), (1e25, 1e30), (1e-25, 0.0), (1e-38, 0.0), (1e-30, 1e-36), (1e-15, 1e-34)])
def test_norm_squares_that_leave_fp32(dtype, stream, T, D, size, eps):
    """Rows whose squares are infinite or nothing in fp32 have norms like all others.  Magnitudes are
    size / 48 to size / 1.5: the smallest at 1e-38, 2^-132, is not below bf16's least."""
    import torch
    cg = _cg()
    g = rng("norm-far", T, D, size)
    rt = torch.float32 if stream == "fp32" else _dt(dtype)
    v = torch.from_numpy(g.integers(64, 257, (2, T, D)) * g.choice([-1.0, 1.0], (2, T, D)) * 2.0 ** -g.integers(0, 4, (2, T, D)))
    v = v * (size / 1.5 / 256)
    r = v[0].to(rt).cuda()
    w, w64 = _rounded(g, dtype, D)
    y, h = torch.empty_like(r), torch.empty(T, D, dtype=_dt(dtype), device="cuda")
    cg.block_norm(None, r, h, T, D, y_out=y, pre_weight=w, eps=eps)
    y64, h64 = ref.block_norm(None, _f64(r), None, None, 1.0, w64, eps)
    assert torch.equal(y, r) and np.all(np.isfinite(h64))
    _close(h, h64, dtype, FP32 * np.abs(h64))
    if dtype == "bf16":  # and the block's output
        x = v[1].to(torch.bfloat16).cuda()
        cg.block_norm(x, None, h, T, D, y_out=y, post_weight=w, scale=0.5, eps=eps)
        y64, h64 = ref.block_norm(_f64(x), None, w64, None, 0.5, None, eps)
        by, bh = _norm_bounds(_f64(x), None, w64, None, 0.5, None, eps, y64, h64)
        _close(y, y64, stream, by)
        _close(h, h64, dtype, bh)


@pytest.mark.parametrize("D", [8, 199, 2049])
def test_norm_infinite_scale(D):
    """Every element is infinite, with its sign, or NaN where it was 0, and no norm is a number."""
    import torch
    cg = _cg()
    g = rng("norm-infinite", D)
    x, x64 = _rounded(g, "fp16", 3, D)
    x[1, D // 2] = 0.0
    x[2] = 0.0
    y, h = torch.empty(3, D, device="cuda"), torch.empty_like(x)
    cg.block_norm(x, torch.ones_like(y), h, 3, D, y_out=y, scale=float("inf"))
    y64, h64 = ref.block_norm(_f64(x), np.ones((3, D)), None, None, np.inf, None, 1e-6)
    assert np.isinf(y64[0]).all() and np.isnan(y64[2]).all() and np.isnan(h64).all()
    _close(y, y64, "fp32", 0.0)
    _close(h, h64, "fp16", 0.0)


# ---- moe_route ----------------------------------------------------------------

def _route(cg, x, bias, k, E=None, **kw):
    import torch
    T = x.shape[0]
    ids = torch.full((T, k), 77, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), 7.0, device="cuda")
    cg.moe_route(x, ids, w, T, x.shape[1] if E is None else E, k, bias=bias, **kw)
    return ids, w


def _check_route(x, bias, got, k, score, groups=1, top_groups=1, group_top=1, renormalize=False, scale=1.0):
    ids, w = got
    want, w64 = ref.route(_f64(x), None if bias is None else _f64(bias), score, groups, top_groups, group_top, k, renormalize, scale)
    assert np.array_equal(ids.cpu().numpy(), want)
    _close(w, w64, "fp32", 1e-12 * np.abs(w64) + 1e-45)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,E,k,groups,top_groups,group_top,biased", [
    (1, 1, 1, 1, 1, 1, False), (1, 8, 2, 1, 1, 1, False), (9, 8, 8, 1, 1, 1, True), (5, 7, 3, 1, 1, 1, True), (33, 64, 6, 1, 1, 1, False),
    (17, 60, 4, 1, 1, 1, False), (12, 65, 9, 5, 2, 2, True), (40, 128, 8, 8, 3, 1, False), (21, 160, 6, 8, 3, 2, False), (50, 256, 8, 8, 4, 2, True),
    (3, 384, 12, 1, 1, 1, True), (4, 1024, 64, 64, 32, 2, True), (2, 1000, 10, 8, 8, 1, False), (3, 64, 64, 64, 64, 1, True), (300, 16, 4, 4, 2, 2, True),
    (5, 513, 5, 27, 4, 2, False), (130, 32, 1, 2, 1, 1, True)])
def test_route_values(score, dtype, T, E, k, groups, top_groups, group_top, biased):
    cg = _cg()
    g = rng("route", T, E, k, score)
    x, _ = _rounded(g, dtype, T, E, scale=2.0)
    bias = _dev((g.standard_normal(E) * 0.2).astype(np.float32)) if biased else None
    for renorm, scale in [(False, 1.0), (True, 2.5)]:
        how = dict(groups=groups, top_groups=top_groups, group_top=group_top, renormalize=renorm, scale=scale)
        got = _route(cg, x, bias, k, score=getattr(cg, "CLOVE_ROUTE_" + score.upper()), **how)
        _check_route(x, bias, got, k, score, **how)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased,groups", [(False, 1), (True, 1), (False, 4), (True, 4)])
def test_route_ties_and_masks(score, biased, groups):
    """Equal values, -inf, +inf and NaN logits, rows with few experts left or none, values
    far from each other (scores that underflow)."""
    cg = _cg()
    E, k = 48, 6
    g = rng("route-ties", score, biased, groups)
    x = np.round(g.standard_normal((14, E)) * 2).astype(np.float32)  # many equal
    x[1] = 0.0
    x[2] = -np.inf
    x[3, 5:] = -np.inf
    x[4, ::2] = np.nan
    x[5] = np.nan
    x[6, 7], x[6, 30] = np.inf, np.inf
    x[7] = np.where(np.arange(E) % 5 == 0, x[7], -np.inf)
    x[8] = np.linspace(-2000, 2000, E)
    x[9] = np.linspace(100, -200, E)
    x[10] = -np.arange(E)[::-1] * 40.0
    x[11, 1:] = -np.inf
    x[12] = 1e30
    x[13] = -3.0e38
    bias = None
    if biased:
        b = np.round(g.standard_normal(E) * 4).astype(np.float32) / 8
        b[3], b[9], b[20] = -np.inf, np.nan, np.inf
        bias = _dev(b)
    t = _dev(x)
    for renorm in (False, True):
        how = dict(groups=groups, top_groups=2 if groups > 1 else 1, group_top=2 if groups > 1 else 1, renormalize=renorm)
        got = _route(cg, t, bias, k, score=getattr(cg, "CLOVE_ROUTE_" + score.upper()), **how)
        _check_route(t, bias, got, k, score, **how)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_values_that_nearly_agree(score):
    """Scores plus bias one part in 2^30 apart: 32 bits cannot tell them, 64 can."""
    cg = _cg()
    T, E, k = 64, 64, 8
    g = rng("route-near", score)
    x = g.standard_normal((T, E)).astype(np.float32)
    x[:, 32:] = x[:, :32] + (g.integers(-2, 3, (T, 32)) * 2.0 ** -22).astype(np.float32)
    b = np.zeros(E, np.float32)
    b[::2], b[1::2] = 2.0 ** -40, -2.0 ** -40
    got = _route(cg, _dev(x), _dev(b), k, score=getattr(cg, "CLOVE_ROUTE_" + score.upper()))
    _check_route(_dev(x), _dev(b), got, k, score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(48, 4), (16, 8), (64, 2), (256, 8)])
def test_route_biases_of_the_lowest_value(score, E, groups):
    """Experts masked by fp32's lowest value, whose sum over two leaves fp32: they come after
    the others, but before none, and whole groups of them too."""
    cg = _cg()
    k, n = 6, E // groups
    g = rng("route-lowest", score, E, groups)
    x = _dev(g.standard_normal((9, E)).astype(np.float32))
    low = np.finfo(np.float32).min
    for masked in (np.arange(E) >= n, np.arange(E) % n != 0, np.arange(E) >= 0, np.arange(E) < n):
        b = np.where(masked, low, (g.standard_normal(E) * 0.2)).astype(np.float32)
        for top_groups in (1, 2, groups):
            how = dict(groups=groups, top_groups=top_groups, group_top=2)
            got = _route(cg, x, _dev(b), k, score=getattr(cg, "CLOVE_ROUTE_" + score.upper()), **how)
            _check_route(x, _dev(b), got, k, score, **how)


def test_route_rows_of_wider_tensors():
    cg = _cg()
    g = rng("route-wide")
    wide, _ = _rounded(g, "fp16", 9, 101)
    x = wide[:, 3:3 + 60]
    _check_route(x, None, _route(cg, x, None, 4), 4, "softmax")


# ---- the experts' products ------------------------------------------------------

def _ids(g, T, k, E, absent=0.0, distinct=True):
    ids = np.stack([g.permutation(E)[:k] if distinct and k <= E else g.integers(0, E, k) for _ in range(T)]).astype(np.int32)
    if absent:
        ids[g.random((T, k)) < absent] = -1
    return ids


class Case:
    def __init__(self, key, T, k, E, R, K, absent=0.0, distinct=True, offset=0, whole=True):
        import torch
        g = self.g = rng("moe", key, T, k, E, R, K)
        self.T, self.k, self.E, self.R, self.K = T, k, E, R, K
        G = -(-K // ref.GROUP)
        self.ids = _ids(g, T, k, E, absent, distinct)
        q = g.integers(0, 256, (E, R, K // 2)).astype(np.uint8)
        s = g.uniform(0.5, 1.5, (E, R, G)).astype(np.float16) / np.float16(max(1.0, 4.6 * K ** 0.5))
        z = g.integers(0, 16, (E, R, G)).astype(np.float16)
        if not whole:
            z = (z + g.uniform(-0.4, 0.4, z.shape)).astype(np.float16)  # rounded to whole numbers by the call
        self.w = ref.dequantized(q, s, z, K)
        def shifted(x, by):  # the same values, `by` elements into an allocation
            t = _dev(x)
            flat = torch.zeros(x.size + by, dtype=t.dtype, device="cuda")
            flat[by:] = t.flatten()
            return flat[by:].view(*x.shape)

        odd = 1 if offset else 0  # (scales and zero points off a dword's start, not by as much)
        self.q, self.s, self.z = shifted(q, offset), shifted(s, odd), shifted(z, 3 * odd)
        self.dev_ids = shifted(self.ids, odd)
        self.slack = (256 + 2 * G + 64) * 2.0 ** -24


def _up(cg, c, x, h):
    cg.moe_w4a16_swiglu(x, c.dev_ids, c.q, c.s, c.z, h, c.T, c.k, c.E, c.R // 2, c.K)


def _check_up(cg, c, x=None):
    import torch
    if x is None:
        x, _ = _rounded(c.g, "fp16", c.T, c.K)
    h = torch.full((c.T * c.k, c.R // 2), 5.0, dtype=torch.float16, device="cuda")
    want, size = ref.swiglu_up(_f64(x), c.ids, c.w, _f64(h))
    _up(cg, c, x, h)
    _close(h, want, "fp16", c.slack * size)
    again = torch.full_like(h, 5.0)
    _up(cg, c, x, again)
    assert torch.equal(h.view(torch.int16), again.view(torch.int16))
    return h, want


def _check_down(cg, c, beta=1.0, alpha=1.0, weighted=True):
    import torch
    h, h64 = _rounded(c.g, "fp16", c.T * c.k, c.K)
    w = _dev(c.g.uniform(-0.5, 1.0, (c.T, c.k)).astype(np.float32)) if weighted else None
    y0, y64 = _rounded(c.g, "fp16", c.T, c.R)
    if beta == 0.0:
        y0.fill_(float("nan"))  # never read
    want, size = ref.down(h64, c.ids, None if w is None else _f64(w), c.w, y64, alpha, beta)
    y = y0.clone()
    cg.moe_w4a16(h, c.dev_ids, w, c.q, c.s, c.z, y, c.T, c.k, c.E, c.R, c.K, alpha=alpha, beta=beta)
    _close(y, want, "fp16", c.slack * size)
    again = y0.clone()
    cg.moe_w4a16(h, c.dev_ids, w, c.q, c.s, c.z, again, c.T, c.k, c.E, c.R, c.K, alpha=alpha, beta=beta)
    assert torch.equal(y, again)
    return y, want


# T, top_k, experts, outputs, K
SIZES = [(1, 1, 1, 1, 2), (1, 2, 4, 3, 128), (1, 8, 128, 64, 256), (1, 8, 16, 768, 1024), (2, 4, 8, 100, 160), (3, 2, 4, 33, 130), (5, 8, 16, 64, 256),
         (4, 2, 8, 48, 2048), (16, 2, 64, 80, 512), (33, 1, 2, 40, 96), (70, 3, 5, 100, 384), (130, 6, 64, 96, 192), (257, 4, 3, 48, 160),
         (40, 8, 8, 130, 1024), (600, 2, 2, 64, 256), (64, 4, 4, 513, 640), (300, 1, 9, 256, 128), (100, 8, 256, 64, 256), (1, 1, 3, 16, 14336),
         (20, 64, 64, 32, 128), (512, 2, 4, 320, 544), (7, 3, 4, 31, 62), (2, 2, 4, 40, 32), (50, 2, 4, 40, 32), (400, 2, 4, 40, 32), (1100, 2, 8, 128, 256), (150, 2, 1024, 16, 64)]


@pytest.mark.parametrize("T,k,E,O,K", SIZES)
def test_up_values(T, k, E, O, K):
    c = Case("up", T, k, E, 2 * O, K, absent=0.1 if T > 2 else 0.0)
    got, want = _check_up(_cg(), c)
    if K <= 1024 and got.numel() > 2000:
        # one rounding only: an fp32 sum off by some 2^-20 moves few of them over a boundary
        assert np.mean(_f64(got) == want.astype(np.float16).astype(np.float64)) > 0.97


@pytest.mark.parametrize("T,k,E,O,K", SIZES)
@pytest.mark.parametrize("beta,alpha,weighted", [(1.0, 1.0, True), (0.0, 0.5, False)])
def test_down_values(T, k, E, O, K, beta, alpha, weighted):
    c = Case("down", T, k, E, O, K, absent=0.1 if T > 2 else 0.0)
    got, want = _check_down(_cg(), c, beta, alpha, weighted)
    if K <= 1024 and got.numel() > 2000:
        assert np.mean(_f64(got) == want.astype(np.float16).astype(np.float64)) > 0.97


# few tiles and a long K: the products go in parts of K (of 2 to 8, the last one shorter)
@pytest.mark.parametrize("T,k,E,O,K", [(14, 7, 8, 128, 8192), (20, 2, 4, 200, 4096), (21, 2, 8, 1023, 8192), (13, 3, 4, 61, 4000), (300, 2, 8, 96, 2080),
                                       (9, 3, 8, 70, 10880), (90, 12, 16, 130, 3136)])
def test_parts_of_k(T, k, E, O, K):
    cg = _cg()
    for absent in (0.0, 0.2):
        _check_up(cg, Case("up-parts", T, k, E, 2 * O, K, absent=absent))
        _check_down(cg, Case("down-parts", T, k, E, O, K, absent=absent))
        _check_down(cg, Case("down-parts-0", T, k, E, O, K, absent=absent), beta=0.0, alpha=-1.5, weighted=False)


@pytest.mark.parametrize("T", [1, 3, 40, 300])
@pytest.mark.parametrize("offset,K", [(1, 128), (4, 256), (8, 96), (16, 256), (2, 66)])
def test_weights_at_any_alignment(T, offset, K):
    cg = _cg()
    _check_up(cg, Case("up-offset", T, 2, 5, 2 * 40, K, offset=offset, whole=False))
    _check_down(cg, Case("down-offset", T, 2, 5, 72, K, offset=offset, whole=False))


@pytest.mark.parametrize("T", [1, 2, 20, 200])
def test_the_same_expert_twice_and_ids_that_are_none(T):
    import torch
    cg = _cg()
    for key in ("up", "down"):
        c = Case("odd-ids", T, 4, 3, 96, 256, distinct=False)
        c.ids[:, 1] = c.ids[:, 0]
        c.ids[T // 2, 2:] = [3, 2 ** 31 - 1]
        c.ids[0, 3] = -2 ** 31
        c.ids[T - 1] = -1  # a token without experts
        c.dev_ids = torch.from_numpy(c.ids).cuda()
        _check_up(cg, c) if key == "up" else _check_down(cg, c)
    c.ids[:] = -1
    c.dev_ids = torch.from_numpy(c.ids).cuda()
    _check_up(cg, c)
    _check_down(cg, c)
    _check_down(cg, c, beta=0.0)


@pytest.mark.parametrize("T,k,E", [(9, 2, 64), (40, 8, 128), (70, 4, 16), (300, 2, 16)])
def test_all_pairs_of_one_expert(T, k, E):
    """The shapes are those of many experts hit, the pairs all the last one's, but for one of the first's."""
    import torch
    cg = _cg()
    for key in ("up", "down"):
        c = Case("one-" + key, T, k, E, 64, 128)
        c.ids[:] = E - 1
        c.ids[T // 2, 0] = 0
        c.dev_ids = torch.from_numpy(c.ids).cuda()
        _check_up(cg, c) if key == "up" else _check_down(cg, c)


@pytest.mark.parametrize("T,E", [(1, 4), (6, 4), (80, 4), (300, 2)])
def test_rows_do_not_meet(T, E):
    """NaN and infinities stay in their token's rows, and what no expert reads is not used."""
    import torch
    cg = _cg()
    k, K, O = 2, 256, 48
    c = Case("nan", T, k, E, 2 * O, K)
    c.ids[0, 1] = -1
    c.dev_ids = torch.from_numpy(c.ids).cuda()
    x, _ = _rounded(c.g, "fp16", T, K)
    if T > 1:
        x[T // 2, 3], x[T - 1, 0] = float("nan"), float("inf")
    h = torch.full((T * k, O), 5.0, dtype=torch.float16, device="cuda")
    _up(cg, c, x, h)
    want, size = ref.swiglu_up(_f64(x), c.ids, c.w, np.full((T * k, O), 5.0))
    rows = [p for p in range(T * k) if T == 1 or p // k not in (T // 2, T - 1)]
    _close(h[rows], want[rows], "fp16", c.slack * size[rows])
    if T > 1:
        assert bool(torch.isnan(h[T // 2 * k:T // 2 * k + k]).all())
    d = Case("nan-down", T, k, E, O, K)
    d.ids[0, 1] = -1
    d.dev_ids = torch.from_numpy(d.ids).cuda()
    hin, _ = _rounded(d.g, "fp16", T * k, K)
    w = torch.rand(T, k, device="cuda")
    hin[1], w[0, 1] = float("nan"), float("nan")  # a pair without a product
    if T > 1:
        hin[(T // 2) * k + 1, 5] = float("inf")
    y = torch.zeros(T, O, dtype=torch.float16, device="cuda")
    cg.moe_w4a16(hin, d.dev_ids, w, d.q, d.s, d.z, y, T, k, E, O, K)
    clean = torch.where(torch.isfinite(hin), hin, 0.0)
    want, size = ref.down(_f64(clean), d.ids, np.nan_to_num(_f64(w)), d.w, np.zeros((T, O)), 1.0, 0.0)
    rows = [t for t in range(T) if T == 1 or t != T // 2]
    _close(y[rows], want[rows], "fp16", d.slack * size[rows])
    if T > 1:
        assert not bool(torch.isfinite(y[T // 2]).all())


@pytest.mark.parametrize("T,k,E,O,K", [(1, 2, 4, 48, 512), (3, 2, 64, 48, 512), (6, 2, 4, 48, 512), (30, 2, 4, 80, 768), (200, 2, 4, 80, 768),
                                       (700, 2, 4, 200, 512), (3, 2, 4, 33, 322)])
def test_scales_of_any_size_and_sign(T, k, E, O, K):
    """Groups with a scale of 0, of either sign, subnormal or large, one after another: the
    accumulators' unit changes by up to 2^34 from a group to the next, and back."""
    import torch
    cg = _cg()
    for key in ("up", "down"):
        c = Case("scales-" + key, T, k, E, 2 * O if key == "up" else O, K)
        g = c.g
        s = (g.choice([0.0, -0.0, 1.0, -1.0, 2.0 ** -24, -(2.0 ** -20), 0.37, 3.0, 0.01], c.s.shape) * 0.05).astype(np.float16)
        s[:, 0] = 0.0  # a row of nothing
        s[:, 1:, -1] = np.where(g.random(s[:, 1:, -1].shape) < 0.5, 0.0, s[:, 1:, -1])
        q, z = c.q.cpu().numpy(), c.z.cpu().numpy()
        c.w, c.s = ref.dequantized(q, s, z, K), _dev(s)
        if key == "up":
            _check_up(cg, c)
        else:
            _check_down(cg, c)


def test_infinite_and_nan_scales_stay_in_their_row():
    import torch
    cg = _cg()
    for T in (1, 40, 300):
        c = Case("bad-scales", T, 2, 4, 64, 384)
        c.s[:, 5, 1], c.s[:, 9, 2] = float("inf"), float("nan")
        h, _ = _rounded(c.g, "fp16", T * 2, 384)
        y = torch.zeros(T, 64, dtype=torch.float16, device="cuda")
        cg.moe_w4a16(h, c.dev_ids, None, c.q, c.s, c.z, y, T, 2, 4, 64, 384)
        want, size = ref.down(_f64(h), c.ids, None, c.w, np.zeros((T, 64)), 1.0, 0.0)
        rows = [r for r in range(64) if r not in (5, 9)]
        _close(y[:, rows], want[:, rows], "fp16", c.slack * size[:, rows])
        assert not bool(torch.isfinite(y[:, [5, 9]]).any())


def _device_products(x, w):
    """x [n, K] by each w [E, R, K], all in 64 bits on the device: [E, n, R]."""
    import torch
    return torch.stack([x @ e.T.contiguous() for e in torch.from_numpy(w).cuda()])


@pytest.mark.parametrize("T,k,E,O,K", [(70001, 8, 4, 32, 64), (150001, 2, 2, 16, 4096)])
def test_more_pairs_than_one_part_takes(T, k, E, O, K):
    """More than 2^19 pairs, and rows of X past 2^31 bytes: parts of the tokens one after another."""
    import torch
    cg = _cg()
    g = torch.Generator(device="cuda").manual_seed(T)
    ids = torch.randint(-1, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    part = slice(T // 2 - 100, T // 2 + 200)  # (where the parts meet) and both ends
    c = Case("parts", 1, k, E, 2 * O, K)
    x = torch.empty(T, K, dtype=torch.float16, device="cuda").normal_(generator=g)
    h = torch.full((T * k, O), 5.0, dtype=torch.float16, device="cuda")
    cg.moe_w4a16_swiglu(x, ids, c.q, c.s, c.z, h, T, k, E, O, K)
    for rows in (slice(0, 50), part, slice(T - 50, T)):
        y = _device_products(x[rows].double(), c.w)
        gate, up = y[..., :O], y[..., O:]
        want = (gate * torch.sigmoid(gate) * up)[ids[rows].clamp(min=0).long().T, torch.arange(y.shape[1], device="cuda")]
        want = torch.where(ids[rows].T[..., None] >= 0, want, 5.0).transpose(0, 1)
        got = h.view(T, k, O)[rows].double()
        assert float((got - want).abs().max()) <= 2.0 ** -11 * float(want.abs().max()) * 1.01 + 1e-4
    d = Case("parts-down", 1, k, E, O, K)
    hin = torch.empty(T * k, K, dtype=torch.float16, device="cuda").normal_(generator=g)
    w = torch.rand(T, k, generator=g, device="cuda")
    out = torch.empty(T, O, dtype=torch.float16, device="cuda")
    cg.moe_w4a16(hin, ids, w, d.q, d.s, d.z, out, T, k, E, O, K)
    for rows in (slice(0, 50), part, slice(T - 50, T)):
        n = rows.stop - rows.start
        y = _device_products(hin.view(T, k, K)[rows].reshape(n * k, K).double(), d.w).view(E, n, k, O)
        y = y.permute(1, 2, 0, 3).gather(2, ids[rows].clamp(min=0).long()[:, :, None, None].expand(n, k, 1, O))[:, :, 0]
        want = (torch.where(ids[rows][..., None] >= 0, y, 0.0) * w[rows].double()[..., None]).sum(1)
        assert float((out[rows].double() - want).abs().max()) <= 2.0 ** -11 * float(want.abs().max()) * 1.01 + 1e-4


def test_parts_share_one_plan():
    """65537 tokens go in parts of 32769 and 32768, and the second's products alone would come
    with twice as many outputs at a time: the call needs what its first part needs, no more."""
    import torch
    cg = _cg()
    T, k, E, O, K = 65537, 8, 2, 512, 32
    c = Case("plan", 1, k, E, O, K)
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    h = torch.empty(T * k, K, dtype=torch.float16, device="cuda").normal_(generator=g)
    y = torch.zeros(T, O, dtype=torch.float16, device="cuda")

    def down(n):
        cg.moe_w4a16(h[:n * k], ids[:n], None, c.q, c.s, c.z, y[:n], n, k, E, O, K)

    need = []
    for n in (32769, T):
        with cg.workspace_query() as q:
            down(n)
        need.append(q.bytes)
    assert need[0] == need[1] < 2 ** 29
    down(T)
    want = y.clone()
    cg.workspace_bind(torch.zeros(need[1], dtype=torch.uint8, device="cuda"))
    try:
        y.zero_()
        down(T)
    finally:
        cg.workspace_bind(None)
    assert torch.equal(y, want)
    products = _device_products(h[-80:].double(), c.w)[ids[-10:].flatten().long(), torch.arange(80, device="cuda")]
    exact = products.view(10, k, O).sum(1)
    assert float((y[-10:].double() - exact).abs().max()) <= 2.0 ** -11 * float(exact.abs().max()) * 1.01 + 1e-4


def test_rows_past_one_launch():
    """More rows than a launch of the norm, and of the router, counts threads for."""
    import torch
    cg = _cg()
    T, D = 2 ** 31 // 64 + 3, 8
    x = torch.empty(T, D, dtype=torch.float16, device="cuda").normal_()
    h = torch.empty_like(x)
    cg.block_norm(None, x, h, T, D)
    for rows in (slice(0, 5), slice(T - 8, T)):
        _, want = ref.block_norm(None, _f64(x[rows]), None, None, 1.0, None, 1e-6)
        _close(h[rows], want, "fp16", FP32 * np.abs(want))
    T, E = 2 ** 25 + 5, 4
    x = x.flatten()[:T * E].view(T, E)
    ids, w = _route(cg, x, None, 1)
    assert bool((ids[:, 0] == x.float().argmax(1)).all())
    _check_route(x[-9:], None, (ids[-9:], w[-9:]), 1, "softmax")


@pytest.mark.parametrize("K,T", [(32, 550), (32, 384), (2, 1)])
def test_more_workgroups_than_one_launch_counts(K, T):
    """1024 experts of 2 x 262400 rows: 2^32 threads are less than the outputs call for."""
    import torch
    cg = _cg()
    k, E, I = 2, 1024, 262400
    R = 2 * I
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.empty(E, R, K // 2, dtype=torch.uint8, device="cuda")
    for e in range(0, E, 64):
        q[e:e + 64] = torch.randint(0, 256, (64, R, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s, z = torch.full((E, R, 1), 2.0 ** -6, dtype=torch.float16, device="cuda"), torch.full((E, R, 1), 8.0, dtype=torch.float16, device="cuda")
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randint(-4, 5, (T * k, K), generator=g, device="cuda").half()
    h, y = torch.full((T * k, I), 5.0, dtype=torch.float16, device="cuda"), torch.full((T, R), 5.0, dtype=torch.float16, device="cuda")
    cg.moe_w4a16_swiglu(x[:T], ids, q, s, z, h, T, k, E, I, K)
    cg.moe_w4a16(x, ids, None, q, s, z, y, T, k, E, R, K)
    for t in sorted({0, T // 2, T - 1}):
        want = 0.0
        for j in range(k):
            b = q[int(ids[t, j])]
            w = (torch.stack([b // 16, b % 16], -1).view(R, K).double() - 8) / 64
            gate, up = (w @ x[t].double()).view(2, I)
            v = gate * torch.sigmoid(gate) * up
            assert bool(((h[t * k + j].double() - v).abs() <= 2.0 ** -11 * v.abs() + 2.0 ** -18 * (1 + v.abs())).all())
            want = want + w @ x[t * k + j].double()
        assert torch.equal(y[t].double(), want.half().double())  # (exact in fp32)


def test_outputs_past_one_grid():
    """More outputs of one pair than a launch's second dimension counts in blocks of 512."""
    import torch
    cg = _cg()
    O = 512 * 65535 + 700
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randint(0, 256, (1, O, 1), generator=g, device="cuda", dtype=torch.uint8)
    one = torch.ones(1, O, 1, dtype=torch.float16, device="cuda")
    y = torch.full((1, O), 7.0, dtype=torch.float16, device="cuda")
    x = torch.tensor([[2.0, 3.0]], dtype=torch.float16, device="cuda")
    cg.moe_w4a16(x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), None, q, one, one * 8, y, 1, 1, 1, O, 2)
    byte = q.view(-1).to(torch.int16)
    want = 2 * (byte // 16 - 8) + 3 * (byte % 16 - 8)  # whole numbers: exact
    assert bool((y.view(-1) == want).all())


@pytest.mark.parametrize("T,k,E,O,K", [(3, 6, 31, 469, 2), (1, 4, 4, 1, 2), (5, 64, 100, 20, 30), (2, 64, 80, 33, 8), (9, 20, 32, 40, 2), (40, 64, 3, 24, 4)])
def test_more_places_than_columns(T, k, E, O, K):
    cg = _cg()
    _check_up(cg, Case("places-up", T, k, E, 2 * O, K, absent=0.1))
    _check_down(cg, Case("places-down", T, k, E, O, K, absent=0.1))


@pytest.mark.parametrize("O,K", [(40, 0), (5, 0)])
def test_no_k(O, K):
    import torch
    cg = _cg()
    T, k, E = 3, 2, 4
    ids = torch.tensor([[0, 1], [2, -1], [3, 3]], dtype=torch.int32, device="cuda")
    none, half = torch.empty(0, dtype=torch.uint8, device="cuda"), torch.empty(0, dtype=torch.float16, device="cuda")
    h = torch.full((T * k, O), 5.0, dtype=torch.float16, device="cuda")
    cg.moe_w4a16_swiglu(half, ids, none, half, half, h, T, k, E, O, K)
    assert bool((h[[0, 1, 2, 4, 5]] == 0).all()) and bool((h[3] == 5).all())
    y = torch.full((T, O), 3.0, dtype=torch.float16, device="cuda")
    cg.moe_w4a16(half, ids, None, none, half, half, y, T, k, E, O, K, beta=2.0)
    assert bool((y == 6).all())


@pytest.mark.parametrize("T", [1, 50])
def test_experts_past_four_gigabytes(T):
    """The last of 1024 experts lies past 2^32 bytes of weights."""
    import torch
    cg = _cg()
    E, R, K, k = 1024, 4096, 2304, 1
    q = torch.zeros(E, R, K // 2, dtype=torch.uint8, device="cuda")
    s, z = torch.ones(E, R, K // 128, dtype=torch.float16, device="cuda"), torch.zeros(E, R, K // 128, dtype=torch.float16, device="cuda")
    g = rng("far", T)
    last = g.integers(0, 256, (R, K // 2)).astype(np.uint8)
    q[-1] = _dev(last)
    s[-1] = 2.0 ** -9
    ids = torch.full((T, k), E - 1, dtype=torch.int32, device="cuda")
    x, x64 = _rounded(g, "fp16", T, K)
    w = ref.dequantized(last, np.full((R, K // 128), 2.0 ** -9), np.zeros((R, K // 128)), K)[None]
    zeros = np.zeros((T, k), np.int32)
    slack = (256 + 2 * 18 + 64) * 2.0 ** -24
    h = torch.zeros(T, R // 2, dtype=torch.float16, device="cuda")
    cg.moe_w4a16_swiglu(x, ids, q, s, z, h, T, k, E, R // 2, K)
    want, size = ref.swiglu_up(x64, zeros, w, np.zeros((T, R // 2)))
    ok = np.abs(want) < 65000
    _close(h[torch.from_numpy(ok).cuda()], want[ok], "fp16", (slack * size)[ok])
    y = torch.zeros(T, R, dtype=torch.float16, device="cuda")
    cg.moe_w4a16(x, ids, None, q, s, z, y, T, k, E, R, K)
    want, size = ref.down(x64, zeros, None, w, np.zeros((T, R)), 1.0, 0.0)
    _close(y, want, "fp16", slack * size)


# ---- workspaces, graphs, streams, the block as a whole ----------------------------

@pytest.mark.parametrize("T,K", [(1, 256), (4, 256), (40, 256), (400, 256), (20, 6144)])
def test_bound_workspace_and_its_size(T, K):
    import torch
    cg = _cg()
    c = Case("workspace", T, 4, 8, 128, K)
    x, _ = _rounded(c.g, "fp16", T, K)
    hin, _ = _rounded(c.g, "fp16", T * 4, K)
    w = torch.rand(T, 4, device="cuda")
    h, y = torch.zeros(T * 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(T, 128, dtype=torch.float16, device="cuda")

    def calls():
        _up(cg, c, x, h)
        cg.moe_w4a16(hin, c.dev_ids, w, c.q, c.s, c.z, y, T, 4, 8, 128, K)
        return h.clone(), y.clone()

    want = calls()
    h.zero_(), y.zero_()
    with cg.workspace_query() as q:
        calls()
    torch.cuda.synchronize()
    assert not bool(h.any()) and not bool(y.any())  # only planned
    if q.bytes == 0:
        return
    ws = torch.zeros(q.bytes, dtype=torch.uint8, device="cuda")
    cg.workspace_bind(ws)
    try:
        got = calls()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert not bool(ws[:cg.CLOVE_WORKSPACE_MIN_BYTES].any())
        cg.workspace_bind(ws[:cg.CLOVE_WORKSPACE_MIN_BYTES])
        h.fill_(3.0), y.fill_(3.0)
        with pytest.raises(cg.CloveError) as e:
            for call in (lambda: _up(cg, c, x, h), lambda: cg.moe_w4a16(hin, c.dev_ids, w, c.q, c.s, c.z, y, T, 4, 8, 128, K)):
                call()
        assert e.value.status == cg.CLOVE_ERR_WORKSPACE
    finally:
        cg.workspace_bind()


class Block:
    """norm, router, experts and the norm after them, as a decoder's sparse MLP block calls them."""

    def __init__(self, T, hidden=256, inter=192, E=16, k=4, seed=0):
        import torch
        g = self.g = rng("block", T, seed)
        self.T, self.D, self.I, self.E, self.k = T, hidden, inter, E, k
        self.up, self.down = Case(("block-up", seed), T, k, E, 2 * inter, hidden), Case(("block-down", seed), T, k, E, hidden, inter)
        self.router, self.router64 = _rounded(g, "fp16", hidden, E, scale=hidden ** -0.5)
        self.pre, self.pre64 = _rounded(g, "fp16", hidden)
        self.post, self.post64 = _rounded(g, "fp16", hidden)
        self.next, self.next64 = _rounded(g, "fp16", hidden)
        self.residual, _ = _rounded(g, "fp32", T, hidden, scale=2.0)
        half = dict(dtype=torch.float16, device="cuda")
        self.x, self.y = torch.empty(T, hidden, **half), torch.empty(T, hidden, **half)
        self.logits, self.h = torch.empty(T, E, **half), torch.zeros(T * k, inter, **half)
        self.ids, self.w = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
        self.stream, self.out = torch.empty_like(self.residual), torch.empty_like(self.x)

    def __call__(self):
        cg, T, D = _cg(), self.T, self.D
        cg.block_norm(None, self.residual, self.x, T, D, pre_weight=self.pre)
        cg.gemm_fp16(self.x, self.router, self.logits, T, self.E, D)
        cg.moe_route(self.logits, self.ids, self.w, T, self.E, self.k, renormalize=True)
        u, d = self.up, self.down
        cg.moe_w4a16_swiglu(self.x, self.ids, u.q, u.s, u.z, self.h, T, self.k, self.E, self.I, D)
        cg.moe_w4a16(self.h, self.ids, self.w, d.q, d.s, d.z, self.y, T, self.k, self.E, D, self.I)
        cg.block_norm(self.y, self.residual, self.out, T, D, y_out=self.stream, post_weight=self.post, pre_weight=self.next, scale=0.7)
        return [t.clone() for t in (self.x, self.ids, self.w, self.h, self.y, self.stream, self.out)]

    def check(self):
        """Each operator against its definition on what it was given."""
        r, x = _f64(self.residual), _f64(self.x)
        zero, x64 = ref.block_norm(None, r, None, None, 1.0, self.pre64, 1e-6)
        _close(self.x, x64, "fp16", _norm_bounds(None, r, None, None, 1.0, self.pre64, 1e-6, zero, x64)[1])
        _check_route(self.logits, None, (self.ids, self.w), self.k, "softmax", renormalize=True)
        ids = self.ids.cpu().numpy()
        h64, size = ref.swiglu_up(x, ids, self.up.w, np.zeros(self.h.shape))
        _close(self.h, h64, "fp16", self.up.slack * size)
        y64, size = ref.down(_f64(self.h), ids, _f64(self.w), self.down.w, np.zeros(self.y.shape), 1.0, 0.0)
        _close(self.y, y64, "fp16", self.down.slack * size)
        s64, o64 = ref.block_norm(_f64(self.y), r, self.post64, None, 0.7, self.next64, 1e-6)
        by, bh = _norm_bounds(_f64(self.y), r, self.post64, None, 0.7, self.next64, 1e-6, s64, o64)
        _close(self.stream, s64, "fp32", by)
        _close(self.out, o64, "fp16", bh)


@pytest.mark.parametrize("T", [1, 3, 24, 200])
def test_block(T):
    block = Block(T)
    block()
    block.check()


def _bits(ts):
    return [t.cpu().numpy().tobytes() for t in ts]


@pytest.mark.parametrize("T", [1, 24, 200])
def test_block_in_a_graph(T):
    """Replays with other inputs, eager work between them, two graphs of one stream."""
    import torch
    blocks = [Block(T, seed=s) for s in (0, 1)]
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        for b in blocks:
            b()  # (scratch of this stream)
        side.synchronize()
        for b in blocks:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                b()
            graphs.append(graph)
    torch.cuda.synchronize()
    for i in range(4):
        for b, graph in zip(blocks, graphs):
            b.residual.copy_(torch.randn_like(b.residual))
            want = _bits(b())
            for t in (b.x, b.h, b.y, b.stream, b.out, b.ids):
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert _bits((b.x, b.ids, b.w, b.h, b.y, b.stream, b.out)) == want, i
            b.check()


def test_parts_of_k_in_a_graph():
    """Parts of K and their sums, replayed with other ids and rows, eager calls of other sizes between."""
    import torch
    cg = _cg()
    T, k, E, O, K = 20, 4, 8, 64, 6144
    c = Case("graph-parts", T, k, E, 2 * O, K)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.empty(T * k, K, dtype=torch.float16, device="cuda")
    ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    h, y = torch.zeros(T * k, O, dtype=torch.float16, device="cuda"), torch.zeros(T, 2 * O, dtype=torch.float16, device="cuda")

    def calls(n=T):
        cg.moe_w4a16_swiglu(x[:n], ids[:n], c.q, c.s, c.z, h[:n * k], n, k, E, O, K)
        cg.moe_w4a16(x[:n * k], ids[:n], None, c.q, c.s, c.z, y[:n], n, k, E, 2 * O, K)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls()
    torch.cuda.synchronize()
    for i in range(4):
        x.normal_(generator=g)
        ids.copy_(torch.randint(-1, E, (T, k), generator=g, device="cuda"))
        h.zero_(), y.zero_()
        calls()
        want = _bits((h, y))
        calls(5)
        h.zero_(), y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert _bits((h, y)) == want, i
        exact, size = ref.down(_f64(x), ids.cpu().numpy(), None, c.w, np.zeros((T, 2 * O)), 1.0, 0.0)
        _close(y, exact, "fp16", c.slack * size)


def test_blocks_on_two_streams_and_threads():
    import torch

    from tests.test_decode_concurrency_gpu import _at_once
    blocks = [Block(T, seed=s) for s, T in enumerate((1, 24, 200, 3))]
    want = [_bits(b()) for b in blocks]
    torch.cuda.synchronize()
    one, streams = torch.cuda.current_stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    for stream_of in (lambda i: one, lambda i: streams[i % 2]):
        got = _at_once(blocks, 10, stream_of)
        for i, runs in enumerate(got):
            assert all(_bits(run) == want[i] for run in runs), i
