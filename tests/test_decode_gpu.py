"""Decode-step operators against their plain 64-bit definitions (_decode_ref).

Tolerances.  An output is rounded once, so it may be half a unit in the last
place off (2^-11 of the value in fp16, 2^-8 in bf16, with the smallest fp16
step near zero), and what the fp32 arithmetic leaves: a score of |t| <= 32 in
base 2 has an absolute error of a few 2^-24 |t| and of 2^-24 sum |q k| in its
dot product, below 1e-5 in all, which is the relative error of its softmax
term; the terms themselves are held to 2^-16 at least.  3e-5 of the largest
value covers both.  Norms and rotations are a handful of fp32 roundings: 2e-6.
"""
import numpy as np
import pytest

from tests import _decode_ref as ref
from tests._util import rng

pytestmark = pytest.mark.gpu

HALF_ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}


def _cg():
    import clove_compute_amd as cg
    return cg


def _dt(name):
    import torch
    return {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}[name]


def _dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(_dt(dtype))


def _f64(t):
    return t.detach().double().cpu().numpy()


def _rounded(g, dtype, *shape, scale=1.0):
    """A device tensor of `dtype` and the values it holds."""
    t = _dev((g.standard_normal(shape) * scale).astype(np.float32), dtype)
    return t, _f64(t)


def _close(got, want, dtype, extra):
    got, want = _f64(got), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]) and np.array_equal(np.isinf(got), inf)
    ok = np.isfinite(want)
    err = np.abs(got[ok] - want[ok])
    bound = HALF_ULP[dtype] * np.abs(want[ok]) * 1.0001 + TINY[dtype] + extra
    worst = np.max(err - bound) if err.size else 0.0
    assert worst <= 0, (worst, float(err.max()))


# ---- qk_norm_rope -------------------------------------------------------------


def _tables(n, R):
    f = 10000.0 ** (-np.arange(0, R, 2) / max(R, 1))
    ang = np.arange(n)[:, None] * f
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,Hq,Hk,D,R,P,interleaved,norm", [
    (1, 32, 8, 64, 64, 16, False, True), (1, 1, 1, 2, 2, 1, False, True), (37, 4, 2, 128, 128, 16, False, True),
    (37, 4, 2, 128, 64, 16, True, True), (5, 6, 3, 80, 40, 7, False, True), (5, 6, 3, 80, 80, 7, True, False),
    (9, 3, 1, 100, 48, 16, False, True), (9, 3, 1, 100, 100, 16, True, True), (4, 2, 2, 96, 96, 32, False, True),
    (3, 2, 1, 5, 4, 3, False, True), (3, 2, 1, 7, 0, 3, False, True), (11, 5, 5, 256, 256, 64, False, True),
    (2, 2, 1, 1024, 1000, 16, False, True), (3, 8, 1, 72, 36, 16, False, False), (600, 8, 2, 64, 64, 16, False, True),
    (3, 2, 2, 64, 0, 16, False, False), (3, 4, 0, 64, 64, 16, False, True), (4, 3, 1, 24, 16, 16, False, True),
    (4, 3, 1, 512, 512, 16, True, True), (70, 3, 1, 136, 64, 16, True, True)])
def test_rope_values(dtype, T, Hq, Hk, D, R, P, interleaved, norm):
    import torch
    cg = _cg()
    g = rng("rope", T, Hq, Hk, D, R)
    width = (Hq + 2 * Hk) * D
    x, x64 = _rounded(g, dtype, T, width, scale=2.0)
    wq, wq64 = _rounded(g, dtype, D) if norm else (None, None)
    wk, wk64 = _rounded(g, dtype, D) if norm else (None, None)
    cos, sin = _tables(50, R)
    pos = g.integers(0, 50, T).astype(np.int32)
    q64, k64, v64 = ref.qk_norm_rope(x64, wq64, wk64, cos, sin, pos, Hq, Hk, D, R, 1e-6, interleaved)
    pages = T // P + 3
    slots = g.permutation(pages * P)[:T].astype(np.int32)
    cache = None
    if Hk:
        k, v = (torch.full((pages, Hk, P, D), 7.0, dtype=_dt(dtype), device="cuda") for _ in range(2))
        cache = cg.KVCache(k, v)
    q_out = torch.empty(T, Hq, D, dtype=_dt(dtype), device="cuda")
    k_out = torch.empty(T, Hk, D, dtype=_dt(dtype), device="cuda") if Hk else None
    cg.qk_norm_rope(x, wq, wk, _dev(cos), _dev(sin), _dev(pos), q_out, T, Hq, Hk, D, rot_dim=R, interleaved=interleaved,
                    k_out=k_out, cache=cache, slots=_dev(slots) if Hk else None)
    most = float(max(np.abs(q64).max(), np.abs(k64).max() if Hk else 0))
    _close(q_out, q64, dtype, 2e-6 * most)
    if Hk:
        _close(k_out, k64, dtype, 2e-6 * most)
        want_k, want_v = np.full((2, pages, Hk, P, D), 7.0)
        got_k = k_out.cpu()
        want_v[slots // P, :, slots % P] = v64
        assert np.array_equal(_f64(v), want_v)
        want_k[slots // P, :, slots % P] = _f64(got_k)
        assert np.array_equal(_f64(k), want_k)


@pytest.mark.parametrize("dtype,D", [("fp16", 64), ("bf16", 128), ("fp16", 36)])
def test_rope_in_place_strides_and_padding(dtype, D):
    import torch
    cg = _cg()
    T, Hq, Hk, P, pages = 6, 4, 2, 4, 3
    g = rng("rope-in-place", D)
    width = (Hq + 2 * Hk) * D
    wide, _ = _rounded(g, dtype, T, width + 24)
    x = wide[:, 8:8 + width]  # rows of a wider tensor, queries and keys rotated where they are
    x64 = _f64(x)
    cos, sin = _tables(20, D)
    pos = np.array([0, 19, 20, -1, 3, 4], np.int32)  # two of them outside the table
    slots = np.array([0, -1, pages * P, 11, 5, -7], np.int32)  # three of them outside the cache
    both = torch.full((pages, 2, Hk, P, D), 3.0, dtype=_dt(dtype), device="cuda")
    cache = cg.KVCache(both[:, 0], both[:, 1])
    w, w64 = _rounded(g, dtype, D)
    q64, k64, v64 = ref.qk_norm_rope(x64, w64, w64, cos, sin, pos, Hq, Hk, D, D, 1e-5, False)
    before = _f64(wide)
    cg.qk_norm_rope(x, w, w, _dev(cos), _dev(sin), _dev(pos), x[:, :Hq * D], T, Hq, Hk, D, eps=1e-5,
                    k_out=x[:, Hq * D:(Hq + Hk) * D], cache=cache, slots=_dev(slots))
    _close(x[:, :Hq * D], q64.reshape(T, -1), dtype, 1e-5)
    _close(x[:, Hq * D:(Hq + Hk) * D], k64.reshape(T, -1), dtype, 1e-5)
    after = _f64(wide)
    assert np.array_equal(after[:, :8], before[:, :8]) and np.array_equal(after[:, 8 + (Hq + Hk) * D:], before[:, 8 + (Hq + Hk) * D:])
    want = np.full((pages, 2, Hk, P, D), 3.0)
    for t, s in enumerate(slots):
        if 0 <= s < pages * P:
            want[s // P, 0, :, s % P] = after[t, 8 + Hq * D:8 + (Hq + Hk) * D].reshape(Hk, D)
            want[s // P, 1, :, s % P] = v64[t]
    assert np.array_equal(_f64(both), want, equal_nan=True)


def test_rope_zero_rows_and_large_values():
    import torch
    cg = _cg()
    D, T = 64, 3
    cos, sin = _tables(4, D)
    x = torch.zeros(T, 3 * D, dtype=torch.bfloat16, device="cuda")
    x[1] = 3e38     # the squares pass fp32's range: 1 / inf
    x[2] = 1e-30
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(T, 1, D, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    cg.qk_norm_rope(x, w, None, _dev(cos), _dev(sin), pos, q, T, 1, 1, D)
    assert torch.equal(q[0], torch.zeros_like(q[0])) and torch.equal(q[1], torch.zeros_like(q[1]))
    _close(q[2], np.full((1, D), float(x[2, 0].double()) * 1e3), "bf16", 1e-30)
    cg.qk_norm_rope(x[:0], w, None, _dev(cos), _dev(sin), pos, q, 0, 1, 1, D)


# ---- paged_attention -----------------------------------------------------------


def _paged(g, dtype, lens, Hk, D, P, spare=2, nan_rest=True):
    """A cache whose rows that no key names are NaN, and its table (-1 past the end)."""
    import torch
    per = [-(-n // P) for n in lens]
    pages = sum(per) + spare
    order = g.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max(per + [1])), -1, np.int32)
    used = np.zeros((pages, P), bool)
    at = 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        for j in range(n):
            used[table[b, j // P], j % P] = True
    k, k64 = _rounded(g, dtype, pages, Hk, P, D)
    v, v64 = _rounded(g, dtype, pages, Hk, P, D)
    if nan_rest:
        rest = _dev(~used)[:, None, :, None]
        k.masked_fill_(rest, float("nan"))
        v.masked_fill_(rest, float("nan"))
    return k, v, k64, v64, table


def _attend(cg, q, cache, table, lens, B, Hq, L, weights=None, **kw):
    import torch
    out = torch.full_like(q, float("nan"))
    cg.paged_attention(q, cache, _dev(table), _dev(np.asarray(lens, np.int32)), out, B, Hq, L, weights=weights, **kw)
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hk,D,P", [
    ([1], 4, 1, 64, 16), ([0], 4, 2, 64, 16), ([33], 1, 1, 128, 16), ([0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65], 8, 2, 64, 16),
    ([700, 3, 0, 511, 512, 513], 32, 8, 64, 16), ([1000, 129], 16, 4, 128, 32), ([257, 40], 5, 5, 80, 24),
    ([100, 7], 14, 2, 72, 7), ([100, 50], 16, 1, 96, 1), ([300], 64, 2, 64, 64), ([90, 200], 33, 1, 128, 16),
    ([130, 31], 8, 2, 100, 16), ([77], 6, 2, 36, 16), ([60, 61], 4, 2, 256, 16), ([60], 4, 2, 250, 16), ([50], 4, 2, 8, 16),
    ([50], 2, 1, 5, 16), ([70], 4, 1, 320, 16), ([40], 2, 2, 1024, 16), ([20], 3, 1, 1, 4), ([3000], 8, 8, 64, 4096),
    ([5000, 12], 8, 2, 128, 128), ([200], 128, 1, 64, 16), ([64], 4, 2, 9, 16), ([64], 4, 2, 15, 16), ([64], 17, 1, 33, 16)])
def test_attention_values(dtype, lens, Hq, Hk, D, P):
    cg = _cg()
    g = rng("attend", tuple(lens), Hq, Hk, D, P)
    k, v, k64, v64, table = _paged(g, dtype, lens, Hk, D, P)
    B, L = len(lens), max(max(lens), 1)
    q, q64 = _rounded(g, dtype, B, Hq, D, scale=1.5)
    w0 = g.uniform(0, 1, (B, L)).astype(np.float32)
    w = _dev(w0)
    cache = cg.KVCache(k, v)
    want, added = ref.attention(q64, k64, v64, table, lens, D ** -0.5)
    out = _attend(cg, q, cache, table, lens, B, Hq, L)
    _close(out, want, dtype, 3e-5 * float(np.abs(v64).max()))
    again = _attend(cg, q, cache, table, lens, B, Hq, L, weights=w)
    assert np.array_equal(_f64(again), _f64(out))  # with the weights, the same bits
    got = _f64(w)
    for b, n in enumerate(lens):
        assert np.array_equal(got[b, n:], w0[b, n:].astype(np.float64))
    assert np.all(np.abs(got - (w0 + added[:, :L])) <= 2.0 ** -23 * (got + 1e-3) + 2e-5 * added[:, :L])


@pytest.mark.parametrize("softcap,window,scale", [(0.0, 1, None), (0.0, 40, None), (5.0, 0, None), (30.0, 100, 0.2), (0.0, 10 ** 6, 1.0), (0.0, 513, None)])
@pytest.mark.parametrize("D", [64, 20])
def test_attention_options(softcap, window, scale, D):
    cg = _cg()
    lens, Hq, Hk, P = [900, 0, 1, 40, 41, 600], 8, 2, 16
    g = rng("attend-options", D)
    k, v, k64, v64, table = _paged(g, "fp16", lens, Hk, D, P)
    q, q64 = _rounded(g, "fp16", len(lens), Hq, D)
    w = _dev(np.zeros((len(lens), 1000), np.float32))
    want, added = ref.attention(q64, k64, v64, table, lens, D ** -0.5 if scale is None else scale, softcap, window)
    out = _attend(cg, q, cg.KVCache(k, v), table, lens, len(lens), Hq, 900, weights=w, softcap=softcap, window=window, scale=scale)
    _close(out, want, "fp16", 3e-5 * float(np.abs(v64).max()))
    assert np.all(np.abs(_f64(w)[:, :900] - added[:, :900]) <= 3e-5 * added[:, :900] + 1e-9)


@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 2), (12, 2)])
def test_attention_absent_pages_and_lengths_past_the_bound(D, Hq):
    """Table entries outside the cache are absent keys; a length past max_context counts as it."""
    cg = _cg()
    lens, P, Hk = [200, 64, 48], 16, 2
    g = rng("attend-absent", D)
    k, v, k64, v64, table = _paged(g, "bf16", lens, Hk, D, P, nan_rest=False)
    table[0, 3], table[0, 7], table[0, 0] = -1, len(k64), 2 ** 31 - 1
    table[1, :] = -5  # a sequence of absent pages only
    q, q64 = _rounded(g, "bf16", 3, Hq, D)
    w = _dev(np.zeros((3, 150), np.float32))
    told = [200, 64, -3]
    want, added = ref.attention(q64, k64, v64, table, [150, 64, 0], D ** -0.5)
    out = _attend(cg, q, cg.KVCache(k, v), table, told, 3, Hq, 150, weights=w)
    _close(out, want, "bf16", 3e-5 * float(np.abs(v64).max()))
    assert np.all(want[1:] == 0)
    assert np.all(np.abs(_f64(w) - added[:, :150]) <= 3e-5 * added[:, :150])


@pytest.mark.parametrize("D", [64, 20])
def test_attention_infinite_and_nan_keys(D):
    """-inf scores weigh nothing (a query of them alone gives 0); a NaN key's query is NaN."""
    import torch
    cg = _cg()
    P, n = 16, 50
    g = rng("attend-inf", D)
    k, v, k64, v64, table = _paged(g, "fp16", [n, n, n], 1, D, P)
    q = torch.zeros(3, 2, D, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    page, row = table[0, 40 // P], 40 % P
    k[page, 0, row, 0] = k64[page, 0, row, 0] = -np.inf
    for j in range(n):
        k[table[1, j // P], 0, j % P, 0] = k64[table[1, j // P], 0, j % P, 0] = -np.inf
    k[table[2, 1], 0, 3, 0] = float("nan")
    with np.errstate(invalid="ignore"):
        want, _ = ref.attention(_f64(q), np.nan_to_num(k64, neginf=-1e30), v64, table, [n, 0, 0], D ** -0.5)
    out = _attend(cg, q, cg.KVCache(k, v), table, [n, n, n], 3, 2, n)
    _close(out[0], want[0], "fp16", 3e-5 * float(np.abs(v64).max()))
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    assert bool(torch.isnan(out[2]).all())


def test_attention_strides_and_interleaved_pages():
    import torch
    cg = _cg()
    lens, Hq, Hk, D, P = [40, 70], 6, 2, 64, 16
    g = rng("attend-strides")
    k, v, k64, v64, table = _paged(g, "fp16", lens, Hk, D, P)
    both = torch.stack((k, v), 1)
    wide, _ = _rounded(g, "fp16", 2, (Hq + 3) * D)
    q = wide[:, D:(Hq + 1) * D]
    out = torch.full((2, Hq * D + 40), 5.0, dtype=torch.float16, device="cuda")
    wide_table = np.full((2, 9), -1, np.int32)
    wide_table[:, :table.shape[1]] = table
    cg.paged_attention(q, cg.KVCache(both[:, 0], both[:, 1]), _dev(wide_table), _dev(np.array(lens, np.int32)), out[:, 8:8 + Hq * D],
                       2, Hq, 70)
    want, _ = ref.attention(_f64(q).reshape(2, Hq, D), k64, v64, table, lens, D ** -0.5)
    _close(out[:, 8:8 + Hq * D], want.reshape(2, -1), "fp16", 3e-5 * float(np.abs(v64).max()))
    assert bool((out[:, :8] == 5).all()) and bool((out[:, 8 + Hq * D:] == 5).all())


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and more than 2^31 elements per tensor: its last pages."""
    import torch
    cg = _cg()
    Hk, D, P, B = 8, 128, 64, 2
    pages = 2 ** 31 // (Hk * D * P) + 40
    g = rng("attend-large")
    k, v = (torch.empty(pages, Hk, P, D, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = [pages - 1, 3, pages - 7, pages - 2]
    table = np.array([rows[:2], rows[2:]], np.int32)
    k64, v64 = np.zeros((2, 4, Hk, P, D))
    for i, r in enumerate(rows):
        for t, c in ((k, k64), (v, v64)):
            t[r], c[i] = _rounded(g, "fp16", Hk, P, D)
    q, q64 = _rounded(g, "fp16", B, 16, D)
    want, _ = ref.attention(q64, k64, v64, np.array([[0, 1], [2, 3]]), [100, 128], D ** -0.5)
    out = _attend(cg, q, cg.KVCache(k, v), table, [100, 128], B, 16, 128)
    _close(out, want, "fp16", 3e-5 * float(np.abs(v64).max()))
    # and the cache write there
    x, x64 = _rounded(g, "fp16", 1, 3 * Hk * D)
    slot = _dev(np.array([(pages - 1) * P + 5], np.int32))
    cg.qk_norm_rope(x, None, None, None, None, None, torch.empty(1, Hk, D, dtype=torch.float16, device="cuda"), 1, Hk, Hk, D,
                    rot_dim=0, cache=cg.KVCache(k, v), slots=slot)
    assert np.array_equal(_f64(v[pages - 1, :, 5]).ravel(), x64[0, 2 * Hk * D:])
    # and a move between its ends
    before = _f64(k[pages - 1, :, 30])
    pos = np.arange(65, dtype=np.int32)[None]
    far, near = np.array([[3, pages - 1]], np.int32), np.ones((1, 65), np.float32)
    k[pages - 1, :, 0] = k[pages - 1, :, 30]
    near[0, 10] = 0.0
    cg.cache_evict(cg.KVCache(k, v), _dev(far), _dev(np.array([65], np.int32)), _dev(near), _dev(pos), _dev(near * 0),
                   _dev(pos * 0), _dev(np.zeros(1, np.int32)), 1, 65, 64)
    assert np.array_equal(_f64(k[3, :, 10]), before)


# ---- cache_evict ------------------------------------------------------------------


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sinks,recent,Hk,D,P,kind", [
    ([65], 64, 4, 8, 2, 64, 16, "tail"), ([100, 0, 3, 64, 65, 99], 64, 4, 16, 2, 64, 16, "tail"),
    ([500, 400], 33, 0, 5, 1, 80, 24, "tail"), ([300, 200], 40, 10, 100, 2, 128, 32, "tail"),  # more protected than fit
    ([300, 130], 128, 4, 16, 2, 20, 7, "ties"), ([700], 200, 0, 0, 1, 64, 16, "equal"), ([90, 91], 1, 0, 1, 2, 64, 16, "tail"),
    ([90], 0, 4, 4, 2, 64, 16, "tail"), ([200], 300, 4, 4, 2, 64, 16, "tail"), ([2500, 40, 2049], 2048, 4, 256, 1, 8, 16, "tail"),
    ([400], 100, 4, 8, 1, 64, 16, "odd"), ([5000, 4097], 1000, 4, 64, 1, 64, 64, "ties"), ([40000], 9000, 4, 64, 1, 8, 64, "ties")])
def test_evict(in_place, lens, budget, sinks, recent, Hk, D, P, kind):
    import torch
    cg = _cg()
    g = rng("evict", tuple(lens), budget, D, kind)
    B, L = len(lens), max(lens)
    k, v, k64, v64, table = _paged(g, "bf16", lens, Hk, D, P, nan_rest=False)
    w = np.exp(1.5 * g.standard_normal((B, L))).astype(np.float32)
    if kind == "ties":
        w = np.round(w)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "odd":  # signs, infinities, NaN, both zeros
        w = np.where(g.random((B, L)) < 0.5, -w, w)
        for x in (np.inf, -np.inf, np.nan, 0.0, -0.0):
            w[:, g.permutation(L)[:30]] = x
    pos = np.stack([g.permutation(L) + 3 for _ in range(B)]).astype(np.int32)
    want = ref.evict(k64, v64, table, lens, w, pos, L, budget, sinks, recent)
    dw, dp, dl = _dev(w), _dev(pos), _dev(np.array(lens, np.int32))
    wo, po, lo = (dw, dp, dl) if in_place else (torch.full_like(dw, 9), torch.full_like(dp, 9), torch.full_like(dl, 9))
    for _ in range(1 if in_place else 2):  # the same inputs again change nothing
        cg.cache_evict(cg.KVCache(k, v), _dev(table), dl, dw, dp, wo, po, lo, B, L, budget, sinks=sinks, recent=recent)
        for got, exact in zip((k, v, wo, po, lo), want):
            got, exact = _f64(got), exact.astype(np.float64)
            assert np.array_equal(got, exact, equal_nan=True)


def test_evict_absent_pages_strides_and_bounds():
    import torch
    cg = _cg()
    g = rng("evict-absent")
    lens, budget, P, Hk, D = [100, 80], 40, 16, 2, 64
    k, v, k64, v64, table = _paged(g, "fp16", lens, Hk, D, P, nan_rest=False)
    table[0, 1], table[1, 3] = -1, len(k64) + 5
    w = g.uniform(0, 1, (2, 130)).astype(np.float32)
    pos = np.tile(np.arange(130, dtype=np.int32), (2, 1))
    want = ref.evict(k64, v64, table, lens, w[:, :90], pos[:, :90], 90, budget, 2, 7)  # 100 counts as 90
    wo, po = torch.full((2, 200), 9.0, device="cuda"), torch.full((2, 150), 9, dtype=torch.int32, device="cuda")
    lo = torch.zeros(2, dtype=torch.int32, device="cuda")
    both = torch.stack((k, v), 1)
    cg.cache_evict(cg.KVCache(both[:, 0], both[:, 1]), _dev(table), _dev(np.array(lens, np.int32)), _dev(w), _dev(pos), wo, po, lo,
                   2, 90, budget, sinks=2, recent=7)
    assert np.array_equal(_f64(both[:, 0]), want[0]) and np.array_equal(_f64(both[:, 1]), want[1])
    assert np.array_equal(wo[:, :90].cpu().numpy(), want[2]) and np.array_equal(po[:, :90].cpu().numpy(), want[3])
    assert bool((wo[:, 90:] == 9).all()) and bool((po[:, 90:] == 9).all())
    assert lo.tolist() == [40, 40]


# ---- penalize_logits -----------------------------------------------------------------


def _logits_case(g, B, V, H, bias, mask, dtype):
    x, x64 = _rounded(g, dtype, B, V, scale=3.0)
    ids = g.integers(-3, V + 3, (B, H)).astype(np.int32)
    ids[:, ::3] = g.integers(0, min(V, 5), ids[:, ::3].shape)
    opts = dict(history=ids, history_lens=g.integers(0, H + 3, B).astype(np.int32),
                prompt_lens=g.integers(-1, H + 1, B).astype(np.int32),
                repetition=g.uniform(0.8, 1.6, B).astype(np.float32), presence=g.uniform(-0.5, 1, B).astype(np.float32),
                frequency=g.uniform(-0.5, 1, B).astype(np.float32))
    if bias:
        opts.update(bias_ids=g.integers(-2, V + 2, (B, bias)).astype(np.int32), bias_values=g.standard_normal((B, bias)).astype(np.float32),
                    bias_counts=g.integers(0, bias + 2, B).astype(np.int32))
    if mask:
        opts["allowed"] = g.integers(-2 ** 31, 2 ** 31, (B, -(-V // 32))).astype(np.int32)
    return x, x64, opts


def _logit_slack(x64, opts):
    """Four fp32 roundings of the largest number on the way."""
    most = np.abs(x64).max() * 1.6 + 40.0
    return 4 * 2.0 ** -24 * most


@pytest.mark.parametrize("dtype,out", [("fp16", "fp16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("B,V,H,bias,mask", [(1, 1, 1, 1, True), (1, 7, 20, 3, True), (2, 1000, 40, 0, False), (3, 4097, 300, 30, True),
                                             (1, 32000, 2000, 300, False), (5, 8191, 1, 2, True), (2, 12290, 700, 9, True)])
def test_logits(dtype, out, B, V, H, bias, mask):
    import torch
    cg = _cg()
    g = rng("logits", B, V, H, bias)
    x, x64, opts = _logits_case(g, B, V, H, bias, mask, dtype)
    want = ref.penalties(x64, **opts)
    y = torch.full((B, V), 5.0, dtype=_dt(out), device="cuda")
    dev = {n: _dev(a) for n, a in opts.items()}
    cg.penalize_logits(x, y, B, V, **dev)
    _close(y, want, out, _logit_slack(x64, opts))
    if dtype == out:  # in place
        cg.penalize_logits(x, x, B, V, **dev)
        assert np.array_equal(_f64(x), _f64(y), equal_nan=True)


@pytest.mark.parametrize("part", ["none", "history", "repetition", "presence", "frequency", "bias", "allowed", "no prompt"])
def test_logits_parts_alone(part):
    import torch
    cg = _cg()
    g = rng("logits-parts", part)
    B, V, H = 3, 2500, 200
    x, x64, full = _logits_case(g, B, V, H, 12, True, "fp32")
    told = {"none": [], "history": ["history", "history_lens", "prompt_lens"], "bias": ["bias_ids", "bias_values"], "allowed": ["allowed"],
            "no prompt": ["history", "history_lens", "presence", "frequency", "repetition"]}
    names = told.get(part) or ([] if part == "none" else ["history", "history_lens", "prompt_lens", part])
    opts = {n: full[n] for n in names}
    want = ref.penalties(x64, **opts)
    y = torch.empty_like(x)
    cg.penalize_logits(x, y, B, V, **{n: _dev(a) for n, a in opts.items()})
    _close(y, want, "fp32", _logit_slack(x64, opts))


def test_logits_infinities_nan_and_strides():
    import torch
    cg = _cg()
    B, V = 2, 70
    wide = torch.full((B, V + 9), 2.0, device="cuda")
    x = wide[:, 3:3 + V]
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = -np.inf, np.inf, np.nan, np.nan
    hist = torch.tensor([[0, 1, 2, 0], [4, 4, 4, 4]], dtype=torch.int32, device="cuda")
    allowed = torch.full((B, 5), -1, dtype=torch.int32, device="cuda")
    allowed[0, 0] = ~(1 << 3)
    y = torch.full((B, V + 2), 8.0, device="cuda")
    rep = torch.tensor([2.0, 4.0], device="cuda")
    cg.penalize_logits(x, y[:, 1:1 + V], B, V, history=hist, history_lens=torch.tensor([4, 2], dtype=torch.int32, device="cuda"),
                       repetition=rep, allowed=allowed)
    got = _f64(y)
    assert got[0, 1] == -np.inf and got[0, 2] == np.inf and np.isnan(got[0, 3]) and got[0, 4] == -np.inf
    assert got[1, 5] == 0.5 and got[1, 6] == 2.0 and (got[:, 0] == 8).all() and (got[:, -1] == 8).all()


# ---- streams, workspaces, graphs, repetition ---------------------------------------------


def _step(cg, st):
    cg.qk_norm_rope(st["qkv"], st["w"], st["w"], st["cos"], st["sin"], st["pos"], st["q"], st["B"], 8, 2, 64, cache=st["cache"],
                    slots=st["slots"])
    cg.paged_attention(st["q"], st["cache"], st["table"], st["lens"], st["o"], st["B"], 8, st["L"], weights=st["weights"])
    cg.cache_evict(st["cache"], st["table"], st["lens"], st["weights"], st["positions"], st["wo"], st["po"], st["lo"], st["B"], st["L"],
                   st["L"] - 60, sinks=4, recent=16)
    cg.penalize_logits(st["logits"], st["y"], st["B"], 5000, history=st["hist"], history_lens=st["lens"], repetition=st["rep"])


def _state(cg):
    import torch
    g = rng("decode-state")
    B, L, P = 3, 1500, 16
    lens = [1500, 700, 1499]
    k, v, _, _, table = _paged(g, "fp16", lens, 2, 64, P, nan_rest=False)
    st = dict(B=B, L=L, cache=cg.KVCache(k, v), k=k, v=v, table=_dev(table), lens=_dev(np.array(lens, np.int32)))
    st["qkv"], _ = _rounded(g, "fp16", B, 12 * 64)
    st["w"], _ = _rounded(g, "fp16", 64)
    st["cos"], st["sin"] = (_dev(t) for t in _tables(2000, 64))
    st["pos"] = _dev(np.array(lens, np.int32))
    st["slots"] = _dev(np.array([table[b, (n - 1) // P] * P + (n - 1) % P for b, n in enumerate(lens)], np.int32))
    st["weights"] = _dev(g.uniform(0, 1, (B, L)).astype(np.float32))
    st["positions"] = _dev(np.stack([g.permutation(L) for _ in range(B)]).astype(np.int32))
    st["logits"], _ = _rounded(g, "fp16", B, 5000)
    st["hist"], st["rep"] = _dev(g.integers(0, 5000, (B, L)).astype(np.int32)), _dev(np.full(B, 1.2, np.float32))
    st["q"], st["o"] = (torch.empty(B, 8, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    st["wo"], st["po"], st["lo"] = torch.empty_like(st["weights"]), torch.empty_like(st["positions"]), torch.empty_like(st["lens"])
    st["y"] = torch.empty_like(st["logits"])
    return st


_MUTABLE = ("k", "v", "weights")
_RESULTS = ("q", "o", "k", "v", "weights", "wo", "po", "lo", "y")


def _fresh(st, kept):
    for n in _MUTABLE:
        st[n].copy_(kept[n])


def test_steps_repeat_and_run_on_workspaces_streams_and_graphs():
    import torch
    cg = _cg()
    st = _state(cg)
    kept = {n: st[n].clone() for n in _MUTABLE}
    _step(cg, st)
    torch.cuda.synchronize()
    first = {n: st[n].clone() for n in _RESULTS}

    def same():
        torch.cuda.synchronize()
        for n in _RESULTS:
            assert torch.equal(st[n], first[n]), n

    _fresh(st, kept)
    _step(cg, st)
    same()
    with cg.workspace_query() as q:
        _step(cg, st)
    assert q.bytes > cg.CLOVE_WORKSPACE_MIN_BYTES
    _fresh(st, kept)
    torch.cuda.synchronize()
    ws = torch.zeros(q.bytes, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    cg.workspace_bind(ws)
    try:
        with torch.cuda.stream(side):
            _step(cg, st)
        same()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _step(cg, st)
        for _ in range(4):
            _fresh(st, kept)
            for n in ("q", "o", "wo", "po", "lo", "y"):
                st[n].zero_()
            torch.cuda.synchronize()
            graph.replay()
            same()
        with pytest.raises(cg.CloveError) as e:
            cg.workspace_bind(ws[:cg.CLOVE_WORKSPACE_MIN_BYTES])
            _step(cg, st)
        assert e.value.status == cg.CLOVE_ERR_WORKSPACE
    finally:
        cg.workspace_bind()


def test_python_checks():
    import torch
    cg = _cg()
    st = _state(cg)
    B, L = st["B"], st["L"]
    with pytest.raises(ValueError):
        cg.KVCache(st["k"], st["v"][:, :1])
    with pytest.raises(ValueError):
        cg.KVCache(st["k"].transpose(1, 2), st["v"].transpose(1, 2))
    with pytest.raises(ValueError):  # another type than the cache's
        cg.paged_attention(st["q"].bfloat16(), st["cache"], st["table"], st["lens"], st["o"], B, 8, L)
    with pytest.raises(ValueError):
        cg.paged_attention(st["q"], st["cache"], st["table"].long(), st["lens"], st["o"], B, 8, L)
    with pytest.raises(ValueError):  # a table of fewer pages than the longest context
        cg.paged_attention(st["q"], st["cache"], st["table"][:, :5], st["lens"], st["o"], B, 8, L)
    with pytest.raises(ValueError):
        cg.paged_attention(st["q"], st["cache"], st["table"], st["lens"].cpu(), st["o"], B, 8, L)
    with pytest.raises(ValueError):  # fewer rows than the batch
        cg.paged_attention(st["q"][:2], st["cache"], st["table"], st["lens"], st["o"], B, 8, L)
    with pytest.raises(ValueError):
        cg.qk_norm_rope(st["qkv"], st["w"], st["w"], st["cos"][:, :7], st["sin"][:, :7], st["pos"], st["q"], B, 8, 2, 64)
    with pytest.raises(ValueError):
        cg.qk_norm_rope(st["qkv"], st["w"][:3], st["w"], st["cos"], st["sin"], st["pos"], st["q"], B, 8, 2, 64)
    with pytest.raises(ValueError):
        cg.cache_evict(st["cache"], st["table"], st["lens"], st["weights"], st["weights"], st["wo"], st["po"], st["lo"], B, L, 9)
    with pytest.raises(ValueError):
        cg.penalize_logits(st["logits"][:, ::2], st["y"], B, 2500)
    with pytest.raises(ValueError):
        cg.penalize_logits(st["logits"].double(), st["y"], B, 5000)
    with pytest.raises(cg.CloveError):
        cg.paged_attention(st["q"], st["cache"], st["table"], st["lens"], st["q"], B, 8, L)


def test_arguments_of_other_kinds_are_errors():
    """What is no tensor, no number or too large a number raises and leaves nothing behind."""
    import torch
    cg = _cg()
    x = torch.ones(2, 64, device="cuda")
    y = torch.zeros_like(x)
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device="cuda")
    q, lens = torch.zeros(2, 128, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        cg.penalize_logits(x.cpu().numpy(), y, 2, 64)
    with pytest.raises(TypeError):
        cg.penalize_logits(x, y, 2, "64")
    with pytest.raises(TypeError):
        cg.penalize_logits(x, y, 2, 64, history=[1, 2])
    with pytest.raises(OverflowError):
        cg.penalize_logits(x, y, 2, 64 + 2 ** 32)
    with pytest.raises(ValueError):
        cg.penalize_logits(x, y, 2 ** 31 - 1, 2 ** 31 - 1)
    with pytest.raises(AttributeError):
        cg.paged_attention(q, None, table, lens, q.clone(), 2, 2, 16)
    with pytest.raises((ValueError, OverflowError)):
        cg.paged_attention(q, cg.KVCache(k, k.clone()), table, lens, q.clone(), 2, 2 ** 31 - 1, 16)
    with pytest.raises(cg.CloveError):  # pages of no rows
        cg.paged_attention(q, cg.KVCache(k[:, :, :0].contiguous(), k[:, :, :0].contiguous()), table, lens, q.clone(), 2, 2, 16)
    with pytest.raises(ValueError):
        cg.KVCache(k.double(), k.double())
    with pytest.raises(ValueError):
        cg.penalize_logits(x, y, 2, 64, history=torch.zeros((), dtype=torch.int32, device="cuda"), history_lens=lens)
    assert not y.any()
    cg.penalize_logits(x, y, 2, 64, stream=torch.cuda.current_stream().cuda_stream)
    cg.penalize_logits(x, x, 2, 64, stream=torch.cuda.current_stream())
    assert torch.equal(x, y)


def test_logits_lists_are_whole():
    """Part of a longer list per row is refused (the distance of rows is their length);
    of a single row it is taken, and nothing past it."""
    import torch
    cg = _cg()
    x = torch.ones(2, 64, device="cuda")
    y, two = torch.empty_like(x), torch.tensor([2.0, 2.0], device="cuda")
    ids = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    lens, values = torch.tensor([16, 16], dtype=torch.int32, device="cuda"), torch.ones(2, 16, device="cuda")
    for part in (slice(0, 4), slice(8, 16)):
        with pytest.raises(ValueError):
            cg.penalize_logits(x, y, 2, 64, history=ids[:, part], history_lens=lens, repetition=two)
        with pytest.raises(ValueError):
            cg.penalize_logits(x, y, 2, 64, bias_ids=ids[:, part], bias_values=values[:, part])
    with pytest.raises(ValueError):
        cg.penalize_logits(x, y, 2, 64, bias_ids=ids, bias_values=values[:, :4].contiguous())
    cg.penalize_logits(x, y, 1, 64, history=ids[:1, 4:8], history_lens=lens, repetition=two, bias_ids=ids[1:, :2],
                       bias_values=values[1:, :2])
    want = torch.ones(64)
    want[4:8], want[16:18] = 0.5, 2.0
    assert torch.equal(y[0].cpu(), want)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sinks,recent,kind", [
    ([17000, 16384, 16390], 4096, 4, 300, "free"), ([33000, 20000], 12000, 0, 1, "ties"), ([18001], 18000, 4, 100, "free"),
    ([18001], 3, 4, 100, "free"), ([16385, 1], 16384, 0, 0, "equal"), ([20000], 9000, 12000, 0, "ties"), ([33001], 9000, 12000, 0, "ties")])
def test_evict_long(in_place, lens, budget, sinks, recent, kind):
    import torch
    cg = _cg()
    g = rng("evict-long", tuple(lens), budget)
    B, L, P = len(lens), max(lens), 128
    k, v, k64, v64, table = _paged(g, "fp16", lens, 1, 8, P, nan_rest=False)
    w = np.exp(1.5 * g.standard_normal((B, L))).astype(np.float32)
    w = {"free": w, "ties": np.round(w), "equal": np.full_like(w, 2.0)}[kind]
    pos = np.stack([g.permutation(L) for _ in range(B)]).astype(np.int32)
    want = ref.evict(k64, v64, table, lens, w, pos, L, budget, sinks, recent)
    dw, dp, dl = _dev(w), _dev(pos), _dev(np.array(lens, np.int32))
    wo, po, lo = (dw, torch.full_like(dp, 9), dl) if in_place else (torch.full_like(dw, 9), torch.full_like(dp, 9), torch.full_like(dl, 9))
    cg.cache_evict(cg.KVCache(k, v), _dev(table), dl, dw, dp, wo, po, lo, B, L, budget, sinks=sinks, recent=recent)
    for got, exact in zip((k, v, wo, po, lo), want):
        assert np.array_equal(_f64(got), exact.astype(np.float64))


def test_logits_histories_and_lists_past_15_bits():
    """40000 ids of a few tokens (counts past 2^15), and a bias list as long."""
    import torch
    cg = _cg()
    g = rng("logits-long")
    B, V, H = 2, 9000, 40000
    for bias in (40000, 5):
        x, x64, opts = _logits_case(g, B, V, H, bias, True, "fp32")
        opts["history"][1] = 8995
        opts["history_lens"] = np.array([H, H], np.int32)
        opts["prompt_lens"] = np.array([100, 0], np.int32)
        want = ref.penalties(x64, **opts)
        y = torch.empty_like(x)
        cg.penalize_logits(x, y, B, V, **{n: _dev(a) for n, a in opts.items()})
        _close(y, want, "fp32", _logit_slack(x64, opts) + 4 * 2.0 ** -24 * np.abs(want[np.isfinite(want)]).max())


@pytest.mark.parametrize("over", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("kind", ["free", "ties", "equal", "odd", "safe"])
def test_evict_a_few_tokens(over, kind):
    """As many tokens over the budget as a step or a few bring, in lengths of one call that differ."""
    import torch
    cg = _cg()
    g = rng("evict-few", over, kind)
    budget, P = 700, 16
    L = budget + over
    lens = [L, L - 1, budget, 5, L]
    B = len(lens)
    k, v, k64, v64, table = _paged(g, "fp16", lens, 2, 64, P, nan_rest=False)
    w = np.exp(1.5 * g.standard_normal((B, L))).astype(np.float32)
    if kind == "ties":
        w = np.round(w)
    elif kind == "equal":
        w[:] = 0.5
    elif kind == "odd":
        for x in (np.inf, -np.inf, np.nan, 0.0, -0.0, -1.0):
            w[:, g.permutation(L)[:3]] = x
    if over > 1:
        w[0, -2:] = 0.0  # the newest slots go, and the slots past the budget with them
    pos = np.stack([g.permutation(L) for _ in range(B)]).astype(np.int32)
    recent = L if kind == "safe" else 20
    want = ref.evict(k64, v64, table, lens, w, pos, L, budget, 4, recent)
    for in_place in (False, True):
        dk, dv = k.clone(), v.clone()
        dw, dp, dl = _dev(w), _dev(pos), _dev(np.array(lens, np.int32))
        wo, po, lo = (dw, dp, dl) if in_place else (torch.full_like(dw, 9), torch.full_like(dp, 9), torch.full_like(dl, 9))
        cg.cache_evict(cg.KVCache(dk, dv), _dev(table), dl, dw, dp, wo, po, lo, B, L, budget, sinks=4, recent=recent)
        for got, exact in zip((dk, dv, wo, po, lo), want):
            assert np.array_equal(_f64(got), exact.astype(np.float64), equal_nan=True)


# ---- other alignments, bounds and lengths ---------------------------------------------------


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 100, 72])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_attention_rows_at_any_alignment(dtype, D, shift):
    """q, out and the cache `shift` elements past an aligned address."""
    import torch
    cg = _cg()
    lens, Hq, Hk, P = [70, 300, 0], 8, 2, 16
    g = rng("attend-align", D, shift)
    k, v, k64, v64, table = _paged(g, dtype, lens, Hk, D, P, nan_rest=False)

    def moved(t):
        flat = torch.full((t.numel() + 64,), float("nan"), dtype=t.dtype, device="cuda")
        out = flat[shift:shift + t.numel()].view(t.shape)
        out.copy_(t)
        return out

    k, v = moved(k), moved(v)
    wide, _ = _rounded(g, dtype, 3, Hq * D + 8)
    q = wide[:, shift:shift + Hq * D]
    out = torch.full((3, Hq * D + 16), 5.0, dtype=_dt(dtype), device="cuda")
    cg.paged_attention(q, cg.KVCache(k, v), _dev(table), _dev(np.array(lens, np.int32)), out[:, shift:shift + Hq * D], 3, Hq, 300)
    want, _ = ref.attention(_f64(q).reshape(3, Hq, D), k64, v64, table, lens, D ** -0.5)
    _close(out[:, shift:shift + Hq * D], want.reshape(3, -1), dtype, 3e-5 * float(np.abs(v64).max()))
    assert bool((out[:, :shift] == 5).all()) and bool((out[:, shift + Hq * D:] == 5).all())


@pytest.mark.parametrize("D", [64, 128, 36])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rope_rows_at_any_alignment(D, shift):
    import torch
    cg = _cg()
    T, Hq, Hk = 5, 3, 1
    g = rng("rope-align", D, shift)
    width = (Hq + 2 * Hk) * D
    wide, _ = _rounded(g, "fp16", T, width + 8)
    x = wide[:, shift:shift + width]
    w, w64 = _rounded(g, "fp16", D)
    cos, sin = _tables(9, D)
    pos = np.array([0, 8, 3, 1, 7], np.int32)
    out = torch.full((T, Hq * D + 8), 5.0, dtype=torch.float16, device="cuda")
    q64, _, _ = ref.qk_norm_rope(_f64(x), w64, w64, cos, sin, pos, Hq, Hk, D, D, 1e-6, False)
    cg.qk_norm_rope(x, w, w, _dev(cos), _dev(sin), _dev(pos), out[:, shift:shift + Hq * D], T, Hq, Hk, D)
    _close(out[:, shift:shift + Hq * D], q64.reshape(T, -1), "fp16", 2e-5)
    assert bool((out[:, :shift] == 5).all()) and bool((out[:, shift + Hq * D:] == 5).all())


@pytest.mark.parametrize("D", [5, 6, 12, 32])
def test_evict_rows_of_every_width(D):
    import torch
    cg = _cg()
    g = rng("evict-width", D)
    lens, budget, P = [300, 120], 100, 16
    k, v, k64, v64, table = _paged(g, "bf16", lens, 3, D, P, nan_rest=False)
    w = g.uniform(0, 1, (2, 300)).astype(np.float32)
    pos = np.stack([g.permutation(300) for _ in range(2)]).astype(np.int32)
    want = ref.evict(k64, v64, table, lens, w, pos, 300, budget, 4, 10)
    dw, dp, dl = _dev(w), _dev(pos), _dev(np.array(lens, np.int32))
    cg.cache_evict(cg.KVCache(k, v), _dev(table), dl, dw, dp, torch.empty_like(dw), torch.empty_like(dp), torch.empty_like(dl), 2, 300,
                   budget, sinks=4, recent=10)
    assert np.array_equal(_f64(k), want[0]) and np.array_equal(_f64(v), want[1])


def test_nothing_cached_and_empty_batches():
    import torch
    cg = _cg()
    k = torch.empty(0, 2, 16, 64, dtype=torch.float16, device="cuda")
    cache = cg.KVCache(k, k.clone())
    q = torch.ones(2, 4, 64, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7)
    lens, table = torch.tensor([3, 0], dtype=torch.int32, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    w = torch.ones(2, 16, device="cuda")
    cg.paged_attention(q, cache, table, lens, out, 2, 4, 16, weights=w)  # pages of a cache that has none
    assert bool((out == 0).all()) and bool((w == 1).all())
    out.fill_(7)
    cg.paged_attention(q, cache, table, lens, out, 2, 4, 0)  # no key may be read
    assert bool((out == 0).all())
    cg.paged_attention(q[:0], cache, table[:0], lens[:0], out[:0], 0, 4, 16)
    cg.penalize_logits(w[:0], w[:0], 0, 16)
    x = torch.ones(2, 16, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    cg.cache_evict(cache, table, lens, w, x, w.clone(), x.clone(), n, 2, 16, 1)
    assert n.tolist() == [1, 0]


@pytest.mark.parametrize("B", [70, 300])
def test_attention_many_sequences(B):
    """More sequences than a wave has lanes, of very different lengths, most of them short."""
    cg = _cg()
    g = rng("attend-many", B)
    lens = [int(x) for x in np.exp(g.uniform(0, np.log(200), B))]
    lens[0], lens[B // 2], lens[-1], lens[5] = 3000, 5000, 0, 4097
    Hq, Hk, D, P = 4, 1, 64, 16
    k, v, k64, v64, table = _paged(g, "fp16", lens, Hk, D, P)
    q, q64 = _rounded(g, "fp16", B, Hq, D)
    want, added = ref.attention(q64, k64, v64, table, lens, D ** -0.5)
    w = _dev(np.zeros((B, 5000), np.float32))
    out = _attend(cg, q, cg.KVCache(k, v), table, lens, B, Hq, 5000, weights=w)
    _close(out, want, "fp16", 3e-5 * float(np.abs(v64).max()))
    assert np.all(np.abs(_f64(w) - added[:, :5000]) <= 3e-5 * added[:, :5000] + 1e-9)


@pytest.mark.parametrize("Hq,Hk,D", [(16, 1, 128), (4, 1, 64), (3, 1, 250)])
def test_attention_long_sequence_joined_in_groups(Hq, Hk, D):
    """Splits enough for joins of joins, and the same lengths behind a larger bound."""
    import torch
    cg = _cg()
    g = rng("attend-groups", Hq, D)
    lens, P = [40000, 9], 64
    k, v, k64, v64, table = _paged(g, "bf16", lens, Hk, D, P, nan_rest=False)
    q, q64 = _rounded(g, "bf16", 2, Hq, D, scale=1.5)
    want, _ = ref.attention(q64, k64, v64, table, lens, D ** -0.5)
    out = _attend(cg, q, cg.KVCache(k, v), table, lens, 2, Hq, 40000)
    _close(out, want, "bf16", 3e-5 * float(np.abs(v64).max()))
    one = torch.full_like(q[:1], float("nan"))
    cg.paged_attention(q[:1], cg.KVCache(k, v), _dev(table[:1]), _dev(np.array(lens[:1], np.int32)), one, 1, Hq, 40000)
    _close(one, want[:1], "bf16", 3e-5 * float(np.abs(v64).max()))


def test_attention_graph_follows_the_lengths():
    """A recorded call cuts the sequences by the lengths of each replay."""
    import torch
    cg = _cg()
    g = rng("attend-graph")
    B, Hq, Hk, D, P, L = 3, 8, 2, 64, 16, 4000
    k, v, k64, v64, table = _paged(g, "fp16", [L] * B, Hk, D, P, nan_rest=False)
    q, q64 = _rounded(g, "fp16", B, Hq, D)
    cache, dt, lens = cg.KVCache(k, v), _dev(table), torch.zeros(B, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    with cg.workspace_query() as need:
        cg.paged_attention(q, cache, dt, lens, out, B, Hq, L)
    ws = torch.zeros(need.bytes, dtype=torch.uint8, device="cuda")
    cg.workspace_bind(ws)
    try:
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            cg.paged_attention(q, cache, dt, lens, out, B, Hq, L)
        for told in ([4000, 4000, 4000], [1, 0, 3999], [0, 0, 0], [200, 2500, 33], [4000, 1, 1]):
            lens.copy_(torch.tensor(told, dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want, _ = ref.attention(q64, k64, v64, table, told, D ** -0.5)
            _close(out, want, "fp16", 3e-5 * float(np.abs(v64).max()))
    finally:
        cg.workspace_bind()


@pytest.mark.parametrize("over", [1, 4])
def test_evict_a_few_wide_tokens(over):
    """Rows of so many heads that the few moved ones take a second kernel."""
    import torch
    cg = _cg()
    g = rng("evict-wide", over)
    budget, P, Hk, D = 20, 8, 16, 1024
    L = budget + over
    lens = [L, 7]
    k, v, k64, v64, table = _paged(g, "fp16", lens, Hk, D, P, nan_rest=False)
    w = g.uniform(1, 2, (2, L)).astype(np.float32)
    w[0, :over] = 0.0
    pos = np.tile(np.arange(L, dtype=np.int32), (2, 1))
    want = ref.evict(k64, v64, table, lens, w, pos, L, budget, 0, 5)
    for in_place in (False, True):
        dk, dv, dw, dp, dl = k.clone(), v.clone(), _dev(w), _dev(pos), _dev(np.array(lens, np.int32))
        wo, po, lo = (dw, dp, dl) if in_place else (torch.full_like(dw, 9), torch.full_like(dp, 9), torch.full_like(dl, 9))
        cg.cache_evict(cg.KVCache(dk, dv), _dev(table), dl, dw, dp, wo, po, lo, 2, L, budget, recent=5)
        for got, exact in zip((dk, dv, wo, po, lo), want):
            assert np.array_equal(_f64(got), exact.astype(np.float64))


@pytest.mark.parametrize("B,longest,D,dtype", [(300, 30, 64, "fp16"), (520, 300, 64, "bf16"), (260, 500, 100, "fp16"), (140, 90, 256, "bf16")])
def test_attention_more_short_sequences_than_the_card_holds(B, longest, D, dtype):
    """One wave to a sequence and head."""
    cg = _cg()
    g = rng("attend-crowd", B, D)
    lens = [int(x) for x in g.integers(0, longest + 1, B)]
    lens[7], lens[8], lens[9] = longest, 0, 1
    Hq, Hk, P = 4, 4, 16
    k, v, k64, v64, table = _paged(g, dtype, lens, Hk, D, P)
    q, q64 = _rounded(g, dtype, B, Hq, D)
    w = _dev(np.zeros((B, longest), np.float32))
    want, added = ref.attention(q64, k64, v64, table, lens, D ** -0.5)
    out = _attend(cg, q, cg.KVCache(k, v), table, lens, B, Hq, longest, weights=w)
    _close(out, want, dtype, 3e-5 * float(np.abs(v64).max()))
    assert np.all(np.abs(_f64(w) - added[:, :longest]) <= 3e-5 * added[:, :longest] + 1e-9)


@pytest.mark.parametrize("dtype,D", [("fp16", 64), ("bf16", 128), ("fp16", 96), ("bf16", 40), ("fp16", 136)])
def test_attention_lengths_around_the_forms_of_the_kernel(dtype, D):
    """Bounds on either side of what one, four and eight waves take at once."""
    cg = _cg()
    g = rng("attend-forms", D)
    Hq, Hk, P = 6, 2, 16
    for longest in (31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 513):
        lens = [longest, 0, max(1, longest // 3), longest - 1]
        k, v, k64, v64, table = _paged(g, dtype, lens, Hk, D, P)
        q, q64 = _rounded(g, dtype, 4, Hq, D)
        w = _dev(np.zeros((4, longest), np.float32))
        want, added = ref.attention(q64, k64, v64, table, lens, D ** -0.5)
        out = _attend(cg, q, cg.KVCache(k, v), table, lens, 4, Hq, longest, weights=w)
        _close(out, want, dtype, 3e-5 * float(np.abs(v64).max()))
        assert np.all(np.abs(_f64(w) - added[:, :longest]) <= 3e-5 * added[:, :longest] + 1e-9)


@pytest.mark.parametrize("dtype,D", [("fp16", 64), ("bf16", 36)])
def test_rope_in_place_of_one_token(dtype, D):
    """Queries and keys of a single row rotated where they are."""
    cg = _cg()
    Hq, Hk = 4, 2
    g = rng("rope-one", D)
    x, x64 = _rounded(g, dtype, 1, (Hq + 2 * Hk) * D)
    w, w64 = _rounded(g, dtype, D)
    cos, sin = _tables(20, D)
    pos = np.array([7], np.int32)
    q64, k64, v64 = ref.qk_norm_rope(x64, w64, w64, cos, sin, pos, Hq, Hk, D, D, 1e-6, False)
    cg.qk_norm_rope(x, w, w, _dev(cos), _dev(sin), _dev(pos), x[:, :Hq * D], 1, Hq, Hk, D, k_out=x[:, Hq * D:(Hq + Hk) * D])
    _close(x[:, :Hq * D], q64.reshape(1, -1), dtype, 1e-5)
    _close(x[:, Hq * D:(Hq + Hk) * D], k64.reshape(1, -1), dtype, 1e-5)
    assert np.array_equal(_f64(x)[:, (Hq + Hk) * D:], v64.reshape(1, -1))


def test_tensors_of_another_device_than_the_current_are_refused():
    import torch
    from tests.test_decode_binding import _Elsewhere
    x = _Elsewhere("cuda:1", 2, 64)  # (has no memory, and need not be there)
    with pytest.raises(ValueError, match="the tensors are on cuda:1, the current device is cuda:0"):
        _cg().penalize_logits(x, x, 2, 64)
    y = torch.ones(2, 64, device="cuda")
    with pytest.raises(ValueError, match="out is on cuda:1"):
        _cg().penalize_logits(y, x, 2, 64)
