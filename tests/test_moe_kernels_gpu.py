"""Every kernel of the experts' products, through calls whose sizes reach it (_moe_plan.CALLS;
test_moe_plan.py holds them to the names on the host): values, tiles of every fill, scales,
rows that are not finite, the rows behind the last pair, graphs, workspaces.

Tolerances are those of test_moe_gpu.py, which derives them.
"""
import numpy as np
import pytest

from tests import _moe_plan as plan
from tests import _moe_ref as ref
from tests._util import rng
from tests.test_decode_gpu import _dev, _f64, _rounded
from tests.test_moe_gpu import Case, _bits, _cg, _close

pytestmark = pytest.mark.gpu

BEHIND = 3  # rows of the output behind the last one


@pytest.fixture(autouse=True)
def _card():
    import torch
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    if cus != plan.CUS:
        pytest.skip(f"the calls are chosen for {plan.CUS} CUs, this card has {cus}")


def _up64(x, ids, w, h):
    """ref.swiglu_up an expert at a time."""
    k, I = ids.shape[1], w.shape[1] // 2
    out, size, flat = h.copy(), np.zeros_like(h), ids.reshape(-1)
    with np.errstate(all="ignore"):
        for e in range(w.shape[0]):
            p = np.flatnonzero(flat == e)
            if p.size == 0:
                continue
            xt, we, wa = x[p // k], w[e].T, np.abs(w[e]).T
            both, sizes = xt @ we, np.abs(xt) @ wa
            g, u, gs, us = both[:, :I], both[:, I:], sizes[:, :I], sizes[:, I:]
            s = 1.0 / (1.0 + np.exp(-g))
            out[p] = g * s * u
            size[p] = 1.1 * gs * np.abs(u) + np.abs(g * s) * us + np.abs(out[p])
    return out, size


def _down64(h, ids, weights, w, y, alpha, beta):
    """ref.down an expert at a time."""
    k, flat = ids.shape[1], ids.reshape(-1)
    out, size = np.zeros(y.shape), np.zeros(y.shape)
    with np.errstate(all="ignore"):
        for e in range(w.shape[0]):
            p = np.flatnonzero(flat == e)
            if p.size == 0:
                continue
            c = np.ones((p.size, 1)) if weights is None else weights.reshape(-1)[p][:, None]
            np.add.at(out, p // k, c * (h[p] @ w[e].T))
            np.add.at(size, p // k, np.abs(c) * (np.abs(h[p]) @ np.abs(w[e]).T))
        out, size = alpha * out, abs(alpha) * size
        if beta:
            out, size = out + beta * y, size + np.abs(beta * y)
    return out, size


class Call:
    """One call of a kernel: `self.run()` makes it on fresh outputs and returns them."""

    def __init__(self, call, key="kernels", **kw):
        import torch
        self.kernel, self.op, T, k, E, O, K = call
        c = self.c = Case((key, *call), T, k, E, 2 * O if self.op == "up" else O, K, **kw)
        self.T, self.k, self.E, self.O, self.K = T, k, E, O, K
        n = T if self.op == "up" else T * k
        self.x, _ = _rounded(c.g, "fp16", n, K)
        self.w = None if self.op == "up" else _dev(c.g.uniform(-0.5, 1.0, (T, k)).astype(np.float32))
        self.alpha, self.beta = 0.75, 1.0
        self.rows = T * k if self.op == "up" else T
        self.before, _ = _rounded(c.g, "fp16", self.rows + BEHIND, O)
        self.y = torch.empty_like(self.before)

    def ids(self, ids):
        import torch
        self.c.ids = np.ascontiguousarray(ids, np.int32).reshape(self.T, self.k)
        self.c.dev_ids = torch.from_numpy(self.c.ids).cuda()

    def scales(self, s):
        c = self.c
        with np.errstate(invalid="ignore"):
            c.w, c.s = ref.dequantized(c.q.cpu().numpy(), s, c.z.cpu().numpy(), c.K), _dev(s)

    def go(self):
        c, cg = self.c, _cg()
        if self.op == "up":
            cg.moe_w4a16_swiglu(self.x, c.dev_ids, c.q, c.s, c.z, self.y, self.T, self.k, self.E, self.O, self.K)
        else:
            cg.moe_w4a16(self.x, c.dev_ids, self.w, c.q, c.s, c.z, self.y, self.T, self.k, self.E, self.O, self.K, alpha=self.alpha, beta=self.beta)

    def run(self):
        self.y.copy_(self.before)
        self.go()
        return self.y.clone()

    def want(self):
        c, before = self.c, _f64(self.before)[:self.rows]
        if self.op == "up":
            return _up64(_f64(self.x), c.ids, c.w, before)
        return _down64(_f64(self.x), c.ids, None if self.w is None else _f64(self.w), c.w, before, self.alpha, self.beta)

    def check(self, rows=None, columns=slice(None)):
        """The outputs against their definition, the same bits twice, what lies behind as it was."""
        got, again, (want, size) = self.run(), self.run(), self.want()
        rows = np.arange(self.rows) if rows is None else rows
        _close(got.cpu()[rows][:, columns], want[rows][:, columns], "fp16", self.c.slack * size[rows][:, columns])
        assert _bits([got]) == _bits([again])
        assert _bits([got[self.rows:]]) == _bits([self.before[self.rows:]])
        return got


calls = pytest.mark.parametrize("call", plan.CALLS, ids=plan.named)


@calls
def test_values(call):
    c = Call(call, absent=0.1 if call[2] > 2 else 0.0)
    c.check()
    if c.op == "down":  # Y is not read, no weights
        c.beta, c.w = 0.0, None
        c.before[:c.rows] = float("nan")
        got = c.run()
        want, size = _down64(_f64(c.x), c.c.ids, None, c.c.w, np.zeros((c.rows, c.O)), c.alpha, 0.0)
        _close(got[:c.rows], want, "fp16", c.c.slack * size)


@pytest.mark.parametrize("call", [c for c in plan.CALLS if c[0] != "any"], ids=plan.named)
def test_scales_off_a_dword(call):
    """Scales, zero points and ids at odd elements, zero points that the call rounds."""
    Call(call, "offset", offset=16, whole=False).check()


@pytest.mark.parametrize("call", plan.TILES, ids=plan.named)
@pytest.mark.parametrize("by", [0, 1, 2])
def test_tiles_of_every_fill(call, by):
    """Experts with no pair, one, a tile of each size less one, whole, and one more, half a tile and
    one more, the others on the last expert; then all pairs on one."""
    c = Call(call, "fill")
    P, E = c.T * c.k, c.E
    ids = np.full(P, E - 1)
    if by < 2:
        some = [[0, 1, 17, 63, 64, 65, 127, 128, 129, 31, 32, 33], [129, 0, 65, 33, 1, 16, 128, 64, 32]][by]
        at = 0
        for e, n in enumerate(some[:E - 1]):
            n = min(n, P - at)
            ids[at:at + n] = e
            at += n
        c.c.g.shuffle(ids)
    c.ids(ids)
    c.check()


@calls
def test_scales_of_any_size_and_sign(call):
    """Groups with a scale of 0, of either sign, subnormal or large, one after another: accumulators in
    units of the group's scale change it by up to 2^34 from a group to the next, and back."""
    c = Call(call, "scales")
    g = c.c.g
    s = (g.choice([0.0, -0.0, 1.0, -1.0, 2.0 ** -24, -(2.0 ** -20), 0.37, 3.0, 0.01], c.c.s.shape) * 0.05).astype(np.float16)
    s[:, 0] = 0.0  # a row of nothing
    s[:, 1::3, 0] = 0.0  # nothing first, and nothing last
    s[:, 2::3, -1] = 0.0
    c.scales(s)
    c.check()


@calls
def test_rows_that_are_not_finite_stay_alone(call):
    c = Call(call, "nan")
    n = c.x.shape[0]
    bad = sorted({n // 3, n // 2, n - 1}) if n > 3 else [n - 1]
    for i, r in enumerate(bad):
        c.x[r, (37 * (i + 1)) % c.K] = [float("nan"), float("inf"), -float("inf")][i % 3]
    hit = {r * c.k + j for r in bad for j in range(c.k)} if c.op == "up" else {r // c.k for r in bad}
    rows = np.array([r for r in range(c.rows) if r not in hit], int)
    keep = c.x.clone()
    got = c.run()
    assert not np.isfinite(_f64(got[sorted(hit)])).any()
    c.x = keep.nan_to_num(0.0, 0.0, 0.0)
    want, size = c.want()
    if rows.size:
        _close(got[rows], want[rows], "fp16", c.c.slack * size[rows])
    # without a pair that reads it a row does nothing
    c.x = keep
    ids = c.c.ids.copy()
    for r in bad:
        if c.op == "up":
            ids[r] = -1
        else:
            ids.reshape(-1)[r] = c.E
            c.w.view(-1)[r] = float("nan")
    c.ids(ids)
    got = c.run()
    c.x = keep.nan_to_num(0.0, 0.0, 0.0)
    if c.w is not None:
        c.w = c.w.nan_to_num(0.0)
    want, size = c.want()
    _close(got[:c.rows], want, "fp16", c.c.slack * size)


@calls
def test_a_row_does_not_depend_on_others(call):
    """The same bits for a token whatever the others chose, and whatever they hold."""
    c = Call(call, "alone")
    t, per = c.T // 2, c.k if c.op == "up" else 1
    row = slice(t * per, t * per + per)
    want = _bits([c.run()[row]])
    for i in range(3):
        ids = c.c.g.integers(-1, c.E, (c.T, c.k)) if i < 2 else np.full((c.T, c.k), c.c.ids[t, 0])
        ids[t] = c.c.ids[t]
        c.ids(ids)
        keep = c.x.view(c.T, -1)[t].clone()
        c.x.normal_()
        c.x.view(c.T, -1)[t] = keep
        assert _bits([c.run()[row]]) == want, i


@calls
def test_infinite_and_nan_scales_stay_in_their_row(call):
    c = Call(call, "bad-scales")
    s = c.c.s.cpu().numpy()
    s[:, 5, -1], s[:, 9, 0] = np.inf, np.nan
    c.scales(s)
    good = np.array([o for o in range(c.O) if o not in (5, 9)])
    before = c.before.clone()
    got = c.check(columns=good)
    ids = c.c.ids.reshape(-1) if c.op == "up" else c.c.ids.max(1)
    rows = np.flatnonzero(ids >= 0)
    if c.op == "down":
        assert not np.isfinite(_f64(got)[rows][:, [5, 9]]).any()
    else:
        assert np.isnan(_f64(got)[rows][:, 9]).all()
    assert _bits([c.before]) == _bits([before])


@calls
def test_zero_points_that_are_not_finite(call):
    """(q - z) 0 is no number either where z is none: in every kernel the outputs of such a row, and no other."""
    c = Call(call, "bad-zeros")
    s, z = c.c.s.cpu().numpy(), c.c.z.cpu().numpy()
    for row, group, zero, scale in [(3, 0, np.nan, 0.0), (6, -1, np.inf, 0.0), (8, 0, -np.inf, 0.01), (11, -1, np.nan, -0.0)]:
        s[:, row, group], z[:, row, group] = scale, zero
    c.c.z = _dev(z)
    c.scales(s)
    good = np.array([o for o in range(c.O) if o not in (3, 6, 8, 11)])
    got = c.check(columns=good)
    assert not np.isfinite(_f64(got)[:c.rows][:, [3, 6, 8, 11]]).any()


@pytest.mark.parametrize("call", [next(c for c in plan.CALLS if c[:2] == k) for k in sorted({c[:2] for c in plan.CALLS})], ids=plan.named)
def test_graphs_and_workspaces(call):
    """Replays with other ids and rows, and eager work between them; the call in a bound workspace of the
    size that it asks for, and its refusal in a smaller one, before anything is written."""
    import torch
    cg = _cg()
    c = Call(call, "graph")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.go()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.go()
    torch.cuda.synchronize()
    for i in range(3):
        c.x.normal_()
        c.c.dev_ids.copy_(torch.from_numpy(c.c.g.integers(-1, c.E, (c.T, c.k)).astype(np.int32)))
        want = _bits([c.run()])
        c.y.copy_(c.before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert _bits([c.y]) == want, i
    with cg.workspace_query() as q:
        c.go()
    # (a token's places are added up at once, gate and up products by an expert's workgroup; all others need scratch)
    assert (q.bytes == 0) == (c.kernel.startswith("token") or (c.op == "up" and c.kernel in ("expert2", "expert8", "thin", "small"))
                              or (c.op == "up" and c.kernel in ("many", "some") and c.T * c.k <= 2048))
    if q.bytes == 0:
        return
    ws = torch.zeros(q.bytes, dtype=torch.uint8, device="cuda")
    try:
        cg.workspace_bind(ws)
        assert _bits([c.run()]) == want
        for short in (cg.CLOVE_WORKSPACE_MIN_BYTES, q.bytes - 256):
            if not cg.CLOVE_WORKSPACE_MIN_BYTES <= short < q.bytes:
                continue
            cg.workspace_bind(ws[:short])
            c.y.copy_(c.before)
            with pytest.raises(cg.CloveError) as e:
                c.go()
            assert e.value.status == cg.CLOVE_ERR_WORKSPACE
            torch.cuda.synchronize()
            assert _bits([c.y]) == _bits([c.before])
    finally:
        cg.workspace_bind()


def test_parts_of_a_call_are_refused_together():
    """65537 tokens go in two parts: a workspace too small for the first is refused before either has
    written, and one of the size asked for holds both."""
    import torch
    cg = _cg()
    T, k, E, O, K = 65537, 8, 2, 512, 32
    c = Case("refused", 1, k, E, O, K)
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    h = torch.empty(T * k, K, dtype=torch.float16, device="cuda").normal_(generator=g)
    y = torch.full((T, O), 3.0, dtype=torch.float16, device="cuda")

    def down():
        cg.moe_w4a16(h, ids, None, c.q, c.s, c.z, y, T, k, E, O, K)

    with cg.workspace_query() as q:
        down()
    ws = torch.zeros(q.bytes, dtype=torch.uint8, device="cuda")
    try:
        for short in (cg.CLOVE_WORKSPACE_MIN_BYTES, q.bytes // 2, q.bytes - 256):
            cg.workspace_bind(ws[:short])
            with pytest.raises(cg.CloveError) as e:
                down()
            assert e.value.status == cg.CLOVE_ERR_WORKSPACE
            torch.cuda.synchronize()
            assert bool((y == 3.0).all())
        cg.workspace_bind(ws)
        down()
    finally:
        cg.workspace_bind()
    products = torch.stack([h.double() @ w.T.contiguous() for w in torch.from_numpy(c.w).cuda()])
    want = products[ids.flatten().long(), torch.arange(T * k, device="cuda")].view(T, k, O).sum(1)
    # (fp32 leaves at most c.slack of the sizes of 8 x 32 terms; then one rounding)
    room = 2.0 ** -11 * want.abs() + 2.0 ** -25 + c.slack * k * K * float(h.abs().max()) * float(np.abs(c.w).max())
    assert bool(((y.double() - want).abs() <= room).all())
