"""paged_attention behind bounds that call for more workgroups than there is room for,
and with more sequences than are cut at all.  The long sequences have the same pages
again and again: each key weighs as much as its like, so that the result is that of one
round of the pages."""
import numpy as np
import pytest

from tests import _decode_ref as ref
from tests._util import rng
from tests.test_decode_gpu import _attend, _cg, _close, _dev, _rounded

pytestmark = pytest.mark.gpu

P, ROUND = 64, 4  # rows of a page, pages of a round


def _case(name, lens, Hq, Hk, D, longest, dtype):
    """lens: of whole rounds, or of at most one.  The cache, tables and what comes out."""
    g = rng(name, len(lens), D)
    B = len(lens)
    k, k64 = _rounded(g, dtype, 3 * ROUND, Hk, P, D)
    v, v64 = _rounded(g, dtype, 3 * ROUND, Hk, P, D)
    q, q64 = _rounded(g, dtype, B, Hq, D, scale=1.5)
    own = np.stack([g.permutation(3 * ROUND)[:ROUND] for _ in range(B)]).astype(np.int32)
    pages = -(-longest // P)
    table = np.tile(own, (1, -(-pages // ROUND)))[:, :pages]
    at = [min(n, ROUND * P) for n in lens]
    assert all(n <= ROUND * P or n % (ROUND * P) == 0 for n in lens)
    want, added = ref.attention(q64, k64, v64, own, at, D ** -0.5)
    return _cg().KVCache(k, v), q, table, want, added, float(np.abs(v64).max())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Hq,Hk,D,longest,kind", [
    (32, 8, 8, 128, 131072, "one long"), (48, 8, 8, 64, 131072, "one long"), (32, 8, 8, 16, 131072, "all long"),
    (32, 4, 4, 12, 262144, "all long"), (1000, 8, 8, 16, 10240, "one long"), (900, 10, 10, 8, 5120, "mixed")])
def test_room_for_fewer_workgroups_than_the_bound_asks_for(B, Hq, Hk, D, longest, kind, dtype):
    g = rng("bounds", B, D, kind)
    one = ROUND * P
    if kind == "one long":
        lens = [int(n) for n in g.integers(0, one + 1, B)]
        lens[B // 3] = longest // one * one
    elif kind == "all long":
        lens = [longest // one * one] * B
    else:
        lens = [int(n) * one for n in g.integers(0, longest // one + 1, B)]
    cache, q, table, want, added, most = _case("bounds" + kind, lens, Hq, Hk, D, longest, dtype)
    out = _attend(_cg(), q, cache, table, lens, B, Hq, longest)
    _close(out, want, dtype, 3e-5 * most)
