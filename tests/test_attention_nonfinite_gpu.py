"""Infinite and NaN values under paged_attention: out = sum p v as the arithmetic has it,
in every form of the kernel.  Infinities of one sign give that infinity, of both
signs NaN, a NaN its own element, and what no key names does not count."""
import numpy as np
import pytest

from tests import _decode_ref as ref
from tests.test_decode_gpu import _attend, _close, _cg, _dev, _f64, _paged, _rounded
from tests._util import rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,Hq,Hk,D,longest", [
    ([20, 7], 4, 2, 64, 20),       # one wave a sequence
    ([200, 90], 4, 2, 64, 200),    # eight
    ([120, 40], 4, 1, 128, 120),   # four, not split
    ([3000, 700], 4, 2, 64, 3000),  # split
    ([3000, 700], 32, 1, 36, 3000),  # split, rows at any alignment, two tiles of heads
    ([300, 90], 4, 2, 256, 300),
    ([70, 33], 2, 1, 5, 70),       # without the matrix cores
    ([70, 33], 2, 1, 320, 70)])
def test_infinite_and_nan_values(dtype, lens, Hq, Hk, D, longest):
    cg = _cg()
    g = rng("values-inf", tuple(lens), Hq, D)
    P = 16
    k, v, k64, v64, table = _paged(g, dtype, lens, Hk, D, P)
    q, q64 = _rounded(g, dtype, len(lens), Hq, D)
    scale = D ** -0.5
    first = ref.attention(q64, k64, v64, table, lens, scale)

    def put(b, j, h, d, x):
        v[table[b, j // P], h, j % P, d] = v64[table[b, j // P], h, j % P, d] = x

    n, last = lens[0], Hk - 1
    # the largest weight of a query, whose parts past the first are 0; the smallest; any
    s = np.array([k64[table[0, j // P], last, j % P] @ q64[0, -1] for j in range(n)])
    put(0, int(s.argmax()), last, 0, np.inf)
    put(0, int(s.argmin()), last, 1, -np.inf)
    put(0, n // 2, last, 2, np.inf)
    put(0, n // 3, last, 3, np.nan)
    put(0, 0, last, 4, np.inf)       # both signs
    put(0, n - 1, last, 4, -np.inf)
    put(1, lens[1] - 1, 0, D - 1, -np.inf)
    with np.errstate(invalid="ignore"):
        want, added = ref.attention(q64, k64, v64, table, lens, scale)
    assert np.isposinf(want[0, -1, 0]) and np.isneginf(want[0, -1, 1]) and np.isnan(want[0, -1, 3:5]).all()
    w = _dev(np.zeros((len(lens), longest), np.float32))
    out = _attend(cg, q, cg.KVCache(k, v), table, lens, len(lens), Hq, longest, weights=w)
    finite = np.abs(v64[np.isfinite(v64)]).max()
    _close(out, want, dtype, 3e-5 * float(finite))
    assert np.array_equal(added, first[1])
    assert np.all(np.abs(_f64(w) - added[:, :longest]) <= 3e-5 * added[:, :longest] + 1e-9)
