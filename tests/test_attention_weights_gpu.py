"""What a softmax weight loses on its way into paged_attention's sum over the values.

Every other error is kept out of the way: scores are one exact product, so that
the weights are known to a few 2^-24, and outputs are small against their terms,
or judged relative to themselves, so that their own rounding does not cover what
the weights have lost.
"""
import numpy as np
import pytest

from tests import _decode_ref as ref

pytestmark = pytest.mark.gpu


def _cg():
    import clove_compute_amd as cg
    return cg


def _run(dtype, q, k, v, n, scale):
    """q [H, D], k, v [H, n, D] of one sequence with as many KV heads as query heads,
    in the element type `dtype`: the output, and the values that it had as inputs."""
    import torch
    cg = _cg()
    t = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    H, D = q.shape
    P = 16
    pages = -(-n // P)
    cache = torch.zeros(2, pages, H, P, D, dtype=t, device="cuda")
    for x, y in zip(cache, (k, v)):
        y = torch.from_numpy(np.ascontiguousarray(y, np.float32)).cuda().to(t)
        for j in range(pages):
            rows = y[:, j * P:(j + 1) * P]
            x[j, :, :rows.shape[1]] = rows
    dq = torch.from_numpy(np.ascontiguousarray(q, np.float32)).cuda().to(t)[None]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = torch.empty_like(dq)
    cg.paged_attention(dq, cg.KVCache(cache[0], cache[1]), table, lens, out, 1, H, n, scale=scale)
    f64 = lambda x: x.double().cpu().numpy()  # noqa: E731
    return f64(out)[0], f64(dq), [f64(x) for x in cache], table.cpu().numpy()


@pytest.mark.parametrize("n", [2, 40, 300])
@pytest.mark.parametrize("dtype,half", [("fp16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
def test_weights_keep_their_bits(dtype, half, n):
    """Two keys' values that nearly cancel: with weights 1 and p, the output is
    (a + b p) / (1 + p), a = -b p rounded to the element type.  The other keys have
    the weight 0 (their scores lie 300 below, in base 2).

    p is off by 3 roundings of the score's factors (|t| <= 1, times ln 2) and one of
    the exponential, 4.1 x 2^-24 of it; the sums of up to three products by at most
    2^-23 each: 10.1 x 2^-24 of |b| p.
    """
    H, D = 16, 128
    scale = float(np.float32(np.log(2.0)))
    f = np.arange(1, H + 1) / 17.0
    f = np.round(f * 128) / 128  # eight bits: both types hold them
    q, k, v = np.zeros((H, D)), np.zeros((H, n, D)), np.zeros((H, n, D))
    q[:, 0] = f
    q[:, 1] = 1.0
    k[:, 1, 0] = -1.0
    k[:, 2:, 1] = -300.0
    p = np.exp(-f * scale)
    b = 1.0 + np.arange(D) / 128.0
    v[:, 1] = b
    import torch
    t = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    v[:, 0] = -torch.from_numpy(p[:, None] * b).to(t).double().numpy()
    v[:, 2:] = 1.0
    got, q64, (k64, v64), table = _run(dtype, q, k, v, n, scale)
    want, _ = ref.attention(q64, k64, v64, table, [n], scale)
    want = want[0]
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    bound = half * np.abs(want) * 1.0001 + tiny + 10.1 * 2.0 ** -24 * b * p[:, None] / (1 + p[:, None])
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))


@pytest.mark.parametrize("dtype,half", [("fp16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
@pytest.mark.parametrize("n,below", [(30, 15), (200, 14), (500, 12), (500, 14), (500, 16), (500, 20), (4096, 16), (4096, 18), (4096, 24), (40000, 18),
                                     (40000, 25)])
def test_weights_far_below_the_largest(dtype, half, n, below):
    """One key `below` above the others in base 2, its value 0: the output is what the
    others' weights of about 2^-below bring, judged relative to itself.

    A weight is off by 3 roundings of its score's factors (|t| < below + 1, times
    ln 2) and one of the exponential; fp16 holds it to 2^-40 of the largest; a lane
    or a matrix product adds at most 2048 of them one after the other, and joins of
    up to 400 parts follow, 2^-24 each.
    """
    H, D = 4, 64
    scale = float(np.float32(np.log(2.0)))
    g = np.random.default_rng(n + below)
    q, k = np.zeros((H, D)), np.zeros((H, n, D))
    q[:, 0] = 1.0
    k[:, :, 0] = -(below + g.integers(0, 8, (H, n)) / 8.0)
    v = g.uniform(2.0, 6.0, (H, n, D))
    at = n // 3
    k[:, at, 0], v[:, at] = 0.0, 0.0
    got, q64, (k64, v64), table = _run(dtype, q, k, v, n, scale)
    want = ref.attention(q64, k64, v64, table, [n], scale)[0][0]
    slack = (3 * (below + 1) * 0.694 + 2 + min(n, 2048) + 400) * 2.0 ** -24 + (2.0 ** (below + 1 - 40) if dtype == "fp16" else 0.0)
    bound = (half * 1.0001 + slack) * np.abs(want) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / np.abs(want)))
