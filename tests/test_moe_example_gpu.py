"""The decode loop of examples/decode_step.py with sparse MLP blocks: experts that all hold
the dense block's weights give the dense decoder's logits, whichever are chosen."""
import pytest

from tests.test_decode_example_gpu import _example

pytestmark = pytest.mark.gpu


def _decoder(ex, **kw):
    cfg = ex.Config(hidden=256, q_heads=4, kv_heads=2, head_dim=64, inter=512, layers=2, vocab=500, page=8, budget=12, sinks=2, recent=6,
                    longest=100, **kw)
    return ex.Decoder(cfg, 3, seed=3)


def test_equal_experts_are_the_dense_block():
    import torch
    ex = _example()
    dense, sparse = _decoder(ex), _decoder(ex, experts=8, top_k=3)
    sparse.embed, sparse.head = dense.embed, dense.head
    for L, D in zip(sparse.layers, dense.layers):
        for name in ("qkv", "o", "qn", "kn"):
            L[name] = D[name]
        for name in ("up", "down"):
            L[name] = [w[None].expand(8, *w.shape).contiguous() for w in D[name]]
    tokens = torch.randint(0, 500, (10, 3), generator=torch.Generator().manual_seed(1)).cuda()
    for step in tokens:
        want, got = dense.step(step).clone(), sparse.step(step)
        # gate and up are rounded to fp16 in the dense block only, and the shares add up to 1 within 2^-22
        assert float((got - want).abs().max()) <= 0.02 * float(want.abs().max())
        assert all(len(set(row)) == 3 and min(row) >= 0 for row in sparse.chosen.tolist())


def test_generates_with_experts_of_their_own():
    import torch
    ex = _example()
    dec = _decoder(ex, experts=16, top_k=4)
    prompt = torch.randint(0, 500, (3, 5), generator=torch.Generator().manual_seed(2)).cuda()
    made = ex.generate(dec, prompt, 20)
    assert made.shape == (3, 20) and bool((made >= 0).all()) and bool(torch.isfinite(dec.scores).all())
    assert dec.lens.tolist() == [12] * 3
