"""Refusals of the sparse MLP block's entry points of the C ABI (no GPU): the status
comes before anything is read.  Pointers are fake addresses."""
import pytest

from clove_compute_amd import _lib
from clove_compute_amd._lib import (CLOVE_ERR_ALIASING as ALIASING, CLOVE_ERR_INVALID_ARG as ARG, CLOVE_ERR_INVALID_DIM as DIM,
                                    CLOVE_ERR_NULL_POINTER as NULL, CLOVE_OK as OK)
from tests.test_decode_capi import L, TAKEN, _planned, call  # noqa: F401

X, R, W, G, P, Y, H, I, S, Z = (0x10000000 * (i + 1) for i in range(10))

NORM = dict(x=X, x_stride=64, residual=R, residual_stride=64, post_weight=W, gate=G, gate_stride=0, scale=1.0, pre_weight=P, y_out=Y,
            y_out_stride=64, h_out=H, h_out_stride=64, T=4, D=64, eps=1e-6, dtype=0, residual_dtype=0, stream=None)
ROUTE = dict(logits=X, logits_stride=64, dtype=0, bias=None, score=0, groups=1, top_groups=1, group_top=1, top_k=4, renormalize=0,
             scale=1.0, ids=I, weights=W, T=4, experts=64, stream=None)
UP = dict(X=X, ids=I, W_q=W, W_scale=S, W_zero=Z, H=H, T=4, top_k=2, experts=8, I=32, K=256, stream=None)
DOWN = dict(H=H, ids=I, weights=G, W_q=W, W_scale=S, W_zero=Z, Y=Y, T=4, top_k=2, experts=8, O=32, K=256, alpha=1.0, beta=1.0, stream=None)


def test_norm_refusals(L):  # noqa: F811
    f = L.clove_block_norm
    for bad, status in [(dict(T=-1), DIM), (dict(D=-1), DIM), (dict(D=32769), DIM), (dict(dtype=2), ARG), (dict(dtype=-1), ARG),
                        (dict(residual_dtype=1), ARG), (dict(dtype=1, residual_dtype=0), ARG), (dict(x=None, residual=None), NULL),
                        (dict(y_out=None, h_out=None), NULL), (dict(x_stride=63), ARG), (dict(residual_stride=63), ARG), (dict(gate_stride=63), ARG),
                        (dict(y_out_stride=0), ARG), (dict(h_out_stride=63), ARG), (dict(x=X + 1), ARG), (dict(h_out=H + 1), ARG),
                        (dict(residual=R + 2, residual_dtype=2), ARG), (dict(y_out=H), ALIASING), (dict(y_out=X + 2), ALIASING),
                        (dict(h_out=R + 128), ALIASING), (dict(y_out=G), ALIASING), (dict(h_out=P), ALIASING), (dict(h_out=W), ALIASING),
                        (dict(y_out=X, residual_dtype=2), ALIASING), (dict(h_out=R, residual_dtype=2), ALIASING),
                        (dict(y_out=R, y_out_stride=65), ALIASING), (dict(y_out=R, h_out=R), ALIASING)]:
        assert call(f, NORM, **bad) == status, bad
    assert call(f, NORM, T=0, x=None, residual=None) == OK
    assert call(f, NORM, D=0) == OK
    for fine in [dict(), dict(y_out=R), dict(y_out=R, h_out=X), dict(h_out=X), dict(y_out=X), dict(y_out=None), dict(h_out=None), dict(x=None),
                 dict(residual=None), dict(post_weight=None, gate=None, pre_weight=None), dict(gate_stride=64, h_out=G), dict(T=1, y_out=G),
                 dict(y_out=R, residual_dtype=2), dict(T=1, y_out=R, y_out_stride=100), dict(D=32768, x_stride=1 << 20, residual_stride=1 << 20,
                                                                                            y_out_stride=1 << 20, h_out_stride=1 << 20)]:
        assert _planned(L, f, NORM, **fine) in TAKEN, fine


def test_route_refusals(L):  # noqa: F811
    f = L.clove_moe_route
    for bad, status in [(dict(T=-1), DIM), (dict(experts=0), DIM), (dict(experts=1025, logits_stride=2000), DIM), (dict(top_k=0), DIM),
                        (dict(top_k=65, experts=128, logits_stride=128), DIM), (dict(top_k=8, experts=7), ARG), (dict(groups=0), DIM),
                        (dict(top_groups=0), DIM), (dict(groups=3), ARG), (dict(groups=4, top_groups=5), ARG), (dict(group_top=0), ARG),
                        (dict(group_top=3), ARG), (dict(score=2), ARG), (dict(score=-1), ARG), (dict(dtype=3), ARG), (dict(dtype=-1), ARG),
                        (dict(groups=128, experts=128, logits_stride=128), ARG), (dict(logits=None), NULL), (dict(ids=None), NULL),
                        (dict(weights=None), NULL), (dict(logits_stride=63), ARG), (dict(logits=X + 1), ARG), (dict(logits=X + 2, dtype=2), ARG),
                        (dict(bias=P + 2), ARG), (dict(ids=I + 2), ARG), (dict(weights=W + 1), ARG), (dict(ids=X), ALIASING),
                        (dict(weights=X + 64), ALIASING), (dict(ids=W), ALIASING), (dict(bias=W + 32), ALIASING)]:
        assert call(f, ROUTE, **bad) == status, bad
    assert call(f, ROUTE, T=0, logits=None) == OK
    for fine in [dict(), dict(bias=P, score=1, groups=8, top_groups=4, group_top=2), dict(top_k=64), dict(experts=1, top_k=1)]:
        assert _planned(L, f, ROUTE, **fine) in TAKEN, fine


@pytest.mark.parametrize("name", ["clove_moe_w4a16_swiglu", "clove_moe_w4a16"])
def test_product_refusals(L, name):  # noqa: F811
    f, args = getattr(L, name), UP if name.endswith("swiglu") else DOWN
    rows, out, src = ("I", "H", "X") if args is UP else ("O", "Y", "H")
    for bad, status in [(dict(T=-1), DIM), ({rows: -1}, DIM), (dict(K=-2), DIM), (dict(top_k=0), DIM), (dict(top_k=65), DIM),
                        (dict(experts=0), DIM), (dict(experts=1025), DIM), (dict(K=255), ARG), ({src: None}, NULL), (dict(ids=None), NULL),
                        (dict(W_q=None), NULL), (dict(W_scale=None), NULL), (dict(W_zero=None), NULL), ({out: None}, NULL),
                        ({src: args[src] + 1}, ARG), (dict(ids=I + 2), ARG), (dict(W_scale=S + 1), ARG), ({out: args[out] + 1}, ARG),
                        ({out: args[src] + 2}, ALIASING), ({out: W + 64}, ALIASING), ({out: S}, ALIASING), ({out: Z}, ALIASING),
                        ({out: I}, ALIASING), ({rows: 2 ** 31 - 1, "K": 2 ** 31 - 2, "experts": 1024}, DIM), (dict(T=2 ** 31 - 1), DIM),
                        (dict(T=2 ** 25, top_k=32), DIM), ({rows: 2 ** 31 - 64, "K": 2, "experts": 1, "T": 1, "top_k": 1}, DIM)]:
        assert call(f, args, **bad) == status, bad
    assert call(f, args, T=0, ids=None) == OK
    assert call(f, args, **{rows: 0}) == OK
    if args is DOWN:
        assert call(f, args, weights=G + 2) == ARG
        assert call(f, args, Y=G) == ALIASING
        assert _planned(L, f, args, weights=None) in TAKEN
    for fine in [dict(), dict(K=0, W_q=None), dict(K=254), dict(W_q=W + 1)]:
        assert _planned(L, f, args, **fine) in TAKEN, fine
