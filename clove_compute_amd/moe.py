"""A sparse MLP block around the linear layers: the norms before and after a
block with its residual, the router, and the products of the experts it chose
on INT4 weights.

Tensors, sizes, streams and errors as in ``decode``; include/clove/gemm_c.h states
the formulas.
"""
from __future__ import annotations

from . import _lib
from .decode import _b


def block_norm(x, residual, h_out, T: int, D: int, y_out=None, post_weight=None, pre_weight=None, gate=None,
               scale: float = 1.0, eps: float = 1e-6, stream=None) -> None:
    """y = residual + scale * gate * norm(x; post_weight), h = norm(y; pre_weight), rows [T, D] of the
    residual stream (the type of x, or fp32).  ``post_weight`` None: x is not normed; ``pre_weight``
    None: weight 1; ``gate`` [D] (one row for all) or [T, D]; ``x`` None: y = residual; ``residual`` None: 0.  ``y_out`` or
    ``h_out`` may be None; they may be the residual and x themselves."""
    st = _b.block_norm(x, residual, h_out, T, D, y_out, post_weight, pre_weight, gate, scale, eps, stream)
    if st:
        _lib.check(st, "block_norm")


def moe_route(logits, ids, weights, T: int, experts: int, top_k: int, score: int = _lib.CLOVE_ROUTE_SOFTMAX, bias=None,
              groups: int = 1, top_groups: int = 1, group_top: int = 1, renormalize: bool = False, scale: float = 1.0,
              stream=None) -> None:
    """``ids`` [T, top_k] int32 and ``weights`` [T, top_k] fp32 of the experts chosen from ``logits`` [T, experts]:
    those of the largest logit, or with ``bias`` [experts] fp32 of the largest score + bias, largest first,
    out of the ``top_groups`` of ``groups`` groups whose ``group_top`` largest add up to most.  -1 and 0 where
    no expert is left.  The weights are the scores, divided by their sum where ``renormalize``, times ``scale``."""
    st = _b.moe_route(logits, ids, weights, T, experts, top_k, score, bias, groups, top_groups, group_top, renormalize, scale, stream)
    if st:
        _lib.check(st, "moe_route")


def moe_w4a16_swiglu(X, ids, W_q, W_scale, W_zero, H, T: int, top_k: int, experts: int, I: int, K: int, stream=None) -> None:
    """H [T top_k, I] = swiglu of the gate and up products of each row of X [T, K] with the experts ``ids``
    [T, top_k]: W_q [experts, 2I, K/2] (gate rows first), W_scale / W_zero [experts, 2I, ceil(K/128)].  Rows of H
    whose id is no expert are left as they are."""
    st = _b.moe_up(X, ids, W_q, W_scale, W_zero, H, T, top_k, experts, I, K, stream)
    if st:
        _lib.check(st, "moe_w4a16_swiglu")


def moe_w4a16(H, ids, weights, W_q, W_scale, W_zero, Y, T: int, top_k: int, experts: int, O: int, K: int, alpha: float = 1.0,
              beta: float = 0.0, stream=None) -> None:
    """Y [T, O] = alpha * sum_j weights[t, j] * (H[t top_k + j] @ W[ids[t, j]]^T) + beta * Y: W_q [experts, O, K/2],
    W_scale / W_zero [experts, O, ceil(K/128)], ``weights`` [T, top_k] fp32 or None (1)."""
    st = _b.moe_down(H, ids, weights, W_q, W_scale, W_zero, Y, T, top_k, experts, O, K, alpha, beta, stream)
    if st:
        _lib.check(st, "moe_w4a16")
