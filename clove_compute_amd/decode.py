"""The decode step around the linear layers: query / key norms with rotation and
the cache write, attention over the paged cache, eviction from it, and the
penalties and masks on the logits.

Buffers are torch tensors on the current HIP device, passed with their sizes as
in ``gemm``; every call goes through the C ABI (include/clove/gemm_c.h states
the formulas), is asynchronous on ``stream`` (default: torch's current stream)
and raises CloveError where the library refuses it.  What the C ABI cannot see
-- device, element type, number of elements, inner strides -- is checked here
(ValueError).  A tensor's rows may be further apart than they are long; the
elements of a row are adjacent.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .gemm import _stream

class _Bound:
    """What every call needs, looked up on the first: the library's functions and
    torch's element types (importing torch and resolving a function by name cost
    a microsecond a call, a third of what the smallest kernels take)."""

    def __getattr__(self, name):
        import torch
        lib = _lib.lib()
        self.f16, self.f32, self.i32 = torch.float16, torch.float32, torch.int32
        self.codes = {torch.float16: _lib.CLOVE_DTYPE_FP16, torch.bfloat16: _lib.CLOVE_DTYPE_BF16,
                      torch.float32: _lib.CLOVE_DTYPE_FP32}
        self.rope, self.attend = lib.clove_qk_norm_rope, lib.clove_paged_attention
        self.evict, self.penalize = lib.clove_cache_evict, lib.clove_penalize_logits
        return self.__dict__[name]


_b = _Bound()


def _code(dtype) -> int:
    c = _b.codes.get(dtype)
    if c is None:
        raise ValueError(f"element type {dtype} is not fp16, bf16 or fp32")
    return c


def _rows(x, name, rows, width, dtype):
    """(address, row stride) of a tensor read as `rows` rows of `width` adjacent
    elements; its first dimension is the row where it has more than one."""
    if x.dtype is not dtype or not x.is_cuda:
        raise ValueError(f"{name} must be {dtype} on the GPU, not {x.dtype} on {x.device}")
    if x.numel() == rows * width and x.is_contiguous():
        return x.data_ptr(), width
    shape, strides = x.shape, x.stride()
    n, inner = shape[0] if shape else 1, 1
    if len(shape) < 2:
        n, shape, strides = 1, (1, *shape), (n, *strides)
    for size, stride in zip(shape[:0:-1], strides[:0:-1]):
        if size != 1 and stride != inner:
            inner = -1
            break
        inner *= size
    if n < rows or inner < width:
        raise ValueError(f"{name} holds {tuple(x.shape)} elements, {rows} rows of {width} adjacent ones are wanted")
    return x.data_ptr(), strides[0] if rows > 1 else max(width, strides[0])


def _lists(x, name, rows, dtype):
    """(address, length) of equally long lists one after another: how far apart they
    lie tells the library how long they are, so no part of longer ones is taken."""
    n = x.shape[-1]
    p, apart = _rows(x, name, rows, n, dtype)
    if rows > 1 and apart != n:
        raise ValueError(f"the rows of {name} must follow one another, not {n} elements every {apart}")
    return p, n


def _flat(x, name, n, dtype):
    """Address of at least `n` adjacent elements (None stays None)."""
    if x is None:
        return None
    if x.dtype is not dtype or not x.is_cuda or x.numel() < n or not x.is_contiguous():
        raise ValueError(f"{name} must be {n} adjacent {dtype} elements on the GPU, not {tuple(x.shape)} {x.dtype}")
    return x.data_ptr()


class KVCache:
    """The paged key-value cache of one layer: ``k``, ``v``
    [num_pages, kv_heads, page_size, head_dim], fp16 or bf16.  Pages are dense
    inside; they may lie further apart than they are long (the same distance in
    both), as in one allocation [num_pages, 2, kv_heads, page_size, head_dim].
    Keeps the tensors; a program makes one per layer and keeps it."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or not (k.is_cuda and v.is_cuda):
            raise ValueError("k and v are GPU tensors [num_pages, kv_heads, page_size, head_dim] of one shape and type")
        if k.shape[0] and not (k[0].is_contiguous() and v[0].is_contiguous()):
            raise ValueError("the pages of k and v must be dense")
        if k.shape[0] > 1 and k.stride(0) != v.stride(0):
            raise ValueError("the pages of k and v must be equally far apart")
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype = k.dtype
        self._c = _lib.KVCacheDesc(k.data_ptr(), v.data_ptr(), k.stride(0) if k.shape[0] > 1 else 0, self.num_pages,
                                   self.page_size, self.kv_heads, self.head_dim, _code(k.dtype))
        self._ref = ctypes.byref(self._c)


def qk_norm_rope(qkv, q_weight, k_weight, cos, sin, positions, q_out, T: int, q_heads: int, kv_heads: int,
                 head_dim: int, rot_dim: int = None, eps: float = 1e-6, interleaved: bool = False, k_out=None,
                 cache: KVCache = None, slots=None, stream=None) -> None:
    """Per-head RMS norm of queries and keys (where the weight is given), rotation of their first
    ``rot_dim`` (default: all) elements by ``cos`` / ``sin`` [max_position, rot_dim / 2] at
    ``positions`` [T], and the write of keys and values into ``slots`` [T] of ``cache``: one pass
    over the fused projection's rows ``qkv`` [T, (q_heads + 2 kv_heads) head_dim]."""
    R = head_dim if rot_dim is None else rot_dim
    dt, i, half, most = qkv.dtype, _b.i32, R // 2, 0
    x, xs = _rows(qkv, "qkv", T, (q_heads + 2 * kv_heads) * head_dim, dt)
    q, qs = _rows(q_out, "q_out", T, q_heads * head_dim, dt)
    k, ks = _rows(k_out, "k_out", T, kv_heads * head_dim, dt) if k_out is not None else (None, 0)
    c = s = None
    if R:
        most = cos.shape[0]
        c, s = _flat(cos, "cos", most * half, _b.f32), _flat(sin, "sin", most * half, _b.f32)
        if cos.numel() != most * half or sin.shape != cos.shape:
            raise ValueError(f"cos and sin are [max_position, {half}], not {tuple(cos.shape)} and {tuple(sin.shape)}")
    st = _b.rope(x, xs, _flat(q_weight, "q_weight", head_dim, dt), _flat(k_weight, "k_weight", head_dim, dt), eps, c, s, most,
                 _flat(positions, "positions", T, i) if R else None, q, qs, k, ks, None if cache is None else cache._ref,
                 _flat(slots, "slots", T, i), T, q_heads, kv_heads, head_dim, R, interleaved, _code(dt), _stream(stream))
    if st:
        _lib.check(st, "qk_norm_rope")


def paged_attention(q, cache: KVCache, block_table, context_lens, out, batch: int, q_heads: int, max_context: int,
                    scale: float = None, softcap: float = 0.0, window: int = 0, weights=None, stream=None) -> None:
    """out = softmax(scale q k^T) v of one new token per sequence over the pages of
    ``block_table`` [batch, pages], ``context_lens`` [batch] keys each (at most ``max_context``).
    ``scale`` defaults to head_dim ** -0.5; ``window`` > 0 sees the last keys only; ``softcap`` > 0
    bounds the scores; ``weights`` [batch, max_context] fp32 gains each key's softmax weight,
    summed over the heads."""
    D, dt, i = cache.head_dim, cache.dtype, _b.i32
    x, xs = _rows(q, "q", batch, q_heads * D, dt)
    o, os_ = _rows(out, "out", batch, q_heads * D, dt)
    t, ts = _rows(block_table, "block_table", batch, -(-max_context // cache.page_size), i)
    w, ws = _rows(weights, "weights", batch, max_context, _b.f32) if weights is not None else (None, 0)
    st = _b.attend(x, xs, cache._ref, t, ts, _flat(context_lens, "context_lens", batch, i), o, os_, w, ws, batch, q_heads,
                   max_context, D ** -0.5 if scale is None else scale, softcap, window, _stream(stream))
    if st:
        _lib.check(st, "paged_attention")


def cache_evict(cache: KVCache, block_table, context_lens, weights, positions, weights_out, positions_out, lens_out,
                batch: int, max_context: int, budget: int, sinks: int = 0, recent: int = 0, stream=None) -> None:
    """Cuts every sequence of the cache down to ``budget`` tokens, in place: those of the first
    ``sinks`` and the newest ``recent`` positions stay, then those of the largest ``weights``
    [batch, max_context]; kept tokens past the budget move into the holes below it.  Outputs hold the
    new weights, positions and lengths, and may be the inputs."""
    f, i = _b.f32, _b.i32
    t, ts = _rows(block_table, "block_table", batch, -(-max_context // cache.page_size), i)
    w, ws = _rows(weights, "weights", batch, max_context, f)
    p, ps = _rows(positions, "positions", batch, max_context, i)
    wo, wos = _rows(weights_out, "weights_out", batch, max_context, f)
    po, pos = _rows(positions_out, "positions_out", batch, max_context, i)
    st = _b.evict(cache._ref, t, ts, _flat(context_lens, "context_lens", batch, i), w, ws, p, ps, wo, wos, po, pos,
                  _flat(lens_out, "lens_out", batch, i), batch, max_context, budget, sinks, recent, _stream(stream))
    if st:
        _lib.check(st, "cache_evict")


def penalize_logits(logits, out, batch: int, vocab: int, history=None, history_lens=None, prompt_lens=None,
                    repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None, bias_counts=None,
                    allowed=None, stream=None) -> None:
    """out = logits [batch, vocab] after the repetition penalty of every token of ``history``
    (divided where positive, multiplied where not), the frequency and presence penalties of its part
    past ``prompt_lens``, the biases of ``bias_ids`` / ``bias_values`` (the last entry for a token
    counts) and the mask ``allowed`` [batch, ceil(vocab / 32)] (int32 words, token v is bit v % 32;
    a clear bit gives -inf).  The rows of ``history`` and of the bias lists follow one another;
    those of the others may lie apart.  fp32 inside; ``out`` is fp32 or of the logits' type."""
    f, i = _b.f32, _b.i32
    x, xs = _rows(logits, "logits", batch, vocab, logits.dtype)
    o, os_ = _rows(out, "out", batch, vocab, out.dtype)
    h = b = bv = m = None
    hs = bs = ms = 0
    if history is not None:
        h, hs = _lists(history, "history", batch, i)
    if bias_ids is not None:
        b, bs = _lists(bias_ids, "bias_ids", batch, i)
        bv, ms = _lists(bias_values, "bias_values", batch, f)
        if ms != bs:
            raise ValueError("bias_ids and bias_values must be equally long")
    if allowed is not None:
        m, ms = _rows(allowed, "allowed", batch, -(-vocab // 32), i)
    st = _b.penalize(x, xs, _code(logits.dtype), o, os_, _code(out.dtype), batch, vocab, h, hs,
                     _flat(history_lens, "history_lens", batch, i), _flat(prompt_lens, "prompt_lens", batch, i),
                     _flat(repetition, "repetition", batch, f), _flat(presence, "presence", batch, f),
                     _flat(frequency, "frequency", batch, f), b, bv, bs, _flat(bias_counts, "bias_counts", batch, i), m, ms,
                     _stream(stream))
    if st:
        _lib.check(st, "penalize_logits")
