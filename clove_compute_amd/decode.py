"""The decode step around the linear layers: query / key norms with rotation and
the cache write, attention over the paged cache, eviction from it, and the
penalties and masks on the logits.

Buffers are torch tensors on the current HIP device, passed with their sizes as
in ``gemm``; every call goes through the C ABI (include/clove/gemm_c.h states
the formulas), is asynchronous on ``stream`` (default: torch's current stream)
and raises CloveError where the library refuses it.  What the C ABI cannot see
-- device (the current one), element type, number of elements, inner strides -- is
checked on the way (ValueError), in compiled code: it is most of a small call's
time.  A tensor's rows may be further apart than they are long; the elements of a
row are adjacent.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os

from . import _lib

_CODES = {"torch.float16": _lib.CLOVE_DTYPE_FP16, "torch.bfloat16": _lib.CLOVE_DTYPE_BF16,
          "torch.float32": _lib.CLOVE_DTYPE_FP32}


class _Bound:
    """The compiled entry points, looked up on the first call: importing torch and
    loading the library take long, and resolving a name a microsecond a call."""

    def __getattr__(self, name):
        import torch  # noqa: F401  (the module is linked to its libraries)
        lib, path = _lib.lib(), os.path.join(os.path.dirname(__file__), "lib", "_decode.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build the HIP library first "
                               "(python -c 'import __graft_entry__ as g; g.build()')")
        loader = importlib.machinery.ExtensionFileLoader("_decode", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_decode", loader))
        loader.exec_module(module)
        module.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in
                      (lib.clove_qk_norm_rope, lib.clove_paged_attention, lib.clove_cache_evict, lib.clove_penalize_logits)))
        self.rope, self.attend, self.evict, self.penalize = (module.qk_norm_rope, module.paged_attention, module.cache_evict,
                                                             module.penalize_logits)
        return self.__dict__[name]


_b = _Bound()


class _CacheAt(_lib.KVCacheDesc):
    """What the compiled module takes: the description and the device of its tensors."""
    _fields_ = [("device", ctypes.c_int)]


class KVCache:
    """The paged key-value cache of one layer: ``k``, ``v``
    [num_pages, kv_heads, page_size, head_dim], fp16 or bf16.  Pages are dense
    inside; they may lie further apart than they are long (the same distance in
    both), as in one allocation [num_pages, 2, kv_heads, page_size, head_dim].
    Keeps the tensors; a program makes one per layer and keeps it."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v are tensors [num_pages, kv_heads, page_size, head_dim] of one shape and type")
        if k.shape[0] and not (k[0].is_contiguous() and v[0].is_contiguous()):
            raise ValueError("the pages of k and v must be dense")
        if k.shape[0] > 1 and k.stride(0) != v.stride(0):
            raise ValueError("the pages of k and v must be equally far apart")
        if k.shape[0] > 1 and k.stride(0) < k[0].numel():  # (the library takes 0 for dense pages)
            raise ValueError("the pages of k and v must lie apart: an expanded tensor has one page only")
        if not (k.is_cuda and v.is_cuda and k.device == v.device):
            raise ValueError("k and v must be on the GPU, on the same one")
        if str(k.dtype) not in _CODES:
            raise ValueError(f"element type {k.dtype} is not fp16, bf16 or fp32")
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype = k.dtype
        self._c = _CacheAt(k.data_ptr(), v.data_ptr(), k.stride(0) if k.shape[0] > 1 else 0, self.num_pages, self.page_size,
                           self.kv_heads, self.head_dim, _CODES[str(k.dtype)], k.get_device())
        self._at = ctypes.addressof(self._c)


def qk_norm_rope(qkv, q_weight, k_weight, cos, sin, positions, q_out, T: int, q_heads: int, kv_heads: int,
                 head_dim: int, rot_dim: int = None, eps: float = 1e-6, interleaved: bool = False, k_out=None,
                 cache: KVCache = None, slots=None, stream=None) -> None:
    """Per-head RMS norm of queries and keys (where the weight is given), rotation of their first
    ``rot_dim`` (default: all) elements by ``cos`` / ``sin`` [max_position, rot_dim / 2] at
    ``positions`` [T], and the write of keys and values into ``slots`` [T] of ``cache``: one pass
    over the fused projection's rows ``qkv`` [T, (q_heads + 2 kv_heads) head_dim]."""
    st = _b.rope(qkv, q_weight, k_weight, cos, sin, positions, q_out, T, q_heads, kv_heads, head_dim, rot_dim, eps,
                 interleaved, k_out, None if cache is None else cache._at, slots, stream)
    if st:
        _lib.check(st, "qk_norm_rope")


def paged_attention(q, cache: KVCache, block_table, context_lens, out, batch: int, q_heads: int, max_context: int,
                    scale: float = None, softcap: float = 0.0, window: int = 0, weights=None, stream=None) -> None:
    """out = softmax(scale q k^T) v of one new token per sequence over the pages of
    ``block_table`` [batch, pages], ``context_lens`` [batch] keys each (at most ``max_context``).
    ``scale`` defaults to head_dim ** -0.5; ``window`` > 0 sees the last keys only; ``softcap`` > 0
    bounds the scores; ``weights`` [batch, max_context] fp32 gains each key's softmax weight,
    summed over the heads."""
    st = _b.attend(q, cache._at, block_table, context_lens, out, batch, q_heads, max_context,
                   cache.head_dim ** -0.5 if scale is None else scale, softcap, window, weights, stream)
    if st:
        _lib.check(st, "paged_attention")


def cache_evict(cache: KVCache, block_table, context_lens, weights, positions, weights_out, positions_out, lens_out,
                batch: int, max_context: int, budget: int, sinks: int = 0, recent: int = 0, stream=None) -> None:
    """Cuts every sequence of the cache down to ``budget`` tokens, in place: those of the first
    ``sinks`` and the newest ``recent`` positions stay, then those of the largest ``weights``
    [batch, max_context]; kept tokens past the budget move into the holes below it.  Outputs hold the
    new weights, positions and lengths, and may be the inputs."""
    st = _b.evict(cache._at, block_table, context_lens, weights, positions, weights_out, positions_out, lens_out, batch,
                  max_context, budget, sinks, recent, stream)
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
    st = _b.penalize(logits, out, batch, vocab, history, history_lens, prompt_lens, repetition, presence, frequency, bias_ids,
                     bias_values, bias_counts, allowed, stream)
    if st:
        _lib.check(st, "penalize_logits")
