"""Refusals of the decode-step entry points of the C ABI (no GPU): the status
comes before anything is read.  Pointers are fake addresses."""
import ctypes

import pytest

from clove_compute_amd import _lib
from clove_compute_amd._lib import (CLOVE_ERR_ALIASING as ALIASING, CLOVE_ERR_INVALID_ARG as ARG, CLOVE_ERR_INVALID_DIM as DIM,
                                    CLOVE_ERR_NULL_POINTER as NULL, CLOVE_OK as OK)

K, V, Q, O, W, T, N = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000, 0x60000000, 0x70000000
X, Y, Z = 0x80000000, 0x90000000, 0xa0000000


@pytest.fixture(scope="module")
def L():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import clove_compute_amd.build as b
        b.build()
    return _lib.lib()


def cache(**kw):
    d = dict(k=K, v=V, page_stride=0, num_pages=8, page_size=16, kv_heads=2, head_dim=64, dtype=0)
    d.update(kw)
    return ctypes.byref(_lib.KVCacheDesc(**d))


def call(fn, args, **kw):
    """`args` with some of them replaced by name."""
    a = dict(args)
    assert set(kw) <= set(a), set(kw) - set(a)
    a.update(kw)
    return fn(*a.values())


ROPE = dict(qkv=X, qkv_stride=512, q_weight=Y, k_weight=Y, eps=1e-6, cos=Z, sin=Z + 0x100000, max_position=100, positions=N, q_out=Q,
            q_out_stride=256, k_out=O, k_out_stride=128, cache=None, slots=T, T=4, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64,
            interleaved=0, dtype=0, stream=None)
ATTEND = dict(q=Q, q_stride=256, cache=None, block_table=T, table_stride=8, context_lens=N, out=O, out_stride=256, weights=None,
              weights_stride=0, batch=4, q_heads=4, max_context=100, scale=0.1, softcap=0.0, window=0, stream=None)
EVICT = dict(cache=None, block_table=T, table_stride=8, context_lens=N, weights=W, weights_stride=100, positions=X, positions_stride=100,
             weights_out=Y, weights_out_stride=100, positions_out=Z, positions_out_stride=100, lens_out=O, batch=4, max_context=100,
             budget=50, sinks=4, recent=8, stream=None)
LOGITS = dict(logits=X, logits_stride=1000, dtype=0, out=Y, out_stride=1000, out_dtype=0, batch=2, vocab=1000, history=T, history_stride=50,
              history_lens=N, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None,
              bias_stride=0, bias_counts=None, allowed=None, allowed_stride=0, stream=None)


def test_cache_descriptor(L):
    f = L.clove_paged_attention
    for bad, status in [(dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(page_size=0), DIM), (dict(kv_heads=0), DIM), (dict(head_dim=0), DIM),
                        (dict(head_dim=1025), DIM), (dict(num_pages=-1), DIM), (dict(page_stride=2047), ARG), (dict(k=None), NULL),
                        (dict(v=None), NULL), (dict(k=K + 1), ARG), (dict(page_size=2 ** 31 - 1, kv_heads=2 ** 31 - 1), DIM)]:
        assert call(f, ATTEND, cache=cache(**bad)) == status, bad
    assert call(f, ATTEND, cache=None) == NULL


def test_rope_refusals(L):
    f = L.clove_qk_norm_rope
    for bad, status in [(dict(T=-1), DIM), (dict(q_heads=-1), DIM), (dict(head_dim=0), DIM), (dict(head_dim=1025), DIM), (dict(rot_dim=-2), DIM),
                        (dict(rot_dim=63), ARG), (dict(rot_dim=66), ARG), (dict(dtype=2), ARG), (dict(qkv=None), NULL), (dict(q_out=None), NULL),
                        (dict(cos=None), NULL), (dict(positions=None), NULL), (dict(qkv_stride=511), ARG), (dict(q_out_stride=255), ARG),
                        (dict(k_out_stride=127), ARG), (dict(qkv=X + 1), ARG), (dict(cos=Z + 2), ARG), (dict(q_out=X + 2), ALIASING),
                        (dict(q_out=X), ALIASING), (dict(k_out=X, k_out_stride=512), ALIASING), (dict(q_out=O), ALIASING), (dict(q_out=Y), ALIASING),
                        (dict(cache=cache(), slots=None), NULL), (dict(cache=cache(head_dim=32)), ARG), (dict(cache=cache(kv_heads=1)), ARG),
                        (dict(cache=cache(dtype=1)), ARG), (dict(cache=cache(k=X)), ALIASING), (dict(cache=cache(v=K)), ALIASING),
                        (dict(cache=cache(k=Q)), ALIASING)]:
        assert call(f, ROPE, **bad) == status, bad
    assert call(f, ROPE, T=0, qkv=None) == OK
    assert call(f, ROPE, q_heads=0, kv_heads=0) == OK


def test_attention_refusals(L):
    f = L.clove_paged_attention
    for bad, status in [(dict(batch=-1), DIM), (dict(q_heads=-2), DIM), (dict(max_context=-1), DIM), (dict(window=-1), DIM), (dict(q_heads=5), ARG),
                        (dict(q=None), NULL), (dict(out=None), NULL), (dict(block_table=None), NULL), (dict(context_lens=None), NULL),
                        (dict(max_context=129), ARG), (dict(q_stride=255), ARG), (dict(out_stride=255), ARG), (dict(softcap=-1.0), ARG),
                        (dict(softcap=float("nan")), ARG), (dict(weights=W, weights_stride=99), ARG), (dict(out=Q), ALIASING), (dict(out=K), ALIASING),
                        (dict(weights=T, weights_stride=100), ALIASING), (dict(weights=O, weights_stride=100), ALIASING),
                        (dict(block_table=T + 2), ARG), (dict(out=O + 1), ARG)]:
        assert call(f, ATTEND, **{"cache": cache(), **bad}) == status, bad
    assert call(f, ATTEND, cache=cache(), batch=0, q=None) == OK


def test_evict_refusals(L):
    f = L.clove_cache_evict
    for bad, status in [(dict(batch=-1), DIM), (dict(budget=-1), DIM), (dict(sinks=-1), DIM), (dict(recent=-1), DIM), (dict(max_context=-1), DIM),
                        (dict(weights=None), NULL), (dict(positions=None), NULL), (dict(weights_out=None), NULL), (dict(positions_out=None), NULL),
                        (dict(lens_out=None), NULL), (dict(context_lens=None), NULL), (dict(block_table=None), NULL), (dict(max_context=129), ARG),
                        (dict(weights_stride=99), ARG), (dict(positions_out_stride=99), ARG), (dict(weights_out=W, weights_out_stride=101), ALIASING),
                        (dict(weights_out=X), ALIASING), (dict(positions_out=W), ALIASING), (dict(weights_out=W + 400), ALIASING),
                        (dict(lens_out=T), ALIASING), (dict(weights=W + 2), ARG), (dict(weights_out=K), ALIASING)]:
        assert call(f, EVICT, **{"cache": cache(), **bad}) == status, bad
    assert call(f, EVICT, cache=cache(), batch=0, weights=None) == OK
    assert call(f, EVICT, cache=None) == NULL


def test_logits_refusals(L):
    f = L.clove_penalize_logits
    for bad, status in [(dict(batch=-1), DIM), (dict(vocab=-1), DIM), (dict(dtype=3), ARG), (dict(out_dtype=1), ARG), (dict(dtype=2, out_dtype=0), ARG),
                        (dict(logits=None), NULL), (dict(out=None), NULL), (dict(history_lens=None), NULL), (dict(bias_ids=W), NULL),
                        (dict(logits_stride=999), ARG), (dict(out_stride=999), ARG), (dict(allowed=W, allowed_stride=31), ARG), (dict(out=Y + 1), ARG),
                        (dict(out=X, out_stride=1001), ALIASING), (dict(out=X + 2), ALIASING), (dict(out=X, out_dtype=2), ALIASING),
                        (dict(out=T), ALIASING), (dict(history_stride=-1), DIM), (dict(history=T + 2), ARG), (dict(out_dtype=2, out=Y + 2), ARG)]:
        assert call(f, LOGITS, **bad) == status, bad
    assert call(f, LOGITS, batch=0, logits=None) == OK
    assert call(f, LOGITS, vocab=0, out=None) == OK


def _planned(L, f, args, **kw):
    """The status of a call that is only planned: nothing is launched, so that the fake
    addresses are safe where there is a GPU too."""
    assert L.clove_workspace_query_begin() == OK
    try:
        return call(f, args, **kw)
    finally:
        L.clove_workspace_query_end()


TAKEN = (OK, _lib.CLOVE_ERR_NO_DEVICE)  # (planning asks for the device, last)


def test_a_single_row_is_its_own_output_whatever_its_stride(L):
    one = dict(qkv=X, q_out=X, k_out=X + 512)
    for strides in [dict(), dict(q_out_stride=512, k_out_stride=512), dict(q_out_stride=300, k_out_stride=128, qkv_stride=700)]:
        assert _planned(L, L.clove_qk_norm_rope, ROPE, T=1, **one, **strides) in TAKEN, strides
    assert _planned(L, L.clove_qk_norm_rope, ROPE, T=1, q_out=X + 2) == ALIASING
    assert _planned(L, L.clove_qk_norm_rope, ROPE, T=2, **one) == ALIASING
    own = dict(cache=cache(), weights_out=W, positions_out=X, weights_out_stride=100, positions_out_stride=101)
    assert _planned(L, L.clove_cache_evict, EVICT, batch=1, **own) in TAKEN
    assert _planned(L, L.clove_cache_evict, EVICT, batch=2, **own) == ALIASING
    assert _planned(L, L.clove_penalize_logits, LOGITS, batch=1, out=X, out_stride=1001) in TAKEN
    assert _planned(L, L.clove_penalize_logits, LOGITS, batch=1, out=X, out_dtype=2) == ALIASING


def test_a_table_ends_with_its_entries(L):
    """Rows of a table inside wider ones: what follows its ceil(100 / 16) = 7 entries may be an output."""
    wide = dict(cache=cache(), table_stride=200)
    evict = dict(wide, weights_stride=100, positions=X, positions_stride=100)
    for after, status in [(28, TAKEN), (24, (ALIASING,))]:
        assert _planned(L, L.clove_paged_attention, ATTEND, **wide, weights=T + after, weights_stride=200) in status, after
        assert _planned(L, L.clove_cache_evict, EVICT, **evict, weights_out=T + after, weights_out_stride=200) in status, after
    assert _planned(L, L.clove_paged_attention, ATTEND, **wide, out=T + 3 * 800 + 28) in TAKEN  # behind the last row's
    assert _planned(L, L.clove_paged_attention, ATTEND, **wide, out=T + 3 * 800 + 24) == ALIASING
