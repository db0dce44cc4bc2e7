// Operators of a decode step around the GEMMs: query / key norms with rotation
// and the cache write, attention of one new token over the paged cache,
// eviction from that cache, penalties and masks on the logits.  Shared by the
// C ABI layer (capi.hip) and their kernels; not installed.
#pragma once

#include "common.hpp"
#include "dispatch.hpp"

namespace clove {

namespace hw {

// Element types of these operators.  Arithmetic is fp32 in every one of them;
// a result is rounded to the element type once, to nearest even, at its store.
template <int DT>
struct Elem;
template <>
struct Elem<CLOVE_DTYPE_FP16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float load(raw x) { return h2f(x); }
    static __device__ __forceinline__ raw store(float f) { return f2h(f); }
};
template <>
struct Elem<CLOVE_DTYPE_BF16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float load(raw x) { return bitcast<float>((unsigned)x << 16); }
    static __device__ __forceinline__ raw store(float f) { return bitcast<uint16_t>(static_cast<__bf16>(f)); }
};
template <>
struct Elem<CLOVE_DTYPE_FP32> {
    typedef float raw;
    static __device__ __forceinline__ float load(raw x) { return x; }
    static __device__ __forceinline__ raw store(float f) { return f; }
};

// Inclusive prefix sum over the wave: DPP row_shr 1, 2, 4, 8 inside the rows of
// 16, then the last lane of a row added to the rows after it.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast31 into rows 2 and 3
    return v;
}

}  // namespace hw

// n / d for 0 <= n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d), m d - 2^(31+s) < d <= 2^s, so that n times it stays
// below 2^(31+s) and floor(n m / 2^(31+s)) is the quotient.
struct FastDiv {
    unsigned m = 1u << 31;
    int shift = 31, d = 1;
    FastDiv() = default;
    explicit FastDiv(int by) : d(by) {
        int s = 0;
        while (((int64_t)1 << s) < by) ++s;
        shift = 31 + s;
        m = (unsigned)((((uint64_t)1 << shift) + (uint64_t)by - 1) / (uint64_t)by);
    }
    __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(unsigned)n * m) >> shift); }
};

// The paged cache of one layer as kernels take it: element (page, head, row, d)
// of k and v lies at page * page_stride + (head * page_size + row) * head_dim + d.
struct PagedCache {
    uint16_t* k = nullptr;
    uint16_t* v = nullptr;
    int64_t page_stride = 0;
    int num_pages = 0, page_size = 0, kv_heads = 0, head_dim = 0;
    int dtype = 0;
};

struct RopeArgs {
    const uint16_t* qkv = nullptr;  // [T] rows of q_heads | kv_heads | kv_heads heads
    int64_t qkv_stride = 0;
    const uint16_t* q_weight = nullptr;  // [head_dim] or null: no norm
    const uint16_t* k_weight = nullptr;
    float eps = 0.0f;
    const float* cos = nullptr;  // [max_position, rot_dim / 2]
    const float* sin = nullptr;
    int max_position = 0;
    const int32_t* positions = nullptr;
    uint16_t* q_out = nullptr;
    int64_t q_out_stride = 0;
    uint16_t* k_out = nullptr;  // null: not wanted
    int64_t k_out_stride = 0;
    PagedCache cache;  // cache.k null: no cache write
    const int32_t* slots = nullptr;
    int T = 0, q_heads = 0, kv_heads = 0, head_dim = 0, rot_dim = 0;
    bool interleaved = false;
    int dtype = 0;
};
clove_status_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t stream);

struct PagedAttentionArgs {
    const uint16_t* q = nullptr;
    int64_t q_stride = 0;
    PagedCache cache;
    const int32_t* block_table = nullptr;
    int64_t table_stride = 0;
    const int32_t* context_lens = nullptr;
    uint16_t* out = nullptr;
    int64_t out_stride = 0;
    float* weights = nullptr;  // null: not accumulated
    int64_t weights_stride = 0;
    int batch = 0, q_heads = 0, max_context = 0;
    float scale = 0.0f, softcap = 0.0f;
    int window = 0;
};
clove_status_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream);

struct EvictArgs {
    PagedCache cache;
    const int32_t* block_table = nullptr;
    int64_t table_stride = 0;
    const int32_t* context_lens = nullptr;
    const float* weights = nullptr;
    int64_t weights_stride = 0;
    const int32_t* positions = nullptr;
    int64_t positions_stride = 0;
    float* weights_out = nullptr;
    int64_t weights_out_stride = 0;
    int32_t* positions_out = nullptr;
    int64_t positions_out_stride = 0;
    int32_t* lens_out = nullptr;
    int batch = 0, max_context = 0, budget = 0, sinks = 0, recent = 0;
};
clove_status_t launch_cache_evict(const EvictArgs& a, hipStream_t stream);

struct LogitsArgs {
    const void* logits = nullptr;
    int64_t logits_stride = 0;
    int dtype = 0;
    void* out = nullptr;
    int64_t out_stride = 0;
    int out_dtype = 0;
    int batch = 0, vocab = 0;
    const int32_t* history = nullptr;
    int64_t history_stride = 0;
    const int32_t* history_lens = nullptr;
    const int32_t* prompt_lens = nullptr;
    const float* repetition = nullptr;
    const float* presence = nullptr;
    const float* frequency = nullptr;
    const int32_t* bias_ids = nullptr;
    const float* bias_values = nullptr;
    int64_t bias_stride = 0;
    const int32_t* bias_counts = nullptr;
    const uint32_t* allowed = nullptr;
    int64_t allowed_stride = 0;
};
clove_status_t launch_penalize_logits(const LogitsArgs& a, hipStream_t stream);

}  // namespace clove
