// Attention of one new token per sequence over the paged cache.
//
//   s_j = scale q.k_j  (softcap: c tanh(s_j / c)),  p = softmax(s),  out = sum_j p_j v_j
//
// in one pass over the keys with a running maximum m and sum l: scores are kept
// in base 2 (t = s log2 e), p_j = 2^(t_j - m) / l.  The bytes are K and V once;
// everything else is small, so the kernel is HBM-bound.
//
// Accumulated weights need every head's final m and l, so the scores go to
// scratch (fp32, one per query head and key) and a second kernel adds
// sum_h 2^(t - m_h) / l_h to each key's weight, in the order of the heads.
#include <algorithm>

#include "decode.hpp"

namespace clove {
namespace paged {

using namespace hw;

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    PagedAttentionArgs a;
    int group;      // query heads per KV head
    float* scores;  // [batch, q_heads, max_context] base 2, -inf where unseen; null: not wanted
    float2* stats;  // [batch, q_heads] (m, l)
};

// score in base 2 of the scaled dot product
__device__ __forceinline__ float base2(const PagedAttentionArgs& a, float dot) {
    if (a.softcap > 0.0f) return a.softcap * kLog2e * tanhf(dot * a.scale / a.softcap);
    return dot * (a.scale * kLog2e);
}

__device__ __forceinline__ int context(const PagedAttentionArgs& a, int b) {
    return min(max(a.context_lens[b], 0), a.max_context);
}

// Element offset of key j's row (of KV head `kh`), or -1 where its page is absent.
__device__ __forceinline__ int64_t row_at(const PagedAttentionArgs& a, int b, int kh, int j) {
    const PagedCache& c = a.cache;
    const int page = j / c.page_size, row = j - page * c.page_size;
    const int id = a.block_table[b * a.table_stride + page];
    if ((unsigned)id >= (unsigned)c.num_pages) return -1;
    return (int64_t)id * c.page_stride + ((int64_t)kh * c.page_size + row) * c.head_dim;
}

// m that can be subtracted: 0 where no score is above -infinity
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// Any head_dim up to 64 E and any alignment: a workgroup per (sequence, query
// head), a key per wave, element lane + 64 e per lane.
template <int DT, int E>
__global__ void __launch_bounds__(256) attend_any(const Params p) {
    using T = Elem<DT>;
    const PagedAttentionArgs& a = p.a;
    __shared__ float part_o[4][64 * E], part_m[4], part_l[4];
    const int b = blockIdx.x / a.q_heads, h = blockIdx.x - b * a.q_heads, kh = h / p.group;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.cache.head_dim;
    const int n = context(a, b), first = a.window > 0 ? max(0, n - a.window) : 0;
    float q[E], o[E], m = -__builtin_inff(), l = 0.0f;
    const uint16_t* qr = a.q + b * a.q_stride + (int64_t)h * D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = lane + 64 * e < D ? T::load(qr[lane + 64 * e]) : 0.0f;
        o[e] = 0.0f;
    }
    float* scores = p.scores ? p.scores + ((int64_t)b * a.q_heads + h) * a.max_context : nullptr;
    for (int j = first + wave; j < n; j += 4) {
        const int64_t at = row_at(a, b, kh, j);
        if (at < 0) {
            if (scores && lane == 0) scores[j] = -__builtin_inff();
            continue;
        }
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) dot = fmaf(q[e], T::load(a.cache.k[at + lane + 64 * e]), dot);
        const float t = base2(a, wave_sum(dot));
        if (scores && lane == 0) scores[j] = t;
        const float top = fmaxf(m, t), sub = finite_max(top);
        const float old = exp2f(m - sub), w = exp2f(t - sub);
        m = t != t ? t : top;  // a NaN stays
        l = l * old + w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) o[e] = fmaf(w, T::load(a.cache.v[at + lane + 64 * e]), o[e] * old);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) part_o[wave][lane + 64 * e] = o[e];
    if (lane == 0) {
        part_m[wave] = m;
        part_l[wave] = l;
    }
    __syncthreads();
    if (wave) return;
    float top = part_m[0];
    for (int w = 1; w < 4; ++w) top = fmaxf(top, part_m[w]);
    const float sub = finite_max(top);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int w = 0; w < 4; ++w) {
        const float f = exp2f(part_m[w] - sub);
        sum += part_l[w] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(part_o[w][lane + 64 * e], f, o[e]);
    }
    uint16_t* out = a.out + b * a.out_stride + (int64_t)h * D;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) out[lane + 64 * e] = T::store(sum == 0.0f ? 0.0f : o[e] / sum);
    if (p.stats && lane == 0) p.stats[(int64_t)b * a.q_heads + h] = float2{sub, sum};
}

// weights[b, j] += sum over the heads, in their order
__global__ void __launch_bounds__(256) add_weights(const Params p, int blocks) {
    const PagedAttentionArgs& a = p.a;
    const int b = blockIdx.x / blocks, j = (blockIdx.x - b * blocks) * 256 + threadIdx.x;
    const int n = context(a, b), first = a.window > 0 ? max(0, n - a.window) : 0;
    if (j < first || j >= n) return;
    const float* s = p.scores + (int64_t)b * a.q_heads * a.max_context + j;
    const float2* st = p.stats + (int64_t)b * a.q_heads;
    float sum = 0.0f;
    for (int h = 0; h < a.q_heads; ++h) {
        const float w = exp2f(s[(int64_t)h * a.max_context] - st[h].x) / st[h].y;
        if (st[h].y != 0.0f) sum += w;
    }
    a.weights[b * a.weights_stride + j] += sum;
}

template <int DT>
void launch_any(const Params& p, hipStream_t stream) {
    const int D = p.a.cache.head_dim;
    const auto kernel = D <= 64 ? attend_any<DT, 1> : D <= 128 ? attend_any<DT, 2> : D <= 256 ? attend_any<DT, 4> : attend_any<DT, 16>;
    CLOVE_LAUNCH(kernel, dim3((unsigned)(p.a.batch * p.a.q_heads)), dim3(256), 0, stream, p);
}

}  // namespace paged

clove_status_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
    clove_status_t st;
    paged::Params p{a, a.q_heads / a.cache.kv_heads, nullptr, nullptr};
    if (a.weights && a.max_context > 0) {
        const size_t heads = (size_t)a.batch * a.q_heads;
        void* buf = nullptr;
        if ((st = acquire_buffer(stream, kBufDecode, heads * (a.max_context * sizeof(float) + sizeof(float2)), &buf)) != CLOVE_OK)
            return st;
        p.stats = static_cast<float2*>(buf);
        p.scores = reinterpret_cast<float*>(p.stats + heads);
    }
    if (a.cache.dtype == CLOVE_DTYPE_FP16) paged::launch_any<CLOVE_DTYPE_FP16>(p, stream);
    else paged::launch_any<CLOVE_DTYPE_BF16>(p, stream);
    if ((st = check_launch()) != CLOVE_OK || !p.scores) return st;
    const int blocks = hw::cdiv(a.max_context, 256);
    CLOVE_LAUNCH(paged::add_weights, dim3((unsigned)(blocks * a.batch)), dim3(256), 0, stream, p, blocks);
    return check_launch();
}

}  // namespace clove
