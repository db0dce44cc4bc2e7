// Attention of one new token per sequence over the paged cache.
//
//   s_j = scale q.k_j  (softcap: c tanh(s_j / c)),  p = softmax(s),  out = sum_j p_j v_j
//
// in one pass over the keys with a running maximum m and sum l: scores are kept
// in base 2 (t = s log2 e), p_j = 2^(t_j - m) / l.  The bytes are K and V once;
// everything else is small, so long caches are bound by HBM: 65536 keys of one
// sequence, 8 KV heads of 128 (268 MB), 53 us, 5.0 TB/s; 16 x 4096 keys of 32 KV
// heads of 128 (1.07 GB) 188 us, 5.7 TB/s, where a copy reaches 5.1.  Short ones are
// bound by the latencies from the lengths to the page table to the rows, and of the
// join: 411 keys 7.8 us, 20 keys 4.3.
//
// Accumulated weights need every head's final m and l, so the scores go to
// scratch (fp32, one per query head and key) and a second kernel adds
// sum_h 2^(t - m_h) / l_h to each key's weight: 5 of 45 us for 48 sequences of
// up to 6144 keys (145 MB of cache, 9 MB of scores written and read again).
#include <algorithm>

#include "decode.hpp"
#include "paged_plan.hpp"

namespace clove {
namespace paged {

using namespace hw;

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    PagedAttentionArgs a;
    FastDiv page;        // by the page size
    int group;           // query heads per KV head
    int tiles;           // tiles of 16 query heads per KV head (MFMA kernel)
    // With more keys than one workgroup per (sequence, KV head, tile) should take,
    // the kernel cuts each sequence by the lengths it finds (Cut)
    bool cuts;
    int fill;            // workgroups that the CUs hold at once
    int rounds;          // most times as many that there are
    int slots;           // most workgroups with keys: all of them, where it does not cut
    float* partials;     // [slots] slabs of `slab` floats, then as many for joined ones
    unsigned* counters;  // [sequence, KV head, tile], then [slots] of groups of `fan` splits
    int slab, fan;       // (a workgroup joins `fan` at most)
    float* scores;       // [batch, q_heads] rows of score_stride, base 2, -inf where unseen; null: not wanted
    int64_t score_stride;
    float2* stats;       // [batch, q_heads] (m, l)
};

// 2^x by the hardware's instruction: within 1 unit in the last place, results
// below 2^-126 as 0, which no sum here can tell from what they are
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// score in base 2 of the scaled dot product
__device__ __forceinline__ float base2(const PagedAttentionArgs& a, float dot) {
    if (a.softcap > 0.0f) return a.softcap * kLog2e * tanhf(dot * a.scale / a.softcap);
    return dot * (a.scale * kLog2e);
}

__device__ __forceinline__ int context(const PagedAttentionArgs& a, int b) {
    return min(max(a.context_lens[b], 0), a.max_context);
}

// Element offset of key j's row (of KV head `kh`), or -1 where its page is absent.
__device__ __forceinline__ int64_t row_at(const Params& p, int b, int kh, int j) {
    const PagedAttentionArgs& a = p.a;
    const PagedCache& c = a.cache;
    const int page = p.page.div(j), row = j - page * c.page_size;
    const int id = a.block_table[b * a.table_stride + page];
    if ((unsigned)id >= (unsigned)c.num_pages) return -1;
    return (int64_t)id * c.page_stride + ((int64_t)kh * c.page_size + row) * c.head_dim;
}

// m that can be subtracted: 0 where no score is above -infinity
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// Any head_dim up to 64 E and any alignment: a workgroup per (sequence, query
// head), a key per wave, element lane + 64 e per lane.  For head_dim outside 8 .. 256
// only, and slow there: nothing is split over the length, K and V are read once for
// each query head (32768 keys, 16 heads on one KV head of 512, 67 MB: 38 ms).
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
    float* scores = p.scores ? p.scores + ((int64_t)b * a.q_heads + h) * p.score_stride : nullptr;
    for (int j = first + wave; j < n; j += 4) {
        const int64_t at = row_at(p, b, kh, j);
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
        const float old = exp2_(m - sub), w = exp2_(t - sub);
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
        const float f = exp2_(part_m[w] - sub);
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

// weights[b, j] += sum over the heads: 256 keys a workgroup, four adjacent ones a
// lane, each wave an eighth of the heads in their order, four heads' scores in
// flight; the eighths are added in theirs.  (48 sequences of up to 6144 keys, 32
// heads: 45.6 us with the attention, 49 with a key to a thread and four parts; 100
// of up to 2000 keys, 8 heads, 16.9 and 22.9.  Sixteen waves 46.1 to 47.)
constexpr int kAddKeys = 256, kAddWaves = 8;
__global__ void __launch_bounds__(64 * kAddWaves) add_weights(const Params p, int blocks) {
    constexpr int U = 4;
    __shared__ __align__(16) float part[kAddWaves][kAddKeys];
    const PagedAttentionArgs& a = p.a;
    const int b = blockIdx.x / blocks, j0 = (blockIdx.x - b * blocks) * kAddKeys;
    const int wave = threadIdx.x / 64, four = threadIdx.x % 64 * 4, own = cdiv(a.q_heads, kAddWaves), h1 = min(a.q_heads, (wave + 1) * own);
    const int n = context(a, b), first = a.window > 0 ? max(0, n - a.window) : 0;
    if (j0 >= n || j0 + kAddKeys <= first) return;
    const int j = j0 + threadIdx.x;
    float* const w = a.weights + b * a.weights_stride + j;
    const bool seen = threadIdx.x < kAddKeys && j >= first && j < n;
    const float before = seen ? *w : 0.0f;
    // (rows of scores are whole 32s; what lies before the first key or past the last is not used)
    const float* s = p.scores + (int64_t)b * a.q_heads * p.score_stride + min(j0 + four, (int)p.score_stride - 4);
    const float2* st = p.stats + (int64_t)b * a.q_heads;
    f32x4 sum = {};
    for (int h0 = wave * own; h0 < h1; h0 += U) {
        f32x4 t[U];
        float2 ml[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = min(h0 + u, h1 - 1);
            t[u] = *reinterpret_cast<const f32x4*>(s + (int64_t)h * p.score_stride);
            ml[u] = st[h];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h0 + u < h1 && ml[u].y != 0.0f) {
                ml[u].y = 1.0f / ml[u].y;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_(t[u][i] - ml[u].x), ml[u].y, sum[i]);
            }
        }
    }
    *reinterpret_cast<f32x4*>(&part[wave][four]) = sum;
    __syncthreads();
    if (!seen) return;
    float total = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < kAddWaves; ++i) total += part[i][threadIdx.x];
    *w = before + total;
}

template <int DT>
void launch_any(const Params& p, hipStream_t stream) {
    const int D = p.a.cache.head_dim;
    const auto kernel = D <= 64 ? attend_any<DT, 1> : D <= 128 ? attend_any<DT, 2> : D <= 256 ? attend_any<DT, 4> : attend_any<DT, 16>;
    CLOVE_LAUNCH(kernel, dim3((unsigned)(p.a.batch * p.a.q_heads)), dim3(256), 0, stream, p);
}

// ---------------------------------------------------------------------------
// head_dim 8 .. 256: MFMA
//
// A workgroup of four waves takes a chunk of the keys (Cut) of one (sequence, KV
// head, tile of up to 16 query heads), each wave every fourth 32 of them;
// workgroups of one wave or eight (W) take all keys of a short sequence.  With keys as
// rows and query heads as columns of v_mfma_f32_16x16x32,
//   S [16 keys x 16 heads] = K [keys x d] Q^T [d x heads]       (two of them)
//   O^T [d x heads] += V^T [d x 32 keys] P^T [32 keys x heads]
// K's operand is K's row in memory (lane l: key l % 16, 8 elements from 8 (l / 16)
// of each 32), and a lane gets four scores of its head (l % 16) per 16 keys: the
// P^T operand of the second product, if its 8 k-slots of lane group g name the
// keys 4 g .. 4 g + 3 of either 16.  So softmax needs no exchange but the
// maximum over the four lane groups, and only V passes through LDS, private to
// the wave, where ds_read_b64_tr_b16 turns its rows.  P is used as the sum of
// 16-bit numbers, two in fp16 (22 bits, kPScale) and three in bf16 (all 24), so
// that what a result loses is its own rounding alone; the MFMAs of the further
// products hide under the loads.
//
// Registers of K are loaded for the wave's next 32 keys as soon as the first
// product has read them, those of V as soon as they are in LDS: 8 to 16 KB (at
// head_dim 128) are in flight per wave nearly all the time.
//
// Workgroups of one (sequence, KV head, tile) publish (O, m, l) past the L2s and
// the last to arrive joins them, or, where they are much to read for one, the
// last of each group its group's, and the last of those the joined ones.  The
// order of a sum is that of the splits whoever does it.
// ---------------------------------------------------------------------------
template <int DT>
struct Mfma;
template <>
struct Mfma<CLOVE_DTYPE_FP16> {
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
    }
};
template <>
struct Mfma<CLOVE_DTYPE_BF16> {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
    }
};

// over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float groups_max(float x) {
    const auto s = __builtin_amdgcn_permlane16_swap(bitcast<unsigned>(x), bitcast<unsigned>(x), false, false);
    const float y = fmaxf(bitcast<float>(s[0]), bitcast<float>(s[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(bitcast<unsigned>(y), bitcast<unsigned>(y), false, false);
    return fmaxf(bitcast<float>(t[0]), bitcast<float>(t[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
    const float y = swap_sum16(x, x);
    return swap_sum32(y, y);
}

// 16-bit numbers that a softmax weight is the sum of
template <int DT>
constexpr int kParts = DT == CLOVE_DTYPE_BF16 ? 3 : 2;
// What it is multiplied by for them, in both sums, O and l, whose quotient is the
// result.  fp16's steps end at 2^-24: of a weight 2^(t - m) <= 1 as it is, the two
// parts hold fewer than 22 bits from 2^-3 down and nothing below 2^-25, and many keys
// far below one whose value is small are then lost (4096 positive ones 2^-24 below it
// came out 3e-3 off, and more the more they cancel).  Times 2^15 they are whole down
// to 2^-18, and what is lost of any weight is at most 2^-40 of the wave's largest.
template <int DT>
constexpr float kPScale = DT == CLOVE_DTYPE_FP16 ? 32768.0f : 1.0f;

template <int NC>
constexpr int row_bytes() { return NC * 64 + 32; }  // a V row in LDS: 8 banks further each row
template <int NC>
constexpr int wave_lds() { return 32 * row_bytes<NC>(); }
// after the keys the same LDS holds the waves' O [16 heads][32 NC + 4] and (m, l) [16]
template <int NC>
constexpr int o_stride() { return 32 * NC + 4; }
static_assert(16 * o_stride<1>() * 4 + 128 <= wave_lds<1>() && 16 * o_stride<8>() * 4 + 128 <= wave_lds<8>(), "O fits where V was");

// Sixteen bytes of a row from element d: the first D - d elements of it where
// there are fewer than 8 (TAIL: rows at any alignment, head_dim any number).
template <bool TAIL>
__device__ __forceinline__ u32x4 load_row(const uint16_t* row, int d, int D) {
    if constexpr (!TAIL) return *reinterpret_cast<const u32x4*>(row + d);
    const int back = max(d + 8 - D, 0);  // the last 8 elements of the row, moved down
    const u32x4 x = load_any16(reinterpret_cast<const unsigned char*>(row + d - back));
    return back ? shift_bytes(x, 2 * back) : x;
}

typedef short i16x4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4v lds_i16x4v;
__device__ __forceinline__ u32x2 lds_turned(const char* p) {
    return bitcast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4v*)p));
}

template <int DT>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
    return (unsigned)Elem<DT>::store(lo) | ((unsigned)Elem<DT>::store(hi) << 16);
}

// All bits of those of two elements that are infinite or NaN.
template <int DT>
__device__ __forceinline__ unsigned nonfinite2(unsigned x) {
    constexpr unsigned exponent = DT == CLOVE_DTYPE_FP16 ? 0x7c007c00u : 0x7f807f80u, one = DT == CLOVE_DTYPE_FP16 ? 0x04000400u : 0x00800080u;
    return ((((x & exponent) + one) >> 15) & 0x00010001u) * 0xffffu;
}

// Four outputs of one row from element d.
template <int DT>
__device__ __forceinline__ void store4(uint16_t* row, int d, int D, bool vec, const f32x4& x) {
    if (vec && d + 4 <= D) {
        *reinterpret_cast<u32x2*>(row + d) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d + i < D) row[d + i] = Elem<DT>::store(x[i]);
}

// Running (m, l, o) of disjoint keys merged: both maxima may be -infinity.
__device__ __forceinline__ void merge(float& m, float& l, f32x4& o, float m2, float l2, const f32x4& o2) {
    const float top = fmaxf(m, m2), sub = finite_max(top);
    const float f = exp2_(m - sub), f2 = exp2_(m2 - sub);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + o2[i] * f2;
}

// How the kernel shares out the keys: into `chunk`s of so many 32s of keys that
// there are about `fill` of them (with KV heads and tiles), or up to `rounds` times
// that where they would be longer than kLongest, a sequence's chunks of one length.
// Every wave works it out for itself from the lengths, 64 sequences at a time.
// (By the bound of the lengths alone, most workgroups of 48 mixed sequences had no
// keys, and those that had some waited for them to pass: 55 us instead of 49.)
struct Cut {
    int b, split, total;     // this workgroup's sequence, its split and how many it has
    int first;               // workgroup of split 0 among those of all sequences, before KV heads and tiles
    int chunk;               // 32s of keys of each split
};

__device__ __forceinline__ int keys32(const PagedAttentionArgs& a, int n) {
    const int first = a.window > 0 ? max(0, n - a.window) & ~31 : 0;
    return cdiv(n - first, 32);
}

// Sequence and split of workgroup `i` (of those before KV heads and tiles);
// .b < 0 where there are fewer.
static_assert(CLOVE_MAX_CONTEXT / 32 <= 0xffffffff / 64, "a wave's sum of lengths has 32 bits");
__device__ __forceinline__ Cut cut(const Params& p, int i, int per) {
    const PagedAttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63;
    int64_t sum = 0;
    int t0 = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int t = b0 + lane < a.batch ? keys32(a, context(a, b0 + lane)) : 0;
        if (b0 == 0) t0 = t;
        sum += wave_sum((unsigned)t);  // (64 of at most 2^25)
    }
    const int chunk = chunk_of(sum, per, p.fill, p.rounds);
    int before = 0;
    Cut c{-1, 0, 0, 0, 0};
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const bool on = b0 + lane < a.batch;
        const int t = b0 == 0 ? t0 : on ? keys32(a, context(a, b0 + lane)) : 0;
        const int splits = on ? splits_of(t, chunk) : 0, upto = before + wave_scan(splits);
        const unsigned long long in = __ballot(on && i >= upto - splits && i < upto);
        if (in) {
            const int who = __ffsll((long long)in) - 1;
            c.b = b0 + who;
            c.total = __builtin_amdgcn_readlane(splits, who);
            c.first = __builtin_amdgcn_readlane(upto, who) - c.total;
            c.split = i - c.first;
            c.chunk = own_chunk(__builtin_amdgcn_readlane(t, who), c.total);
            return c;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return c;
}

// A slab: O [16 heads][quads] of four, then (m, l) [16].  All slabs are one
// buffer: the slab is part of a lane's offset, as lanes may read different ones.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t slabs_of(const Params& p) {
    return __builtin_amdgcn_make_buffer_rsrc(p.partials, (short)0, p.partials ? 2 * p.slots * p.slab * 4 : 0, 0x00020000);
}
__device__ __forceinline__ void publish(const Params& p, const __amdgpu_buffer_rsrc_t& r, int slab, int h, int quad, int quads, float M, float L,
                                        const f32x4& O) {
    const int at = slab * p.slab * 4;
    __builtin_amdgcn_raw_buffer_store_b128(bitcast<u32x4>(O), r, at + (h * quads + quad) * 16, 0, kCpolSc1);
    if (quad == 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{bitcast<unsigned>(M), bitcast<unsigned>(L)}, r, at + 256 * quads + 8 * h, 0, kCpolSc1);
}

// `count` slabs `step` apart from slab `first`, joined in their order, U at a time in flight
template <int U>
__device__ __forceinline__ void join(const Params& p, const __amdgpu_buffer_rsrc_t& r, int first, int step, int count, int h, int quad, int quads,
                                     float& M, float& L, f32x4& O) {
    M = -__builtin_inff();
    L = 0.0f;
    O = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < count; s0 += U) {
        u32x4 x[U];
        u32x2 ml[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (first + min(s0 + u, count - 1) * step) * p.slab * 4;
            ml[u] = __builtin_amdgcn_raw_buffer_load_b64(r, at + 256 * quads + 8 * h, 0, kCpolSc1);
            x[u] = __builtin_amdgcn_raw_buffer_load_b128(r, at + (h * quads + quad) * 16, 0, kCpolSc1);
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, bitcast<float>(ml[u][0]));
        const float sub = finite_max(top), f = exp2_(M - sub);
        M = top;
        L *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < count) {
                const float g = exp2_(bitcast<float>(ml[u][0]) - sub);
                const f32x4 y = bitcast<f32x4>(x[u]);
                L = fmaf(bitcast<float>(ml[u][1]), g, L);
#pragma unroll
                for (int i = 0; i < 4; ++i) O[i] = fmaf(y[i], g, O[i]);
            }
    }
}

// The same by the whole workgroup, done(head, quad, M, L, O) for each of its
// heads' quads: teams of as many threads as there are quads take runs of the
// slabs, and the first merges theirs in their order.
template <typename F>
__device__ __forceinline__ void join_all(const Params& p, const __amdgpu_buffer_rsrc_t& r, char* lds, int first, int step, int count, int quads, int items, F done) {
    const int teams = max(1, min(64 * kW / items, count / 8)), run = cdiv(count, teams), tid = threadIdx.x;
    if (teams == 1) {
        for (int i = tid; i < items; i += 64 * kW) {
            const int h = i / quads, quad = i - h * quads;
            float M, L;
            f32x4 O;
            count <= 4 ? join<4>(p, r, first, step, count, h, quad, quads, M, L, O)
                       : join<16>(p, r, first, step, count, h, quad, quads, M, L, O);
            done(h, quad, M, L, O);
        }
        return;
    }
    f32x4* const team_o = reinterpret_cast<f32x4*>(lds);
    float2* const team_ml = reinterpret_cast<float2*>(lds + 64 * kW * 16);
    const int team = tid / items, item = tid - team * items, h = item / quads, quad = item - h * quads;
    const int mine = min(run, count - team * run);  // none for a thread past the teams
    float M = -__builtin_inff(), L = 0.0f;
    f32x4 O{0.f, 0.f, 0.f, 0.f};
    if (team < teams && mine > 0) join<16>(p, r, first + team * run * step, step, mine, h, quad, quads, M, L, O);
    team_o[tid] = O;
    team_ml[tid] = float2{M, L};
    __syncthreads();
    if (team == 0) {
        for (int t = 1; t < teams; ++t) {
            const float2 ml = team_ml[t * items + item];
            merge(M, L, O, ml.x, ml.y, team_o[t * items + item]);
        }
        done(h, quad, M, L, O);
    }
}

// Workgroups of four waves that a CU holds at once, by head_dim / 32: what the
// registers leave, which are bounded to it (a workgroup has one wave on each SIMD;
// rows at any alignment hold one fewer at 6)
constexpr int kResident[8] = {5, 4, 3, 2, 2, 2, 1, 1};
template <int NC, bool TAIL, int W>
constexpr int resident() { return W == kW ? kResident[NC - 1] - (TAIL && NC == 6 ? 1 : 0) : 1; }

template <int DT, int NC, bool TAIL, int W>
__global__ void __launch_bounds__(64 * W, (resident<NC, TAIL, W>())) attend(const Params p) {
    extern __shared__ __align__(16) char lds[];
    __shared__ int last;
    const PagedAttentionArgs& a = p.a;
    const PagedCache& cache = a.cache;
    // Workgroups go to the XCDs in turn: KV heads are the fastest index, so that
    // each XCD has its share of every sequence.  Tiles of the same keys lie eight
    // workgroups apart: on one XCD, whose L2 the first of them fills.
    int unit = blockIdx.x, tile = 0;
    if (p.tiles > 1) {
        const int run = unit / (8 * p.tiles), in_run = unit - run * 8 * p.tiles;
        tile = in_run >> 3;
        unit = 8 * run + (in_run & 7);
    }
    const int seq = unit / cache.kv_heads, kh = unit - seq * cache.kv_heads, per = cache.kv_heads * p.tiles;
    Cut c{seq, 0, 1, seq, 0};
    if constexpr (W == kW)
        if (p.cuts) c = cut(p, seq, per);
    const int b = c.b, split = c.split, total = c.total;
    if (b < 0 || b >= a.batch) return;
    const int pair = (b * cache.kv_heads + kh) * p.tiles + tile, slab0 = (c.first * cache.kv_heads + kh) * p.tiles + tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
    const int D = cache.head_dim, G = min(16, p.group - 16 * tile), h0 = kh * p.group + 16 * tile;
    const int n = context(a, b), first = a.window > 0 ? max(0, n - a.window) : 0, base = first & ~31;
    const int begin = base + split * c.chunk * 32, end = W == kW && p.cuts ? min(n, begin + c.chunk * 32) : n;
    const bool vec = !TAIL;

    u32x4 q[NC];
    const uint16_t* qr = a.q + b * a.q_stride + (int64_t)(h0 + min(row, G - 1)) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 32 * c + 8 * g;
        q[c] = row < G && d < D ? load_row<TAIL>(qr, d, D) : u32x4{0u, 0u, 0u, 0u};
    }

    // the pages of this lane's two keys (16 apart) of the wave's 32 from key j
    const int32_t* table = a.block_table + b * a.table_stride;
    // (read by the bound of the lengths and judged by the length, which the first
    // look-up so need not await: a table row has ceil(max_context / page_size) entries)
    auto page_of = [&](int j) { return j < a.max_context ? table[p.page.div(j)] : -1; };
    auto offset_of = [&](int j, int id, bool& ok) {
        ok = j >= first && j < end && (unsigned)id < (unsigned)cache.num_pages;
        const int in_page = j - p.page.div(j) * cache.page_size;
        return ok ? (int64_t)id * cache.page_stride + ((int64_t)kh * cache.page_size + in_page) * D : (int64_t)0;
    };
    u32x4 k[2][NC], v[2][NC];
    int64_t off[2];
    unsigned seen = 0, seen_next = 0;  // bit i: key i of the 32 is there
    int id[2];
    auto look_up = [&](int j) {
        id[0] = page_of(j + row);
        id[1] = page_of(j + 16 + row);
    };
    auto resolve = [&](int j) {
        bool ok0, ok1;
        off[0] = offset_of(j + row, id[0], ok0);
        off[1] = offset_of(j + 16 + row, id[1], ok1);
        seen_next = (unsigned)(__ballot(ok0) & 0xffffu) | ((unsigned)(__ballot(ok1) & 0xffffu) << 16);
    };
    // (an absent key's loads go to the first row of the cache and are dropped;
    // where none of the 32 is there, nothing is loaded)
    auto load = [&](u32x4(&x)[2][NC], const uint16_t* from) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 32 * c + 8 * g;
                x[r][c] = load_row<TAIL>(from + off[r], d < D ? d : 0, D);
            }
    };
    // lanes past the end of the row hold zeros there
    auto clip = [&](u32x4(&x)[2][NC]) {
        if (32 * (NC - 1) + 8 * g >= D) x[0][NC - 1] = x[1][NC - 1] = u32x4{0u, 0u, 0u, 0u};
    };

    float m = -__builtin_inff(), l = 0.0f;
    f32x4 o[2 * NC];
#pragma unroll
    for (int c = 0; c < 2 * NC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    char* const vs = lds + wave * wave_lds<NC>();
    const char* const turned = vs + (4 * g + (row >> 2)) * row_bytes<NC>() + 8 * (row & 3);
    float* score_row = p.scores && row < G ? p.scores + ((int64_t)b * a.q_heads + h0 + row) * p.score_stride : nullptr;

    int j = begin + 32 * wave;
    look_up(j);
    resolve(j);
    if (seen_next) {
        load(k, cache.k);
        load(v, cache.v);
    }
    look_up(j + 32 * W);
    for (; j < end; j += 32 * W) {
        seen = seen_next;
        f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        if (seen) {
            clip(k);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s[0] = Mfma<DT>::mul(k[0][c], q[c], s[0]);
                s[1] = Mfma<DT>::mul(k[1][c], q[c], s[1]);
            }
        }
        resolve(j + 32 * W);
        if (seen_next) load(k, cache.k);
        look_up(j + 64 * W);
        if (seen) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][i] = base2(a, s[r][i]);
            if (seen != 0xffffffffu) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!((seen >> (16 * r + 4 * g + i)) & 1u)) s[r][i] = -__builtin_inff();
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    if (!((seen >> (16 * r + row)) & 1u))
#pragma unroll
                        for (int c = 0; c < NC; ++c) v[r][c] = u32x4{0u, 0u, 0u, 0u};
            }
            clip(v);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    *reinterpret_cast<u32x4*>(vs + (16 * r + row) * row_bytes<NC>() + 64 * c + 16 * g) = v[r][c];
        } else {
            s[0] = s[1] = f32x4{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        }
        if (score_row) {  // rows are long enough for whole 32 keys
            *reinterpret_cast<f32x4*>(score_row + j + 4 * g) = s[0];
            *reinterpret_cast<f32x4*>(score_row + j + 16 + 4 * g) = s[1];
        }
        if (seen_next) load(v, cache.v);
        if (!seen) continue;

        float top = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(s[0][i], s[1][i]));
        top = groups_max(top);
        const float sub = finite_max(top);
        if (__any(top != m)) {
            const float f = exp2_(m - sub);
            l *= f;
#pragma unroll
            for (int c = 0; c < 2 * NC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][i] *= f;
            m = top;
        }
        u32x4 w[kParts<DT>];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                float x = exp2_(s[r][i] - sub) * kPScale<DT>, y = exp2_(s[r][i + 1] - sub) * kPScale<DT>;
                l += x + y;
#pragma unroll
                for (int k = 0; k < kParts<DT>; ++k) {  // each part what the ones before it leave, rounded
                    const unsigned h = pack2<DT>(x, y);
                    w[k][2 * r + i / 2] = h;
                    x -= Elem<DT>::load((uint16_t)(h & 0xffffu));
                    y -= Elem<DT>::load((uint16_t)(h >> 16));
                }
            }
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) {
            const u32x2 x = lds_turned(turned + 32 * c), y = lds_turned(turned + 16 * row_bytes<NC>() + 32 * c);
            const u32x4 vt{x[0], x[1], y[0], y[1]};
#pragma unroll
            for (int k = 0; k < kParts<DT>; ++k) o[c] = Mfma<DT>::mul(vt, w[k], o[c]);
        }
    }
    // An infinite value times a weight is infinite, but not times a weight's parts, some
    // of which are 0 or negative.  So where a sum comes out infinite or NaN, which is
    // seldom, the wave goes over its keys again for such values alone: times 1 for a
    // weight above 0, times the weight where that is 0 or NaN.
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 2 * NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = fmaf(o[c][i], 0.0f, z[i]);
    const float any = (z[0] + z[1]) + (z[2] + z[3]);
    if (__builtin_expect(__any(any != any), 0)) {
        f32x4 special[2 * NC];
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) special[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float sub = finite_max(m);
#pragma unroll 1
        for (j = begin + 32 * wave; j < end; j += 32 * W) {
            look_up(j);
            resolve(j);
            if (!seen_next) continue;
            load(k, cache.k);
            clip(k);
            f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s[0] = Mfma<DT>::mul(k[0][c], q[c], s[0]);
                s[1] = Mfma<DT>::mul(k[1][c], q[c], s[1]);
            }
            u32x4 there;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    float x[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool in = (seen_next >> (16 * r + 4 * g + i + e)) & 1u;
                        x[e] = in ? exp2_(base2(a, s[r][i + e]) - sub) : 0.0f;
                        x[e] = x[e] > 0.0f ? 1.0f : x[e];
                    }
                    there[2 * r + i / 2] = pack2<DT>(x[0], x[1]);
                }
            load(v, cache.v);
            clip(v);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const bool in = (seen_next >> (16 * r + row)) & 1u;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[r][c][i] &= in ? nonfinite2<DT>(v[r][c][i]) : 0u;
                    *reinterpret_cast<u32x4*>(vs + (16 * r + row) * row_bytes<NC>() + 64 * c + 16 * g) = v[r][c];
                }
            }
#pragma unroll
            for (int c = 0; c < 2 * NC; ++c) {
                const u32x2 x = lds_turned(turned + 32 * c), y = lds_turned(turned + 16 * row_bytes<NC>() + 32 * c);
                special[c] = Mfma<DT>::mul(u32x4{x[0], x[1], y[0], y[1]}, there, special[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[c][i] = special[c][i] != 0.0f ? special[c][i] : o[c][i];
    }
    l = groups_sum(l);

    // the waves, merged in their order
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(lds + wave * wave_lds<NC>());
    if (row < G) {
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) *reinterpret_cast<f32x4*>(mine + row * o_stride<NC>() + 16 * c + 4 * g) = o[c];
        if (g == 0) *reinterpret_cast<float2*>(mine + 16 * o_stride<NC>() + 2 * row) = float2{m, l};
    }
    __syncthreads();
    const int quads = cdiv(D, 4), items = G * quads;
    auto finish = [&](int h, int quad, float M, float L, const f32x4& O) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = L == 0.0f ? 0.0f : O[i] / L;
        store4<DT>(a.out + b * a.out_stride + (int64_t)(h0 + h) * D, 4 * quad, D, vec, x);
        if (p.stats && quad == 0) p.stats[(int64_t)b * a.q_heads + h0 + h] = float2{finite_max(M), L * (1.0f / kPScale<DT>)};
    };
    const __amdgpu_buffer_rsrc_t slabs = slabs_of(p);
    for (int i = threadIdx.x; i < items; i += 64 * W) {
        const int h = i / quads, quad = i - h * quads;
        float M = -__builtin_inff(), L = 0.0f;
        f32x4 O{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float* x = reinterpret_cast<const float*>(lds + w * wave_lds<NC>());
            const float2 ml = *reinterpret_cast<const float2*>(x + 16 * o_stride<NC>() + 2 * h);
            merge(M, L, O, ml.x, ml.y, *reinterpret_cast<const f32x4*>(x + h * o_stride<NC>() + 4 * quad));
        }
        if (W != kW || total == 1) finish(h, quad, M, L, O);
        else publish(p, slabs, slab0 + split * per, h, quad, quads, M, L, O);
    }
    if constexpr (W != kW) return;
    if (total == 1) return;
    int from = slab0, step = per, count = total;
    if (total > p.fan) {
        const int group = split / p.fan, members = min(p.fan, total - group * p.fan), lead = slab0 + group * p.fan * per;
        if (!splitk_arrive_is_last(p.counters + a.batch * per + lead, members, &last)) return;
        join_all(p, slabs, lds, lead, per, members, quads, items, [&](int h, int quad, float M, float L, const f32x4& O) {
            publish(p, slabs, p.slots + lead, h, quad, quads, M, L, O);
        });
        from += p.slots;
        step *= p.fan;
        count = cdiv(total, p.fan);
    }
    if (!splitk_arrive_is_last(p.counters + pair, count, &last)) return;
    join_all(p, slabs, lds, from, step, count, quads, items, finish);
}

constexpr int kWide = 8;  // waves of the wide form, for head_dim up to 128 (registers)

typedef void (*Kernel)(const Params);
struct Form {
    Kernel kernel;
    int lds;
};
template <int DT, int NC, bool TAIL, int W>
Form form() { return Form{attend<DT, NC, TAIL, W>, W * wave_lds<NC>()}; }
template <int DT, bool TAIL, int W>
Form pick(int nc) {
    switch (nc) {
        case 1: return form<DT, 1, TAIL, W>();
        case 2: return form<DT, 2, TAIL, W>();
        case 3: return form<DT, 3, TAIL, W>();
        case 4: return form<DT, 4, TAIL, W>();
    }
    if constexpr (W != kWide) {
        switch (nc) {
            case 5: return form<DT, 5, TAIL, W>();
            case 6: return form<DT, 6, TAIL, W>();
            case 7: return form<DT, 7, TAIL, W>();
            case 8: return form<DT, 8, TAIL, W>();
        }
    }
    return Form{nullptr, 0};
}

template <int DT>
clove_status_t launch_mfma(const Params& p, bool whole, int waves, hipStream_t stream) {
    const int nc = cdiv(p.a.cache.head_dim, 32);
    const Form f = waves == kWide ? pick<DT, false, kWide>(nc)
                   : waves == 1   ? (whole ? pick<DT, false, 1>(nc) : pick<DT, true, 1>(nc))
                                  : (whole ? pick<DT, false, kW>(nc) : pick<DT, true, kW>(nc));
    const int units = p.slots / p.tiles, grid = p.tiles > 1 ? cdiv(units, 8) * 8 * p.tiles : units;
    const clove_status_t st = ensure_lds(reinterpret_cast<const void*>(f.kernel), f.lds);
    if (st != CLOVE_OK) return st;
    CLOVE_LAUNCH(f.kernel, dim3((unsigned)grid), dim3(64 * waves), (size_t)f.lds, stream, p);
    return CLOVE_OK;
}

}  // namespace paged

clove_status_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    const PagedCache& c = a.cache;
    paged::Params p{};
    p.a = a;
    p.page = FastDiv(c.page_size);
    p.group = a.q_heads / c.kv_heads;
    p.score_stride = (int64_t)hw::cdiv(a.max_context, 32) * 32;
    if (a.weights && a.max_context > 0) {
        const size_t heads = (size_t)a.batch * a.q_heads;
        void* buf = nullptr;
        if ((st = acquire_buffer(stream, kBufDecode, heads * (p.score_stride * sizeof(float) + sizeof(float2)) + 16, &buf)) != CLOVE_OK)
            return st;
        p.scores = static_cast<float*>(buf);
        p.stats = reinterpret_cast<float2*>(p.scores + heads * p.score_stride);
    }
    if (c.head_dim < 8 || c.head_dim > 256) {
        if (c.dtype == CLOVE_DTYPE_FP16) paged::launch_any<CLOVE_DTYPE_FP16>(p, stream);
        else paged::launch_any<CLOVE_DTYPE_BF16>(p, stream);
    } else {
        p.tiles = hw::cdiv(p.group, 16);
        const bool whole = c.head_dim % 8 == 0 && c.page_stride % 8 == 0 && a.q_stride % 8 == 0 && a.out_stride % 4 == 0 &&
                           aligned16(a.q) && aligned16(c.k) && aligned16(c.v) && (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0;
        const int per = c.kv_heads * p.tiles;
        const int64_t pairs = (int64_t)a.batch * per;
        // a window need not start at a whole 32 keys
        const int span = std::max(1, a.window > 0 ? (int)std::min<int64_t>(a.max_context, (int64_t)a.window + 31) : a.max_context);
        // Few sequences: fewer chunks are fewer to join.  One of 65536 keys 58.3 -> 55.8
        // us, of 8192 20.5 -> 17.2.  Up to eight at head_dim 64, two of four workgroups a
        // CU: 4 x 2048, 8192, 32768 keys 12.3, 24.6, 51.0 -> 12.4, 18.9, 46.1, lengths of
        // 32768 down by halves 30.2 -> 26.7; past that mixed sequences want them all (48
        // with weights 45.6 against 49.6, though 48 x 32768 564 -> 543).  Of longer rows
        // one instead of two is for one sequence only: 4 x 32768 keys of 128 103.8 -> 97.6,
        // but the halves 47.9 -> 62.8.  Rows at any alignment, whose loads are slower, want
        // all too (51 against 78).
        const bool fewer = whole && a.batch <= (c.head_dim <= 64 ? 8 : 1);
        p.fill = dev.num_cus * (fewer ? (c.head_dim <= 64 ? 2 : 1) : paged::kResident[hw::cdiv(c.head_dim, 32) - 1]);
        // One wave to a workgroup: nothing to merge where the keys are one wave's anyway
        // and its heads' outputs few (one sequence of 20 keys, head_dim 64, 4.7 -> 4.3
        // us; with 16 heads of 256 13.1 -> 15.4), and where there are more sequences of
        // up to 512 keys than the CUs hold workgroups of four (200 x 8 heads of 64 with
        // 20, 90, 250, 500 keys 9.1, 12.8, 30.4, 49.6 -> 6.2, 10.8, 21.8, 44.0 us; mixed
        // ones of up to 1000 36.9 -> 48.7, one of them outlasting the rest)
        const bool alone = (span <= 32 && std::min(p.group, 16) * c.head_dim <= 512) || (span <= 512 && pairs > p.fill);
        // Eight waves where they take a sequence's keys in one go and four would split
        // it: 200 keys of 1 and 64 sequences, 8 heads of 64, 7.6, 12.9 -> 6.2, 9.7 us;
        // twice as many keys are better split (7.75 against 8.2)
        const bool wide = !alone && whole && c.head_dim <= 128 && span > 32 * paged::kW && span <= 32 * paged::kWide;
        const int waves = alone ? 1 : wide ? paged::kWide : paged::kW;
        p.slab = 16 * hw::cdiv(c.head_dim, 4) * 4 + 32;
        p.slots = (int)pairs;
        const paged::Plan plan = paged::plan(a.batch, per, span, p.fill);
        p.cuts = waves == paged::kW && plan.cuts;
        if (p.cuts) {
            p.rounds = (int)plan.rounds;
            p.slots = (int)plan.slots;
            // what a workgroup reads in about 3 us; another round of arrivals takes as long
            p.fan = std::max(16, std::min(64, (128 << 10) / (std::min(p.group, 16) * c.head_dim * 4)));
            Scratch scratch;
            if ((st = acquire_scratch(stream, (size_t)2 * p.slots * p.slab * 4, (size_t)(pairs + p.slots), &scratch)) != CLOVE_OK) return st;
            p.partials = scratch.partials;
            p.counters = scratch.counters;
        }
        st = c.dtype == CLOVE_DTYPE_FP16 ? paged::launch_mfma<CLOVE_DTYPE_FP16>(p, whole, waves, stream)
                                         : paged::launch_mfma<CLOVE_DTYPE_BF16>(p, whole, waves, stream);
        if (st != CLOVE_OK) return st;
    }
    if ((st = check_launch()) != CLOVE_OK || !p.scores) return st;
    const int blocks = hw::cdiv(a.max_context, paged::kAddKeys);
    CLOVE_LAUNCH(paged::add_weights, dim3((unsigned)(blocks * a.batch)), dim3(64 * paged::kAddWaves), 0, stream, p, blocks);
    return check_launch();
}

}  // namespace clove
