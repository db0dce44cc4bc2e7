// Products of (token, place) pairs with the INT4 weights of the experts chosen
// for them:
//
//   SwiGLU:  H[p, i] = fp16(silu(X[t] . W[e, i]) * (X[t] . W[e, I + i]))
//   down:    Y[t, o] = alpha sum_j w[t, j] (H[p] . W[e, o]) + beta Y[t, o]
//   W[e, r, k] = (q - z[e, r, k / 128]) s[e, r, k / 128]
//
// q - z is exact in fp16, so a group's sum on MFMA is an fp32 sum of exact
// products, folded into the fp32 accumulator with its scale; SwiGLU and the
// weighted sum over a token's places are fp32, and a result is rounded once.
//
// What bounds it is the weights of the experts hit for few tokens, the matrix
// instructions for many.  Three ways, by shape (choose() in moe_plan.hpp):
//  * few pairs: moe_few_down (a token's places added up by one workgroup) and
//    moe_few (an expert's pairs meet its weights, straight from memory);
//  * moe_tile multiplies tiles of weight rows by tiles of one expert's pairs, which
//    moe_sort has listed by expert (up to 2048 pairs each workgroup finds its own);
//  * moe_any, the same for any K and alignment.
// Down without moe_few_down: the places of a token are added up from fp32 partial
// results in place order (moe_combine), so that a call gives the same bits every time.
// Where tiles leave CUs idle they split K, and the parts are added up in order, by
// moe_combine or, before SwiGLU, moe_swiglu.
#include <type_traits>

#include "i4w_bits.hpp"
#include "moe.hpp"
#include "moe_plan.hpp"

namespace clove {
namespace moe {

using namespace hw;

struct Params {
    MoeArgs a;
    int* off;      // [experts + 1] or null: where an expert's pairs begin in `order`
    int* order;    // [T top_k]: pairs, those of one expert after those of the one before
    float* part;   // down: [splits][T top_k, ldp] products with the outputs o0 .. o0 + on - 1
    int o0, on, ldp;
    FastDiv k;     // by top_k
    FastDiv x;     // a pair's row of X: by top_k, or 1
    int splits, split_groups;  // moe_tile: parts of K, groups of a part
    int rows_t;    // tiles of weight rows
    int P, G;
    int64_t x_bytes;  // of X
    bool by_expert;   // moe_few
    int ng;           // moe_few*: groups of a unit
};

// Workgroup e lists the pairs of expert e; where they begin is the number of pairs of
// lower experts, which it counts itself: no workgroup waits for another.  A thread
// lists its own pairs behind those of the threads before it, so the ids are read
// twice and nothing waits but for the one scan of the counts between.  65536 ids of
// 128 experts: 11 us, of 8 experts and 4096 ids 4.8, latencies of the two passes.  (Every
// workgroup reads all ids, from the L2 after the first: 262 KB each, 34 MB together.)
constexpr int kSortThreads = 1024;
__global__ void __launch_bounds__(kSortThreads) moe_sort(const int32_t* ids, int P, int E, int* off, int* order) {
    __shared__ int lds[2][kSortThreads / 64];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, step = 4 * blockDim.x;
    int less = 0, mine = 0;
    const int whole = P & ~3;
    auto load = [&](int p) { return *reinterpret_cast<const u32x4u*>(ids + p); };
#pragma unroll 4
    for (int p = 4 * tid; p < whole; p += step) {
        const u32x4 v = load(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            less += v[i] < (unsigned)e;
            mine += v[i] == (unsigned)e;
        }
    }
    const bool tail = tid < P - whole;  // of the last, partial four ids one a thread
    const unsigned last = tail ? (unsigned)ids[whole + tid] : ~0u;
    less += last < (unsigned)e;
    mine += last == (unsigned)e;
    const int upto = wave_scan(mine);
    less = wave_sum(less);
    if (lane == 63) lds[0][wave] = upto;
    if (lane == 0) lds[1][wave] = less;
    __syncthreads();
    int begin = 0, count = 0, at = upto - mine;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
        begin += lds[1][w];
        if (w < wave) at += lds[0][w];
        count += lds[0][w];
    }
    if (tid == 0) {
        off[e] = begin;
        if (e == E - 1) off[E] = begin + count;
    }
    if (mine == 0) return;
    at += begin;
#pragma unroll 4
    for (int p = 4 * tid; p < whole; p += step) {
        const u32x4 v = load(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (v[i] == (unsigned)e) order[at++] = p + i;
    }
    if (last == (unsigned)e) order[at] = whole + tid;
}

// Tile `tile` of BC pairs.  Expert e's tiles are numbered off[e] / BC + e and on:
// there are at most off[e + 1] / BC + 1 - off[e] / BC of them, so no two experts'
// meet and the last number is below P / BC + experts.  False: a number that no
// tile has.
struct Tile {
    int e, first, count;  // its pairs: order[first ..), at most BC of them
};
__device__ __forceinline__ bool find_tile(const int* off, int E, int tile, int BC, int lane, Tile* t) {
    int n = 0;
    for (int e = lane; e - lane < E; e += 64) n += __popcll(__ballot(e < E && off[min(e, E)] / BC + e <= tile));
    t->e = n - 1;
    const int begin = off[t->e], end = off[t->e + 1];
    t->first = begin + (tile - (begin / BC + t->e)) * BC;
    t->count = min(BC, end - t->first);
    return t->count > 0;
}

// Any K and alignment.  64 weight rows (SwiGLU: 32 gate and the 32 up rows of the
// same outputs) by 32 pairs, four waves of 16 rows; a 128-k group at a time comes
// through registers to LDS, the weights unpacked on the way.  No stage is loaded ahead
// and its unpacking is scalar: 100 tokens on 6 of 64 experts of 2 x 1408 rows of 2046 123 us
// (of 2048, with moe_tile, 57), 1 on 8 of 128 of 2 x 768 rows of 2046 37 (moe_few 6.8), 2048
// on 2 of 8 of 2 x 11008 rows of 4094 2590 (747).
constexpr int ALD = 136;

template <bool SWIGLU>
__global__ void __launch_bounds__(256) moe_any(const Params p) {
    __shared__ __attribute__((aligned(16))) uint16_t ws[AR][ALD];
    __shared__ __attribute__((aligned(16))) uint16_t xs[AC][ALD];
    __shared__ int pair[AC];
    const MoeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, h = lane >> 4;
    const int tr = blockIdx.x % p.rows_t;
    Tile t;
    if (!find_tile(p.off, a.experts, blockIdx.x / p.rows_t, AC, lane, &t)) return;
    if (tid < AC) pair[tid] = p.order[t.first + min(tid, t.count - 1)];
    __syncthreads();
    constexpr int OR = SWIGLU ? AR / 2 : AR;  // outputs of a tile
    const int r0 = p.o0 + tr * OR, O = a.O, K = a.K, G = p.G;
    const int64_t R = SWIGLU ? 2 * (int64_t)O : O;
    // weight row of tile row i (past the end: the last one, whose results go nowhere)
    auto row = [&](int i) { return (SWIGLU && i >= OR ? (int64_t)O : 0) + min(r0 + i % OR, O - 1) + t.e * R; };
    f32x4 acc[2] = {};
    for (int g = 0; g < G; ++g) {
        {
            // weights: 64 rows x 4 pieces of 16 bytes
            const int i = tid >> 2, c = tid & 3;
            const int64_t r = row(i);
            const uint8_t* src = a.W + r * (K / 2) + 64 * g + 16 * c;
            const int n = K / 2 - (64 * g + 16 * c);
            u32x4 w = {0u, 0u, 0u, 0u};
            if (n >= 16) w = load_any16(src);
            else
                for (int b = 0; b < n; ++b) w[b >> 2] |= (unsigned)src[b] << (8 * (b & 3));
            const float z = rintf(h2f(a.zero[r * G + g]));
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                unsigned o[4];
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    o[b] = pack2h((float)((w[d] >> (8 * b + 4)) & 15u) - z, (float)((w[d] >> (8 * b)) & 15u) - z);
                *reinterpret_cast<u32x4*>(&ws[i][32 * c + 8 * d]) = u32x4{o[0], o[1], o[2], o[3]};
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // rows of X: 32 x 16 pieces of 8
            const int i = (tid >> 4) + 16 * j, c = tid & 15;
            const int q = pair[i];
            const uint16_t* src = a.X + (int64_t)(SWIGLU ? p.k.div(q) : q) * K + 128 * g + 8 * c;
            const int n = K - (128 * g + 8 * c);
            u32x4 x = {0u, 0u, 0u, 0u};
            if (n >= 8) x = load_any16(reinterpret_cast<const unsigned char*>(src));
            else
                for (int b = 0; b < n; ++b) x[b >> 1] |= (unsigned)src[b] << (16 * (b & 1));
            *reinterpret_cast<u32x4*>(&xs[i][8 * c]) = x;
        }
        __syncthreads();
        f32x4 P[2] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f16x8 wf = bitcast<f16x8>(*reinterpret_cast<const u32x4*>(&ws[16 * wave + l16][32 * s + 8 * h]));
#pragma unroll
            for (int j = 0; j < 2; ++j)
                P[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    bitcast<f16x8>(*reinterpret_cast<const u32x4*>(&xs[16 * j + l16][32 * s + 8 * h])), wf, P[j], 0, 0, 0);
        }
        const float sc = h2f(a.scale[row(16 * wave + l16) * G + g]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[j][v] = fmaf(sc, P[j][v], acc[j][v]);
        __syncthreads();
    }
    // a lane holds weight row l16 of its wave and pairs 4 h .. 4 h + 3 of each 16
    if constexpr (SWIGLU) {
        float* up = reinterpret_cast<float*>(ws);  // [32 outputs][32 pairs], one more apart
        if (wave >= 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) up[(16 * (wave - 2) + l16) * 33 + 16 * j + 4 * h + v] = acc[j][v];
        }
        __syncthreads();
        if (wave >= 2) return;
        const int o = r0 + 16 * wave + l16;
        if (o >= O) return;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = 16 * j + 4 * h + v;
                if (c >= t.count) continue;
                const float x = acc[j][v];
                a.Y[(int64_t)pair[c] * O + o] = f2h(x / (1.0f + expf(-x)) * up[(16 * wave + l16) * 33 + c]);
            }
    } else {
        const int o = r0 + 16 * wave + l16;
        if (o >= p.o0 + p.on) return;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = 16 * j + 4 * h + v;
                if (c < t.count) p.part[(int64_t)pair[c] * p.ldp + o - p.o0] = acc[j][v];
            }
    }
}

// ---------------------------------------------------------------------------
// Few pairs (K % 32 == 0, 16-byte aligned X and W): the weights are the time.  A wave
// takes 16 WF weight rows and up to NG = 4 groups of K at once, all their loads in
// flight together and straight to registers (16 bytes a lane: lane group h of 16
// holds k = 32 h .. 32 h + 31 of a row's group); the rows of X it meets and the
// groups' constants go through a part of LDS that is the wave's own, so no wave
// waits for another before the sums meet at the end.  One token on 8 of 128 experts,
// with weights from HBM: 2 x 768 rows of 2048 (13.4 MB) 6.8 us, 2048 rows of 768 back
// (6.7 MB) 5.9, of which a launch takes 4; 20 tokens on 6 of 64 experts of 2 x 1408 rows
// of 2048 (55 experts hit, 169 MB) 40 us, 4.2 TB/s.  On
// v_mfma_f32_16x16x32_f16 with X as the "A" operand: a lane holds weight row
// l % 16 and X rows 4 h .. 4 h + 3; step q of a group takes dword q of every lane,
// k = 32 h + 8 q .. + 7 of lane group h.
// ---------------------------------------------------------------------------
constexpr int XLD = 128 * NG + 8;     // halves of a row of X in LDS

template <int WF, int TB>
struct Unit {
    u32x4 x[TB], w[WF][NG];
    uint16_t s[WF], z[WF];  // entry lane + 64 i: row (lane + 64 i) / NG, group (lane + 64 i) % NG
};
template <int WF, int TB>
struct UnitLds {
    uint16_t x[TB][XLD];
    unsigned c[16 * WF][NG];  // scale, zero point
    static constexpr int BYTES = TB * XLD * 2 + 16 * WF * NG * 4;
};

// Groups g0 .. g0 + ng - 1 of rows row(i) (i < 16 WF, rows of all experts' weights) and
// of n rows of X that begin at element xrow(i).  Everything unconditional, from
// clamped addresses.
template <int WF, int TB, class Row, class XRow>
__device__ __forceinline__ void load_unit(Unit<WF, TB>& u, const MoeArgs& a, int G, int g0, int ng, int n, int lane, Row row,
                                          XRow xrow) {
    const int K = a.K, l16 = lane & 15, h = lane >> 4;
#pragma unroll
    for (int i = 0; i < WF; ++i) {
        const int r = (lane + 64 * i) / NG, g = min(g0 + min(lane % NG, ng - 1), G - 1);
        const int64_t at = row(r) * G + g;
        u.s[i] = a.scale[at];
        u.z[i] = a.zero[at];
    }
#pragma unroll
    for (int f = 0; f < WF; ++f) {
        const uint8_t* w = a.W + row(16 * f + l16) * (K / 2);
#pragma unroll
        for (int j = 0; j < NG; ++j)
            if (j < ng)
                u.w[f][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w + min(64 * (g0 + j) + 16 * h, K / 2 - 16)));
    }
    __builtin_amdgcn_sched_barrier(0);  // (the weights, which come from farthest away, first)
#pragma unroll
    for (int i = 0; i < TB; ++i)
        if (i < n) u.x[i] = *reinterpret_cast<const u32x4*>(a.X + xrow(i) + min(128 * g0 + 8 * lane, K - 8));
    __builtin_amdgcn_sched_barrier(0);
}

// The constants and X to the wave's part of LDS: past K, and past the unit's groups, 0.
template <int WF, int TB>
__device__ __forceinline__ void stage_unit(const Unit<WF, TB>& u, UnitLds<WF, TB>& l, int K, int g0, int ng, int n, int lane) {
#pragma unroll
    for (int i = 0; i < WF; ++i) {
        const int e = lane + 64 * i;
        l.c[e / NG][e % NG] = e % NG < ng ? (unsigned)u.s[i] | ((unsigned)u.z[i] << 16) : 0u;
    }
    const bool in = 8 * lane < 128 * ng && 128 * g0 + 8 * lane < K;
#pragma unroll
    for (int i = 0; i < TB; ++i)
        if (i < n) *reinterpret_cast<u32x4*>(&l.x[i][8 * lane]) = in ? u.x[i] : u32x4{0u, 0u, 0u, 0u};
    asm volatile("" ::: "memory");  // (one wave's LDS accesses take effect in order)
}

// acc += factor * the unit's products
template <int WF, int TB>
__device__ __forceinline__ void add_unit(const Unit<WF, TB>& u, const UnitLds<WF, TB>& l, int ng, int n, int lane, float factor,
                                         f32x4 (&acc)[WF]) {
    const int l16 = lane & 15, h = lane >> 4;
    const uint16_t* x = l.x[min(l16, n - 1)] + 32 * h;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
        if (j >= ng) break;
        f16x8 xf[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) xf[q] = bitcast<f16x8>(*reinterpret_cast<const u32x4*>(x + 128 * j + 8 * q));
#pragma unroll
        for (int f = 0; f < WF; ++f) {
            const unsigned c = l.c[16 * f + l16][j];
            const _Float16 nz = (_Float16)(-rintf(h2f((uint16_t)(c >> 16))) * (1.0f / 512.0f));
            const f16x2 zz = {nz, nz};
            f32x4 P = {};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                P = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[q], i4w::unpack8(u.w[f][j][q], zz), P, 0, 0, 0);
            const float sc = h2f((uint16_t)c) * 512.0f * factor;
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[f][v] = fmaf(sc, P[v], acc[f][v]);
        }
    }
}

// A workgroup takes the pairs of one expert, TB at a time, and 32 weight rows (SwiGLU:
// 16 gate rows and the up rows of the same outputs); its waves share K.  The expert is
// `slot` (p.by_expert), or that of pair `slot`, whose other pairs' workgroups end.
template <bool SWIGLU, int TB, bool PF>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3, 3))) moe_few(const Params p) {
    constexpr int WF = 2, OR = SWIGLU ? 16 : 32;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const MoeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), KS = blockDim.x >> 6;
    const int l16 = lane & 15, h = lane >> 4;
    const int slot = blockIdx.x / p.rows_t, r0 = p.o0 + (blockIdx.x - slot * p.rows_t) * OR, O = a.O, K = a.K, G = p.G;
    int id = a.ids[min(lane, p.P - 1)];  // (beside the slot's own id, not behind it)
    const int e = p.by_expert ? slot : __builtin_amdgcn_readfirstlane(a.ids[slot]);
    if ((unsigned)e >= (unsigned)a.experts) return;
    // [KS] units, then each wave's list of pairs, then the sums of the waves
    UnitLds<WF, TB>& l = reinterpret_cast<UnitLds<WF, TB>*>(smem)[wave];
    int* list = reinterpret_cast<int*>(smem + KS * UnitLds<WF, TB>::BYTES) + wave * p.P;
    float* red = reinterpret_cast<float*>(smem + KS * UnitLds<WF, TB>::BYTES + (KS * p.P * 4 + 15) / 16 * 16);
    int count = 0;
    for (int q0 = 0; q0 < p.P; q0 += 64) {
        const bool is = q0 + lane < p.P && id == e;
        const uint64_t m = __ballot(is);
        if (q0 + 64 < p.P) id = a.ids[min(q0 + 64 + lane, p.P - 1)];
        if (m && count == 0 && !p.by_expert && q0 + __builtin_ctzll(m) != slot) return;
        if (is) list[count + __popcll(m & (((uint64_t)1 << lane) - 1))] = q0 + lane;
        count += __popcll(m);
    }
    asm volatile("" ::: "memory");
    const int64_t base = (int64_t)e * (SWIGLU ? 2 : 1) * O;
    auto row = [&](int i) { return base + (SWIGLU && i >= 16 ? O : 0) + min(r0 + (SWIGLU ? i & 15 : i), O - 1); };
    for (int b0 = 0; b0 < count; b0 += TB) {
        const int n = min(TB, count - b0);
        auto xrow = [&](int i) {
            const int q = __builtin_amdgcn_readfirstlane(list[b0 + min(i, n - 1)]);
            return (int64_t)(SWIGLU ? p.k.div(q) : q) * K;
        };
        f32x4 acc[WF] = {};
        const int ng = p.ng;
        int g0 = wave * ng;
        Unit<WF, TB> u;
        if (g0 < G) load_unit(u, a, G, g0, min(ng, G - g0), n, lane, row, xrow);
        while (g0 < G) {
            const int m = min(ng, G - g0);
            stage_unit(u, l, K, g0, m, n, lane);
            const int g1 = g0 + KS * ng;
            if constexpr (PF) {
                Unit<WF, TB> next;
                if (g1 < G) load_unit(next, a, G, g1, min(ng, G - g1), n, lane, row, xrow);
                add_unit(u, l, m, n, lane, 1.0f, acc);
                u = next;
            } else {
                add_unit(u, l, m, n, lane, 1.0f, acc);
                if (g1 < G) load_unit(u, a, G, g1, min(ng, G - g1), n, lane, row, xrow);
            }
            g0 = g1;
        }
        __syncthreads();  // (the sums of the pairs before have been read)
#pragma unroll
        for (int f = 0; f < WF; ++f)
#pragma unroll
            for (int v = 0; v < 4; ++v) red[((wave * WF + f) * 4 + v) * 64 + lane] = acc[f][v];
        __syncthreads();
        // thread: weight row l16, X row 4 h + v with v = its wave (modulo the waves there are)
        for (int v = wave; v < 4; v += KS) {
            const int c = 4 * h + v;
            float sum[WF];
#pragma unroll
            for (int f = 0; f < WF; ++f) {
                sum[f] = red[(f * 4 + v) * 64 + lane];
                for (int w = 1; w < KS; ++w) sum[f] += red[((w * WF + f) * 4 + v) * 64 + lane];
            }
            if (c >= n) continue;
            const int64_t q = list[b0 + c];
            if constexpr (SWIGLU) {
                const float x = sum[0];
                if (r0 + l16 < O) a.Y[q * O + r0 + l16] = f2h(x / (1.0f + expf(-x)) * sum[1]);
            } else {
#pragma unroll
                for (int f = 0; f < WF; ++f)
                    if (r0 + 16 * f + l16 < p.o0 + p.on) p.part[q * p.ldp + r0 - p.o0 + 16 * f + l16] = sum[f];
            }
        }
    }
}

// Down for few tokens: a workgroup takes one token and 16 WF outputs, its waves the
// (place, K part) units in turn, each weighted as it is added; no partial results in
// memory and one launch.
template <int WF>
__global__ void __launch_bounds__(1024) moe_few_down(const Params p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const MoeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), KS = blockDim.x >> 6;
    const int l16 = lane & 15;
    const int t = blockIdx.x / p.rows_t, r0 = (blockIdx.x - t * p.rows_t) * 16 * WF, O = a.O, K = a.K, G = p.G;
    UnitLds<WF, 1>& l = reinterpret_cast<UnitLds<WF, 1>*>(smem)[wave];
    float* red = reinterpret_cast<float*>(smem + KS * UnitLds<WF, 1>::BYTES);
    const int ng = p.ng, parts = cdiv(G, ng), units = a.top_k * parts;
    f32x4 acc[WF] = {};
    // unit i: place i / parts, groups from ng (i % parts); those without an expert are passed over
    auto at = [&](int i, int64_t* q, int* e, int* g0) {
        for (; i < units; i += KS) {
            const int j = i / parts;
            *q = (int64_t)t * a.top_k + j;
            *e = __builtin_amdgcn_readfirstlane(a.ids[*q]);
            *g0 = (i - j * parts) * ng;
            if ((unsigned)*e < (unsigned)a.experts) break;
        }
        return i;
    };
    int64_t q = 0, q1 = 0;
    int e = 0, g0 = 0, e1 = 0, g1 = 0;
    auto load = [&](Unit<WF, 1>& u, int64_t pair, int expert, int g) {
        load_unit(u, a, G, g, min(ng, G - g), 1, lane, [&](int i) { return (int64_t)expert * O + min(r0 + i, O - 1); },
                  [&](int) { return pair * K; });
    };
    Unit<WF, 1> u;
    int i = at(wave, &q, &e, &g0);
    if (i < units) load(u, q, e, g0);
    while (i < units) {
        const int m = min(ng, G - g0);
        const float weight = a.weights ? a.weights[q] : 1.0f;
        stage_unit(u, l, K, g0, m, 1, lane);
        Unit<WF, 1> next;
        const int i1 = at(i + KS, &q1, &e1, &g1);
        if (i1 < units) load(next, q1, e1, g1);
        add_unit(u, l, m, 1, lane, weight, acc);
        u = next;
        i = i1, q = q1, e = e1, g0 = g1;
    }
    // X row 0: entry 0 of lanes 0 .. 15
    if (lane < 16) {
#pragma unroll
        for (int f = 0; f < WF; ++f) red[(wave * WF + f) * 16 + lane] = acc[f][0];
    }
    __syncthreads();
    if (tid >= 16 * WF || r0 + tid >= O) return;
    float sum = red[tid];
    for (int w = 1; w < KS; ++w) sum += red[w * 16 * WF + tid];
    uint16_t* y = a.Y + (int64_t)t * O + r0 + tid;
    sum *= a.alpha;
    if (a.beta != 0.0f) sum = fmaf(a.beta, h2f(*y), sum);
    *y = f2h(sum);
}

// ---------------------------------------------------------------------------
// K % 32 == 0, 16-byte aligned X and W: tiles of BR weight rows by BC pairs of one
// expert, everything a stage needs (a 128-k group or half of one) by LDS DMA, in the
// layout of i4w_gemm.hpp: X rows and weight rows in 16-byte chunks swizzled by the
// row, then the aligned dwords that hold each row's scale and zero point.  The rows
// of X are those of the tile's pairs, gathered by the DMA's per-lane offsets.
//
// A wave owns 32 FW weight rows by 32 FX pairs on v_mfma_f32_32x32x16_f16 with X
// as the "A" operand: a lane holds one weight row of each block and 16 pairs.
// SwiGLU: of every 32 rows 16 are gate rows and 16 the up rows of the same
// outputs, which meet through v_permlane16_swap.
//
// The accumulators are kept in units of the current group's scale: at a group's
// start they are multiplied by (last scale / this scale), and the group's MFMAs add
// to them.  That is as many VALU operations as folding group sums into a second
// set of accumulators, and half the registers: a wave holds 64 x 128 outputs with
// two waves on a SIMD, so that an unpacked weight meets four blocks of pairs.  A
// group whose scale is 0 leaves the unit as it is and its weights are made 0 (or
// NaN, where the zero point is infinite or NaN, as in the other kernels).
//
// 4096 pairs on 8 experts of 2 x 11008 rows of 4096 take 744 to 800 us by the card, 0.92
// to 0.99 PFLOP/s (a library product of fp16 weights reaches 1.20): matrix pipe and VALU,
// mostly unpacking, are busy for 55 % of the cycles each and do not fill each other's
// gaps.  What a tile costs beside its groups of K is its beginning (three dependent
// latencies: the experts' offsets, its pairs, its first stage) and its end (stores that
// nothing else of the workgroup runs beside), together some ten groups' time.  65536
// pairs on 128 experts of 2048 rows of 768: 282 us, 537 MB of fp32 products and six
// groups of K.  540 pairs on 64 experts of 2 x 1408 rows of 2048 (197 MB): 58 us, 3.4
// TB/s, sixteen groups, and nine pairs to a tile of 32.
// ---------------------------------------------------------------------------
template <int WR_, int WC_, int FW_, int FX_, int S_, int KS_>
struct Cfg {
    static constexpr int WR = WR_, WC = WC_, FW = FW_, FX = FX_, S = S_, KS = KS_;  // KS: 16-k steps a stage
    static constexpr int NW = WR * WC, NT = 64 * NW, BR = 32 * FW * WR, BC = 32 * FX * WC, SPG = 8 / KS;
    static constexpr int XRB = 32 * KS, WRB = 8 * KS;  // bytes of an X row and a weight row
    static constexpr int X_BYTES = BC * XRB, W_BYTES = BR * WRB, SC_BYTES = BR * 4;
    static constexpr int OFF_W = X_BYTES, OFF_SC = OFF_W + W_BYTES, OFF_ZR = OFF_SC + SC_BYTES, STAGE = OFF_ZR + SC_BYTES;
    static constexpr int DX = X_BYTES / (1024 * NW), DW = W_BYTES / (1024 * NW), DS = 2 * BR / (64 * NW);
    // elements of a row of one wave's 32 turned pairs (outputs: fp16 with SwiGLU, else fp32)
    static constexpr int turned_row(bool swiglu) { return swiglu ? 16 * FW + 8 : 32 * FW + 4; }
    static constexpr int OFF_P = S * STAGE, LDS = OFF_P + 4 * BC;  // then the tile's pairs
    // DMA instructions of stage t of a wave (scales and zero points with a group's first)
    static constexpr int dmas(int t) { return DX + DW + (t % SPG == 0 ? DS : 0); }
    static_assert((KS == 8 || KS == 4) && WC == 1, "k-steps, waves");
    static_assert(X_BYTES % (1024 * NW) == 0 && W_BYTES % (1024 * NW) == 0 && (2 * BR) % (64 * NW) == 0, "DMA split");
    static_assert(S >= 2 && S <= 4 && LDS <= 160 * 1024 && BC <= NT && OFF_P >= (CLOVE_MAX_EXPERTS + 8) * 4 && NW * 32 * (32 * FW + 4) * 4 <= OFF_P, "stages");
};

template <class CF, bool SWIGLU>
__global__ void __launch_bounds__(CF::NT) moe_tile(const Params p) {
    using namespace i4w;
    constexpr int FW = CF::FW, FX = CF::FX, S = CF::S, BR = CF::BR, BC = CF::BC, KS = CF::KS, SPG = CF::SPG;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const MoeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % CF::WR, wc = wave / CF::WR;

    // ---- the tile: workgroups are dealt to the 8 XCDs in turn, and each XCD takes a
    // contiguous run of the tiles there are, the pair tiles of one row tile after each
    // other (they share its weights in the XCD's L2) ----
    const int E = a.experts;
    constexpr int CHUNKS = CLOVE_MAX_EXPERTS / 64;
    int* const pairs = reinterpret_cast<int*>(smem + CF::OFF_P);
    // (no lists: the workgroup counts the pairs of every expert itself, each thread holds
    // its ids until the tile is known; where a DMA has not written yet)
    int* const counts = reinterpret_cast<int*>(smem);
    u32x4 id[SCAN / 4];
    int begin[CHUNKS], n[CHUNKS], tiles = 0;  // lane l: of expert 64 i + l (all loads in flight together)
    if (p.off) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            if (64 * i >= E) break;
            const int x = min(64 * i + lane, E - 1);
            begin[i] = p.off[x];
            n[i] = 64 * i + lane < E ? p.off[x + 1] - begin[i] : 0;
        }
    } else {
#pragma unroll
        for (int i = 0; i < SCAN / 4; ++i) {
            const int q = 4 * (i * CF::NT + tid);
            id[i] = u32x4{~0u, ~0u, ~0u, ~0u};
            if (q + 4 <= p.P) id[i] = *reinterpret_cast<const u32x4u*>(a.ids + q);
            else
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (q + v < p.P) id[i][v] = (unsigned)a.ids[q + v];
        }
        for (int e = tid; e < E; e += CF::NT) counts[e] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SCAN / 4; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (id[i][v] < (unsigned)E) atomicAdd(&counts[id[i][v]], 1);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            if (64 * i >= E) break;
            begin[i] = 0;
            n[i] = 64 * i + lane < E ? counts[64 * i + lane] : 0;
        }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
        if (64 * i < E) tiles += cdiv(n[i], BC);
    tiles = wave_sum(tiles);
    const int64_t items = (int64_t)tiles * p.rows_t, per = cdiv64(items, 8);
    const int64_t slot = blockIdx.x / 8, item = (blockIdx.x % 8) * per + slot;
    if (slot >= per || item >= items) return;
    const int number = (int)(item / p.rows_t);  // some tile of its expert
    int e = 0, before = 0, first = 0, count = 0, done = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        if (64 * i >= E) break;
        const int upto = done + wave_scan(cdiv(n[i], BC));
        const uint64_t m = __ballot(upto > number);
        if (m) {
            const int l = __builtin_ctzll(m);
            e = 64 * i + l;
            first = __builtin_amdgcn_readlane(begin[i], l);
            count = __builtin_amdgcn_readlane(n[i], l);
            before = __builtin_amdgcn_readlane(upto, l) - cdiv(count, BC);
            break;
        }
        done = __builtin_amdgcn_readlane(upto, 63);
    }
    const int nt = cdiv(count, BC);  // tiles of pairs of the expert
    const int in = (int)(item - (int64_t)before * p.rows_t), tk = in / nt, skip = (in - tk * nt) * BC;
    const int tr = SWIGLU ? tk : tk / p.splits, split = SWIGLU ? 0 : tk - tr * p.splits;
    first += skip;
    count = min(BC, count - skip);
    // the tile's pairs to LDS
    if (p.off) {
        if (tid < BC) pairs[tid] = p.order[first + min(tid, count - 1)];
    } else {
        // a thread's matches come after those of the threads before it
        int mine = 0;
#pragma unroll
        for (int i = 0; i < SCAN / 4; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) mine += id[i][v] == (unsigned)e;
        const int upto = wave_scan(mine);
        int* const waves = counts + CLOVE_MAX_EXPERTS;
        if (lane == 63) waves[wave] = upto;
        __syncthreads();
        int at = upto - mine - skip;
#pragma unroll
        for (int w = 0; w < CF::NW; ++w)
            if (w < wave) at += waves[w];
#pragma unroll
        for (int i = 0; i < SCAN / 4; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (id[i][v] == (unsigned)e) {
                    if ((unsigned)at < (unsigned)count) pairs[at] = 4 * (i * CF::NT + tid) + v;
                    ++at;
                }
    }
    __syncthreads();

    constexpr int OR = SWIGLU ? BR / 2 : BR;  // outputs of a tile
    const int r0 = p.o0 + tr * OR, O = a.O, K = a.K, G = p.G;
    const int end = SWIGLU ? O : p.o0 + p.on;
    const int R = SWIGLU ? 2 * O : O;
    // weight row of tile row i (past the end: the last one, whose results go nowhere)
    auto row = [&](int i) {
        if constexpr (SWIGLU) return ((i & 16) ? O : 0) + min(r0 + 16 * (i >> 5) + (i & 15), O - 1);
        else return min(r0 + i, O - 1);
    };
    const unsigned lds0 =
        __builtin_amdgcn_readfirstlane((unsigned)(size_t)((__attribute__((address_space(3))) unsigned char*)smem));

    // ---- DMA descriptors and per-lane offsets.  An offset of 2^31 lies past every
    // buffer (all are shorter) and reads zeros ----
    constexpr unsigned kPast = 0x80000000u;
    const int64_t srow0 = (int64_t)e * R * G * 2;
    const uintptr_t sb = reinterpret_cast<uintptr_t>(a.scale) + srow0, zb = reinterpret_cast<uintptr_t>(a.zero) + srow0;
    const int so = (int)(sb & 3), zo = (int)(zb & 3);
    const unsigned sbytes = ((unsigned)R * G * 2 + 2u + 3u) & ~3u;
    const u32x4 rx = make_rsrc(a.X, (unsigned)p.x_bytes);
    const u32x4 rw = make_rsrc(a.W + (int64_t)e * R * (K / 2), (unsigned)R * (K / 2));
    const u32x4 rs = make_rsrc(reinterpret_cast<const void*>(sb & ~(uintptr_t)3), sbytes);
    const u32x4 rz = make_rsrc(reinterpret_cast<const void*>(zb & ~(uintptr_t)3), sbytes);
    constexpr int XC = CF::XRB / 16, WC16 = CF::WRB / 16;  // 16-byte chunks of a row
    int offx[CF::DX], offw[CF::DW], offs[CF::DS];
    auto xrow = [&](int i) { return 64 / XC * (wave * CF::DX + i) + lane / XC; };
    auto xchunk = [&](int i) { return (lane % XC) ^ swz_x<KS>(xrow(i)); };
#pragma unroll
    for (int i = 0; i < CF::DX; ++i) {
        const int q = pairs[min(xrow(i), count - 1)];
        offx[i] = p.x.div(q) * K * 2 + 16 * xchunk(i);
    }
#pragma unroll
    for (int i = 0; i < CF::DW; ++i) {
        const int r = 64 / WC16 * (wave * CF::DW + i) + lane / WC16;
        offw[i] = row(r) * (K / 2) + 16 * ((lane % WC16) ^ swz_w<KS>(r));
    }
#pragma unroll
    for (int i = 0; i < CF::DS; ++i) {
        const int j = wave * CF::DS + i;
        offs[i] = row(64 * (j % (BR / 64)) + lane) * G * 2 + (j >= BR / 64 ? zo : so);
    }
    // stages of the tile
    const int first_stage = split * p.split_groups * SPG, NS = min(cdiv(K, 16 * KS), first_stage + p.split_groups * SPG);
    // stage t to buffer b; HS: its place in the group
    auto issue = [&](int t, int b, bool starts) {
        const unsigned st = __builtin_amdgcn_readfirstlane(lds0 + (unsigned)(b * CF::STAGE));
        if (16 * KS * (t + 1) > K) {
#pragma unroll
            for (int i = 0; i < CF::DX; ++i)
                dma16(rx, st + (wave * CF::DX + i) * 1024, 16 * KS * t + 8 * xchunk(i) < K ? offx[i] : (int)kPast, t * CF::XRB);
        } else {
#pragma unroll
            for (int i = 0; i < CF::DX; ++i) dma16(rx, st + (wave * CF::DX + i) * 1024, offx[i], t * CF::XRB);
        }
#pragma unroll
        for (int i = 0; i < CF::DW; ++i) dma16(rw, st + CF::OFF_W + (wave * CF::DW + i) * 1024, offw[i], t * CF::WRB);
        if (starts) {
            const int g = t / SPG;
#pragma unroll
            for (int i = 0; i < CF::DS; ++i) {
                const int j = wave * CF::DS + i;
                const bool is_zero = j >= BR / 64;
                dma4(is_zero ? rz : rs, st + (is_zero ? CF::OFF_ZR : CF::OFF_SC) + (j % (BR / 64)) * 256, (offs[i] + 2 * g) & ~3, 0);
            }
        }
    };

    // ---- fragments: X row x, step s at XRB x + 16 ((KS h + s) ^ swz(x)); weight row r,
    // 32-k chunk c at WRB r + 16 ((NWC h + c) ^ swz(r)) ----
    const int h = lane >> 5, l32 = lane & 31;
    const int xrow0 = wc * 32 * FX + l32, wrow0 = wr * 32 * FW + l32;
    constexpr int NWC = KS / 4;
    unsigned xoff[KS], woff[NWC];
#pragma unroll
    for (int s = 0; s < KS; ++s) xoff[s] = xrow0 * CF::XRB + 16 * ((KS * h + s) ^ swz_x<KS>(xrow0));
#pragma unroll
    for (int c = 0; c < NWC; ++c) woff[c] = CF::OFF_W + wrow0 * CF::WRB + 16 * ((NWC * h + c) ^ swz_w<KS>(wrow0));
    int soff[FW];  // bit 1: which half of the dword holds the scale at group 0, bit 0: the zero point
#pragma unroll
    for (int i = 0; i < FW; ++i) {
        const int at = row(wrow0 + 32 * i) * G * 2;
        soff[i] = ((at + so) & 2) | (((at + zo) >> 1) & 1);
    }

    f32x16 acc[FW][FX] = {};
    float unit[FW];
    f16x2 zz[FW], mul[FW];
#pragma unroll
    for (int i = 0; i < FW; ++i) unit[i] = 1.0f;
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
        if (first_stage + t < NS) issue(first_stage + t, t, t % SPG == 0);
    int stage = 0, stage_next = S - 1;
    // (FXU blocks of 32 pairs; the others of a ragged tile multiply nothing)
    auto k_loop = [&](auto blocks) {
        constexpr int FXU = decltype(blocks)::value;
        for (int t0 = first_stage; t0 < NS; t0 += SPG) {
#pragma unroll
            for (int hs = 0; hs < SPG; ++hs) {
                const int t = t0 + hs;
                if (SPG > 1 && t >= NS) break;
                // stage t landed (what was issued after it may stay in flight), then the
                // barrier: every wave's part of it has, and every wave has read stage t - 1,
                // whose buffer the next issue writes
                const int ahead = min(S - 2, NS - 1 - t);
                if (S > 3 && ahead >= 2) wait_vm<vmcnt_imm(CF::dmas(0) + CF::dmas(1))>();
                else if (S > 2 && ahead >= 1 && hs == 0) wait_vm<vmcnt_imm(CF::dmas(1))>();
                else if (S > 2 && ahead >= 1) wait_vm<vmcnt_imm(CF::dmas(0))>();
                else wait_vm<vmcnt_imm(0)>();
                dma::stage_barrier<0xc07f>();
                if (t + S - 1 < NS) issue(t + S - 1, stage_next, (hs + S - 1) % SPG == 0);
                const unsigned st = __builtin_amdgcn_readfirstlane(lds0 + (unsigned)(stage * CF::STAGE));
                stage_next = stage;
                stage = stage + 1 == S ? 0 : stage + 1;
                float ratio[FW];
                u32x4 wraw[FW][NWC];
#pragma unroll
                for (int c = 0; c < NWC; ++c)
#pragma unroll
                    for (int i = 0; i < FW; ++i) wraw[i][c] = lds_read16(st + woff[c] + 32 * CF::WRB * i);
                if (hs == 0) {
                    const int odd = (t / SPG) & 1;
#pragma unroll
                    for (int i = 0; i < FW; ++i) {
                        const unsigned sd = lds_read4(st + CF::OFF_SC + (wrow0 + 32 * i) * 4);
                        const unsigned zd = lds_read4(st + CF::OFF_ZR + (wrow0 + 32 * i) * 4);
                        const float sc = h2f((uint16_t)((soff[i] >> 1) ^ odd ? sd >> 16 : sd));
                        const float z = rintf(h2f((uint16_t)((soff[i] & 1) ^ odd ? zd >> 16 : zd)));
                        const bool none = sc == 0.0f;
                        ratio[i] = none ? 1.0f : unit[i] / sc;
                        unit[i] = none ? unit[i] : sc;
                        const _Float16 nz = (_Float16)(z * (none ? 0.0f : -1.0f / 512.0f));
                        zz[i] = f16x2{nz, nz};
                        mul[i] = none ? f16x2{(_Float16)0.0f, (_Float16)0.0f} : f16x2{(_Float16)2048.0f, (_Float16)32768.0f};
                    }
                }
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    f16x8 xf[FXU], wf[FW];
#pragma unroll
                    for (int j = 0; j < FXU; ++j) xf[j] = bitcast<f16x8>(lds_read16(st + xoff[s] + 32 * CF::XRB * j));
#pragma unroll
                    for (int i = 0; i < FW; ++i) {
                        const u32x4& q = wraw[i][s >> 2];
                        wf[i] = unpack8((s & 3) == 0 ? q.x : (s & 3) == 1 ? q.y : (s & 3) == 2 ? q.z : q.w, mul[i], zz[i]);
                    }
#pragma unroll
                    for (int i = 0; i < FW; ++i)
#pragma unroll
                        for (int j = 0; j < FXU; ++j) {
                            if (hs == 0 && s == 0) acc[i][j] *= ratio[i];
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[j], wf[i], acc[i][j], 0, 0, 0);
                        }
                }
            }
        }
    };
    // An expert's last tile may be half empty (4096 pairs on 8 experts: 762 us without the
    // second loop, 748 with it; 65536 on 128 426 and 418)
    if (FX > 1 && count <= 16 * FX) k_loop(std::integral_constant<int, (FX + 1) / 2>());
    else k_loop(std::integral_constant<int, FX>());
#pragma unroll
    for (int i = 0; i < FW; ++i) unit[i] *= 512.0f;  // (q - z) 2^-9 back to q - z
#pragma unroll
    for (int i = 0; i < FW; ++i)
#pragma unroll
        for (int j = 0; j < FX; ++j) acc[i][j] *= unit[i];

    // ---- stores.  A lane holds one weight row of pairs 8 q + 4 h + v of each 32: the wave
    // turns them in LDS, 32 pairs at a time in a part of its own, and stores 16 bytes of a
    // pair's row a lane (4-byte stores, four times as many, were 20 % of the call that
    // multiplies 65536 pairs by rows of 768) ----
    __syncthreads();  // (the last stage has been read)
    const int c0 = wc * 32 * FX;
    if constexpr (SWIGLU) {
        constexpr int LD = CF::turned_row(true), LPP = 2 * FW;  // halves of a turned row, lanes a pair
        uint16_t* turned = reinterpret_cast<uint16_t*>(smem) + wave * 32 * LD;
#pragma unroll
        for (int j = 0; j < FX; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int v = 0; v < 4; v += 2)
#pragma unroll
                    for (int i = 0; i < FW; ++i) {
                        // (gate, up) of pair v to lane l, of pair v + 1 to lane l ^ 16
                        const auto sw = __builtin_amdgcn_permlane16_swap(bitcast<unsigned>(acc[i][j][4 * q + v]),
                                                                         bitcast<unsigned>(acc[i][j][4 * q + v + 1]), false, false);
                        const float x = bitcast<float>(sw[0]), u = bitcast<float>(sw[1]);
                        turned[(8 * q + 4 * h + v + (l32 >> 4)) * LD + 16 * i + (l32 & 15)] = f2h(x / (1.0f + expf(-x)) * u);
                    }
            asm volatile("" ::: "memory");  // (one wave's LDS accesses take effect in order)
            const int o = r0 + 16 * FW * wr + 8 * (lane % LPP), n = O - o;
#pragma unroll
            for (int k = 0; k < 32; k += 64 / LPP) {
                const int c = k + lane / LPP, at = c0 + 32 * j + c;
                if (c >= 32 || at >= count || n <= 0) continue;
                const u32x4 y = *reinterpret_cast<const u32x4*>(turned + c * LD + 8 * (lane % LPP));
                uint16_t* to = a.Y + (int64_t)pairs[at] * O + o;
                if (n >= 8) {
                    *reinterpret_cast<u32x4u*>(to) = y;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < n) to[i] = (uint16_t)(y[i >> 1] >> (16 * (i & 1)));
                }
            }
            asm volatile("" ::: "memory");
        }
    } else {
        constexpr int LD = CF::turned_row(false), LPP = 8 * FW;  // floats of a turned row, lanes a pair
        float* turned = reinterpret_cast<float*>(smem) + wave * 32 * LD;
#pragma unroll
        for (int j = 0; j < FX; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int i = 0; i < FW; ++i) turned[(8 * q + 4 * h + v) * LD + 32 * i + l32] = acc[i][j][4 * q + v];
            asm volatile("" ::: "memory");
            const int o = r0 + 32 * FW * wr + 4 * (lane % LPP);
#pragma unroll
            for (int k = 0; k < 32; k += 64 / LPP) {
                const int c = k + lane / LPP, at = c0 + 32 * j + c;
                if (at >= count || o >= end) continue;
                // (rows of the products have room for whole fours)
                *reinterpret_cast<f32x4*>(p.part + ((int64_t)split * p.P + pairs[at]) * p.ldp + o - p.o0) =
                    *reinterpret_cast<const f32x4*>(turned + c * LD + 4 * (lane % LPP));
            }
            asm volatile("" ::: "memory");
        }
    }
}

// Y[t, o0 + o] = alpha sum_j w[t, j] part[t top_k + j, o] + beta Y, places in order; a
// place without an expert is left out.  A thread takes four outputs of one token, and
// eight places' parts are in flight at once: 8192 tokens of 8 places and 2048 outputs, 570
// MB, 120 us, 4.7 TB/s.
__global__ void __launch_bounds__(128) moe_combine(const Params p) {
    const MoeArgs& a = p.a;
    const int t = blockIdx.x, o = 512 * blockIdx.y + 4 * threadIdx.x;
    const int n = min(4, p.on - o);
    if (n <= 0) return;
    const float* part = p.part + (int64_t)t * a.top_k * p.ldp + o;
    const int32_t* ids = a.ids + (int64_t)t * a.top_k;
    f32x4 sum = {};
    for (int j0 = 0; j0 < a.top_k; j0 += 8) {
        f32x4 v[8];
        float w[8];
        bool there[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            there[j] = j0 + j < a.top_k && (unsigned)ids[min(j0 + j, a.top_k - 1)] < (unsigned)a.experts;
            w[j] = 0.0f;
            v[j] = f32x4{};
            if (there[j]) {
                w[j] = a.weights ? a.weights[(int64_t)t * a.top_k + j0 + j] : 1.0f;
                v[j] = *reinterpret_cast<const f32x4*>(part + (int64_t)(j0 + j) * p.ldp);
            }
        }
#pragma unroll 2
        for (int s = 1; s < p.splits; ++s) {
            const float* more = part + ((int64_t)s * p.P + j0) * p.ldp;
            f32x4 m[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = *reinterpret_cast<const f32x4*>(more + (int64_t)min(j, a.top_k - 1 - j0) * p.ldp);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (there[j]) v[j] += m[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = fmaf(w[j], v[j][i], sum[i]);
    }
    uint16_t* y = a.Y + (int64_t)t * a.O + p.o0 + o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum[i] *= a.alpha;
        if (a.beta != 0.0f && i < n) sum[i] = fmaf(a.beta, h2f(y[i]), sum[i]);
    }
    if (n == 4) {
        *reinterpret_cast<u32x2u*>(y) = u32x2{pack2h(sum[0], sum[1]), pack2h(sum[2], sum[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) y[i] = f2h(sum[i]);
    }
}

// H[q, i] from the parts of K of the pairs' gate and up products, part[s][q][i] and
// [I + i], in order: some 4 us, a launch and a memory latency for two parts
__global__ void __launch_bounds__(128) moe_swiglu(const Params p) {
    const MoeArgs& a = p.a;
    const int q = blockIdx.x, i = 512 * blockIdx.y + 4 * threadIdx.x, I = a.O / 2, n = min(4, I - i);
    if (n <= 0 || (unsigned)a.ids[q] >= (unsigned)a.experts) return;
    const float* part = p.part + (int64_t)q * p.ldp + i;
    f32x4 g = {}, u = {};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s, part += (int64_t)p.P * p.ldp) {
        g += *reinterpret_cast<const f32x4*>(part);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] += part[I + min(j, n - 1)];
    }
    uint16_t* h = a.Y + (int64_t)q * I + i;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < n) h[j] = f2h(g[j] / (1.0f + expf(-g[j])) * u[j]);
}

namespace {

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

// ---- few pairs ----
// Waves that share K: four, two once workgroups of two cover the CUs eight times (32 tokens
// on 8 of 128 experts of 2 x 768 rows of 2048: 47 us against 54; 8 tokens 24 and 24.6; 1
// token 8.5 against 7.0).
int few_waves(int64_t workgroups, int cus) { return workgroups >= 8 * (int64_t)cus ? 2 : 4; }

template <bool SWIGLU, int TB, bool PF>
clove_status_t run_few(Params p, int cus, hipStream_t stream) {
    p.rows_t = cdiv(p.on, SWIGLU ? 16 : 32);
    p.by_expert = p.P > p.a.experts;
    const int64_t grid = (int64_t)(p.by_expert ? p.a.experts : p.P) * p.rows_t;
    const int KS = few_waves(grid, cus);
    if (too_many(grid, 64 * KS)) return CLOVE_ERR_INVALID_DIM;
    p.ng = min(NG, cdiv(p.G, KS));
    // (units, lists, sums: see the kernel)
    const int lds = KS * UnitLds<2, TB>::BYTES + (KS * p.P * 4 + 15) / 16 * 16 + KS * 2048;
    auto k = moe_few<SWIGLU, TB, PF>;
    if (ensure_lds(reinterpret_cast<const void*>(k), lds) != CLOVE_OK) return CLOVE_ERR_LAUNCH;
    CLOVE_LAUNCH(k, dim3((unsigned)grid), dim3(64 * KS), lds, stream, p);
    return check_launch();
}

template <int WF>
clove_status_t run_few_down(Params p, int KS, hipStream_t stream) {
    p.rows_t = cdiv(p.a.O, 16 * WF);
    // as many units as waves where the groups allow it
    const int parts = max(cdiv(p.G, NG), min(p.G, cdiv(KS, p.a.top_k)));
    p.ng = cdiv(p.G, parts);
    KS = min(KS, p.a.top_k * cdiv(p.G, p.ng));
    if (too_many((int64_t)p.a.T * p.rows_t, 64 * KS)) return CLOVE_ERR_INVALID_DIM;
    CLOVE_LAUNCH(moe_few_down<WF>, dim3((unsigned)(p.a.T * p.rows_t)), dim3(64 * KS), KS * (UnitLds<WF, 1>::BYTES + 64 * WF), stream, p);
    return check_launch();
}

// ---- tiles ----
template <class CF, bool SWIGLU>
clove_status_t run_tile(Params p, hipStream_t stream) {
    p.rows_t = cdiv(p.on, SWIGLU ? CF::BR / 2 : CF::BR) * p.splits;
    const int64_t tiles = ((int64_t)p.P / CF::BC + p.a.experts) * p.rows_t;
    if (too_many(tiles + 7, CF::NT)) return CLOVE_ERR_INVALID_DIM;
    auto k = moe_tile<CF, SWIGLU>;
    if (ensure_lds(reinterpret_cast<const void*>(k), CF::LDS) != CLOVE_OK) return CLOVE_ERR_LAUNCH;
    CLOVE_LAUNCH(k, dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(CF::NT), CF::LDS, stream, p);
    return check_launch();
}

// Shapes (plan() chooses)
using Many = Cfg<4, 1, 2, 4, 2, 4>;   // 256 x 128
using Some = Cfg<4, 1, 1, 2, 2, 8>;   // 128 x 64
using Thin = Cfg<4, 1, 1, 1, 3, 8>;   // 128 x 32
using Small = Cfg<2, 1, 1, 1, 4, 8>;  // 64 x 32

template <class CF>
constexpr bool is(Shape s) {
    return CF::BR == dims(s).rows && CF::BC == dims(s).pairs;
}
static_assert(is<Many>(Shape::kMany) && is<Some>(Shape::kSome) && is<Thin>(Shape::kThin) && is<Small>(Shape::kSmall), "moe_plan.hpp");

template <bool SWIGLU>
clove_status_t run_shape(Shape s, const Params& p, hipStream_t stream) {
    if (s == Shape::kMany) return run_tile<Many, SWIGLU>(p, stream);
    if (s == Shape::kSome) return run_tile<Some, SWIGLU>(p, stream);
    if (s == Shape::kThin) return run_tile<Thin, SWIGLU>(p, stream);
    return run_tile<Small, SWIGLU>(p, stream);
}

// The call's kernels and scratch, settled by the first of its parts, whose pairs are the most
struct Held {
    bool begun = false;
    Choice by;
    void* p = nullptr;
    size_t bytes = 0;
};

template <bool SWIGLU>
clove_status_t run(const MoeArgs& a, int cus, hipStream_t stream, Held& held) {
    Params p{};
    p.a = a;
    p.P = a.T * a.top_k;
    p.G = cdiv(a.K, 128);
    p.k = FastDiv(a.top_k);
    p.x = FastDiv(SWIGLU ? a.top_k : 1);
    p.splits = 1;
    p.split_groups = p.G;
    p.x_bytes = (int64_t)(SWIGLU ? a.T : p.P) * a.K * 2;
    const bool aligned = a.K > 0 && a.K % 32 == 0 && aligned16(a.X) && aligned16(a.W);
    if (!held.begun) held.by = choose({SWIGLU, aligned, a.T, a.top_k, a.experts, a.O, a.K, cus});
    held.begun = true;
    const Choice& by = held.by;
    if constexpr (!SWIGLU)
        if (by.way == Way::kToken) return by.blocks == 1 ? run_few_down<1>(p, by.waves, stream) : run_few_down<2>(p, by.waves, stream);
    // Scratch: the lists of the pairs by expert, for down the products with `chunk` outputs at a
    // time, the products of parts of K up to 64 MB
    const bool lists = (by.way == Way::kTiles && p.P > SCAN * 128) || by.way == Way::kAny;
    const size_t off = lists ? round256((size_t)(a.experts + 1) * 4) : 0, order = lists ? round256((size_t)p.P * 4) : 0;
    if (by.way == Way::kTiles) {
        p.split_groups = cdiv(p.G, by.splits);
        p.splits = cdiv(p.G, p.split_groups);
    }
    if (!SWIGLU || p.splits > 1) p.ldp = ((SWIGLU ? 2 * a.O : min(by.chunk, a.O)) + 3) & ~3;
    const size_t bytes = off + order + (size_t)p.splits * p.P * p.ldp * 4;
    if (bytes > held.bytes) {
        if (const clove_status_t st = acquire_buffer(stream, kBufMoe, bytes, &held.p); st != CLOVE_OK) return st;
        held.bytes = bytes;
    }
    p.off = lists ? static_cast<int*>(held.p) : nullptr;
    p.order = reinterpret_cast<int*>(static_cast<char*>(held.p) + off);
    p.part = reinterpret_cast<float*>(static_cast<char*>(held.p) + off + order);
    if (lists) {
        const int threads = min(kSortThreads, cdiv(p.P, 256) * 64);
        CLOVE_LAUNCH(moe_sort, dim3((unsigned)a.experts), dim3((unsigned)threads), 0, stream, a.ids, p.P, a.experts, p.off, p.order);
    }
    if (SWIGLU && p.splits > 1) {
        // (the products of gate and up rows as of any others, and SwiGLU of their sums)
        p.a.O = p.on = 2 * a.O;
        if (const clove_status_t st = run_shape<false>(by.shape, p, stream); st != CLOVE_OK) return st;
        CLOVE_LAUNCH(moe_swiglu, dim3((unsigned)p.P, (unsigned)cdiv(a.O, 512)), dim3(128), 0, stream, p);
        return check_launch();
    }
    for (int64_t o = 0; o < a.O; o += by.chunk) {
        p.o0 = (int)o;
        p.on = min(by.chunk, a.O - p.o0);
        clove_status_t st = CLOVE_OK;
        if (by.way == Way::kExpert) {
            st = by.pairs == 2 ? run_few<SWIGLU, 2, true>(p, cus, stream) : run_few<SWIGLU, 8, false>(p, cus, stream);
        } else if (by.way == Way::kTiles) {
            st = run_shape<SWIGLU>(by.shape, p, stream);
        } else {
            p.rows_t = cdiv(p.on, SWIGLU ? AR / 2 : AR);
            const int64_t grid = ((int64_t)p.P / AC + a.experts) * p.rows_t;
            if (too_many(grid, 256)) return CLOVE_ERR_INVALID_DIM;
            CLOVE_LAUNCH(moe_any<SWIGLU>, dim3((unsigned)grid), dim3(256), 0, stream, p);
            st = check_launch();
        }
        if (st != CLOVE_OK) return st;
        if constexpr (!SWIGLU)
            CLOVE_LAUNCH(moe_combine, dim3((unsigned)a.T, (unsigned)cdiv(p.on, 512)), dim3(128), 0, stream, p);
    }
    return check_launch();
}

}  // namespace
}  // namespace moe

clove_status_t launch_moe_w4a16(const MoeArgs& a, bool swiglu, hipStream_t stream) {
    using namespace moe;
    DeviceInfo dev;
    if (const clove_status_t st = current_device_info(&dev); st != CLOVE_OK) return st;
    const int64_t per_token = (int64_t)(swiglu ? 1 : a.top_k) * a.K * 2, most = tokens_at_a_time(swiglu, a.top_k, a.K);
    if (most < 1) return CLOVE_ERR_INVALID_DIM;
    Held held;
    for (int64_t t = 0; t < a.T;) {
        // (equal parts)
        const int n = (int)cdiv64(a.T - t, cdiv64(a.T - t, most));
        MoeArgs part = a;
        part.T = n;
        part.X = a.X ? a.X + t * (per_token / 2) : nullptr;
        part.ids = a.ids + t * a.top_k;
        part.weights = a.weights ? a.weights + t * a.top_k : nullptr;
        part.Y = a.Y + t * (swiglu ? a.top_k : 1) * a.O;
        const clove_status_t st = swiglu ? run<true>(part, dev.num_cus, stream, held) : run<false>(part, dev.num_cus, stream, held);
        if (st != CLOVE_OK) return st;
        t += n;
    }
    return CLOVE_OK;
}

}  // namespace clove
