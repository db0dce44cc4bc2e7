// Norms of queries and keys per head, position rotation and the cache write of
// keys and values, one pass over the fused QKV projection's rows.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w,  (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// in fp32 from the loaded element to the one rounding at the store.  Every
// element is read once and written once, a handful of flops each: HBM-bound
// for many tokens, launch-bound for one.
#include <algorithm>
#include <type_traits>

#include "decode.hpp"

namespace clove {
namespace rope {

using namespace hw;

struct Params {
    RopeArgs a;
    FastDiv page;  // by the page size
    int heads;     // queries, keys and, with a cache, values
    FastDiv parts; // waves per token, each with `rounds` times the heads a wave holds at once
    int rounds;
};

// Where head `h` of token t goes: up to two places (a dense row and the cache).
template <typename P>
struct Places {
    P* dense;
    P* cached;
};
__device__ __forceinline__ Places<uint16_t> places(const Params& q, int t, int h, int slot) {
    const RopeArgs& a = q.a;
    Places<uint16_t> p{nullptr, nullptr};
    const int kh = h - a.q_heads, vh = kh - a.kv_heads;
    if (kh < 0) {
        p.dense = a.q_out + (int64_t)t * a.q_out_stride + (int64_t)h * a.head_dim;
        return p;
    }
    if (vh < 0 && a.k_out) p.dense = a.k_out + (int64_t)t * a.k_out_stride + (int64_t)kh * a.head_dim;
    if (slot >= 0) {
        const int page = q.page.div(slot);
        if (page < a.cache.num_pages) {
            const int64_t at = (int64_t)page * a.cache.page_stride +
                               ((int64_t)(vh < 0 ? kh : vh) * a.cache.page_size + (slot - page * a.cache.page_size)) *
                                   a.cache.head_dim;
            p.cached = (vh < 0 ? a.cache.k : a.cache.v) + at;
        }
    }
    return p;
}

template <typename T>
__device__ __forceinline__ void put(const Places<T>& p, int d, T x) {
    if (p.dense) p.dense[d] = x;
    if (p.cached) p.cached[d] = x;
}

// Any head_dim, stride and alignment: one wave per (token, head), an element
// pair per lane.
template <int DT>
__global__ void __launch_bounds__(256) rope_any(const Params p) {
    using E = Elem<DT>;
    const RopeArgs& a = p.a;
    const int lane = threadIdx.x & 63, D = a.head_dim, R = a.rot_dim, half = R >> 1;
    const int64_t tasks = (int64_t)a.T * p.heads;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < tasks; i += (int64_t)gridDim.x * 4) {
        const int t = (int)(i / p.heads), h = (int)(i - (int64_t)t * p.heads);
        const uint16_t* x = a.qkv + (int64_t)t * a.qkv_stride + (int64_t)h * D;
        const Places<uint16_t> to = places(p, t, h, a.cache.k ? a.slots[t] : -1);
        if (h >= a.q_heads + a.kv_heads) {  // a value: moved as it is
            if (to.cached)
                for (int d = lane; d < D; d += 64) to.cached[d] = x[d];
            continue;
        }
        if (!to.dense && !to.cached) continue;
        const uint16_t* w = h < a.q_heads ? a.q_weight : a.k_weight;
        float r = 1.0f;
        if (w) {
            float sum = 0.0f;
            for (int d = lane; d < D; d += 64) {
                const float v = E::load(x[d]);
                sum = fmaf(v, v, sum);
            }
            r = 1.0f / sqrtf(wave_sum(sum) / (float)D + a.eps);
        }
        auto y = [&](int d) { return w ? E::load(x[d]) * r * E::load(w[d]) : E::load(x[d]); };
        const int pos = R ? a.positions[t] : 0;
        const bool known = (unsigned)pos < (unsigned)a.max_position;
        for (int j = lane; j < half; j += 64) {
            const int d0 = a.interleaved ? 2 * j : j, d1 = a.interleaved ? 2 * j + 1 : j + half;
            const float c = known ? a.cos[(int64_t)pos * half + j] : __builtin_nanf("");
            const float s = known ? a.sin[(int64_t)pos * half + j] : __builtin_nanf("");
            const float u = y(d0), v = y(d1);
            put(to, d0, E::store(fmaf(u, c, -(v * s))));
            put(to, d1, E::store(fmaf(v, c, u * s)));
        }
        for (int d = R + lane; d < D; d += 64) put(to, d, E::store(known || !R ? y(d) : __builtin_nanf("")));
    }
}

// Rows of whole chunks of CH elements (16 bytes for CH = 8): a lane holds one
// unit of two chunks -- CH pairs of the rotation, or 2 CH elements that it passes
// over -- LPH lanes a head, 64 / LPH heads a wave at once, all of one token, so
// that the rotation's factors and the norms' weights are loaded once and used
// for every head of the wave.  With few tokens each wave takes one round of
// heads, so that the loads of a token are in flight together; with many, rounds
// follow each other with the next head's elements loaded ahead.
// 8192 tokens of 32 + 16 heads of 128 (206 MB): 44 us, 4.7 TB/s (236 with rope_any);
// 200 tokens 4.3, one 2.6.
template <int CH>
struct Chunk {
    typedef unsigned words __attribute__((ext_vector_type(CH / 2)));
    typedef float floats __attribute__((ext_vector_type(CH >= 4 ? 4 : 2)));
};
template <>
struct Chunk<2> {
    typedef unsigned words __attribute__((ext_vector_type(1)));
    typedef float floats __attribute__((ext_vector_type(2)));
};

// over the LPH lanes of a head (a power of two), every lane the same sum
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    auto dpp = [](float x, auto ctl) { return bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(x), decltype(ctl)::value, 0xf, 0xf, false)); };
    if constexpr (LPH >= 2) v = v + dpp(v, std::integral_constant<int, 0xb1>{});   // quad_perm 1032: l ^ 1
    if constexpr (LPH >= 4) v = v + dpp(v, std::integral_constant<int, 0x4e>{});   // quad_perm 2301: l ^ 2
    if constexpr (LPH >= 8) v = v + dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror: the other four of eight
    if constexpr (LPH >= 16) v = v + dpp(v, std::integral_constant<int, 0x140>{}); // row_mirror: the other eight of the row
    if constexpr (LPH >= 32) v = swap_sum16(v, v);
    if constexpr (LPH >= 64) v = swap_sum32(v, v);
    return v;
}

template <int DT, int CH, int LPH>
__global__ void __launch_bounds__(256) rope_units(const Params p) {
    using E = Elem<DT>;
    using W = typename Chunk<CH>::words;
    using F = typename Chunk<CH>::floats;
    constexpr int HS = 64 / LPH;
    const RopeArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = p.parts.div(wave), D = a.head_dim, R = a.rot_dim, half = R >> 1;
    if (t >= a.T) return;
    const int u = lane & (LPH - 1), h0 = (wave - t * p.parts.d) * (p.rounds * HS) + lane / LPH;
    // the lane's two chunks
    const bool turns = u * 2 * CH < R;
    int d0, d1;
    if (!turns || a.interleaved) {
        d0 = u * 2 * CH;
        d1 = d0 + CH;
    } else {
        d0 = u * CH;
        d1 = d0 + half;
    }
    const bool on0 = d0 < D, on1 = d1 < D;
    const uint16_t* x = a.qkv + (int64_t)t * a.qkv_stride;
    auto load = [&](const uint16_t* from, W (&y)[2]) {
        y[0] = on0 ? *reinterpret_cast<const W*>(from + d0) : W(0);
        y[1] = on1 ? *reinterpret_cast<const W*>(from + d1) : W(0);
    };
    W next[2] = {W(0), W(0)};
    if (h0 < p.heads) load(x + (int64_t)h0 * D, next);
    const int slot = a.cache.k ? a.slots[t] : -1;
    const int pos = R ? a.positions[t] : 0;
    const bool known = !R || (unsigned)pos < (unsigned)a.max_position;
    float c[CH], sn[CH];
    if (turns && known) {
        constexpr int FW = CH >= 4 ? 4 : 2;
#pragma unroll
        for (int i = 0; i < CH / FW; ++i) {
            const F fc = *reinterpret_cast<const F*>(a.cos + (int64_t)pos * half + u * CH + FW * i);
            const F fs = *reinterpret_cast<const F*>(a.sin + (int64_t)pos * half + u * CH + FW * i);
#pragma unroll
            for (int e = 0; e < FW; ++e) {
                c[FW * i + e] = fc[e];
                sn[FW * i + e] = fs[e];
            }
        }
    }
    W wq[2] = {W(0), W(0)}, wk[2] = {W(0), W(0)};
    if (a.q_weight) load(a.q_weight, wq);
    if (a.k_weight) load(a.k_weight, wk);

    for (int i = 0; i < p.rounds; ++i) {
        const int h = h0 + i * HS;
        W raw[2] = {next[0], next[1]};
        if (i + 1 < p.rounds && h + HS < p.heads) load(x + (int64_t)(h + HS) * D, next);
        if (h >= p.heads) continue;  // (whole heads: no lane of this one is left behind)
        const Places<uint16_t> to = places(p, t, h, slot);
        if (h < a.q_heads + a.kv_heads) {
            const bool query = h < a.q_heads, norm = query ? a.q_weight != nullptr : a.k_weight != nullptr;
            float y[2][CH];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < CH; ++e) y[k][e] = E::load((uint16_t)(raw[k][e / 2] >> (16 * (e & 1))));
            float r = 1.0f;
            if (norm) {
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < CH; ++e) sum = fmaf(y[k][e], y[k][e], sum);
                r = 1.0f / sqrtf(head_sum<LPH>(sum) / (float)D + a.eps);
            }
            if (!known) r = __builtin_nanf("");
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < CH; ++e) {
                    const unsigned w = query ? wq[k][e / 2] : wk[k][e / 2];
                    y[k][e] = norm ? y[k][e] * r * E::load((uint16_t)(w >> (16 * (e & 1)))) : y[k][e] * r;
                }
            if (turns && known) {
                auto turn = [&](float& v, float& w, int j) {
                    const float v2 = fmaf(v, c[j], -(w * sn[j]));
                    w = fmaf(w, c[j], v * sn[j]);
                    v = v2;
                };
                if (a.interleaved) {
#pragma unroll
                    for (int j = 0; j < CH; ++j) turn(y[2 * j / CH][2 * j % CH], y[2 * j / CH][2 * j % CH + 1], j);
                } else {
#pragma unroll
                    for (int j = 0; j < CH; ++j) turn(y[0][j], y[1][j], j);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < CH; e += 2)
                    raw[k][e / 2] = (unsigned)E::store(y[k][e]) | ((unsigned)E::store(y[k][e + 1]) << 16);
        }
        if (to.dense) {
            if (on0) *reinterpret_cast<W*>(to.dense + d0) = raw[0];
            if (on1) *reinterpret_cast<W*>(to.dense + d1) = raw[1];
        }
        if (to.cached) {
            if (on0) *reinterpret_cast<W*>(to.cached + d0) = raw[0];
            if (on1) *reinterpret_cast<W*>(to.cached + d1) = raw[1];
        }
    }
}

template <int DT, int CH>
void launch_units(Params& p, int lph, int cus, hipStream_t stream) {
    typedef void (*Kernel)(const Params);
    const Kernel kernel = lph == 4    ? (Kernel)rope_units<DT, CH, 4>
                          : lph == 8  ? (Kernel)rope_units<DT, CH, 8>
                          : lph == 16 ? (Kernel)rope_units<DT, CH, 16>
                          : lph == 32 ? (Kernel)rope_units<DT, CH, 32>
                                      : (Kernel)rope_units<DT, CH, 64>;
    // one round per wave until there are 16 waves per CU, then as many as keep that
    const int most = cdiv(p.heads, 64 / lph);
    p.rounds = (int)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)p.a.T * most / (16 * cus)));
    p.parts = FastDiv(cdiv(most, p.rounds));
    const int64_t waves = (int64_t)p.a.T * p.parts.d;
    CLOVE_LAUNCH(kernel, dim3((unsigned)cdiv64(waves, 4)), dim3(256), 0, stream, p);
}

}  // namespace rope

clove_status_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    const clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    rope::Params p{};
    p.a = a;
    p.heads = a.q_heads + (a.cache.k ? 2 : a.k_out ? 1 : 0) * a.kv_heads;
    if (a.cache.k) p.page = FastDiv(a.cache.page_size);
    // The largest chunk that rows, halves of the rotation and addresses are whole
    // multiples of (an address of 2 ch bytes; the factors' too)
    int ch = 8;
    for (; ch > 1; ch >>= 1) {
        const uintptr_t bytes = (uintptr_t)2 * ch - 1, factors = ch >= 4 ? 15 : 7;
        auto at = [&](const void* x) { return (reinterpret_cast<uintptr_t>(x) & bytes) == 0; };
        auto table = [&](const void* x) { return !a.rot_dim || (reinterpret_cast<uintptr_t>(x) & factors) == 0; };
        if (a.head_dim % ch == 0 && a.rot_dim % (2 * ch) == 0 && a.qkv_stride % ch == 0 && a.q_out_stride % ch == 0 &&
            a.k_out_stride % ch == 0 && a.cache.page_stride % ch == 0 && at(a.qkv) && at(a.q_out) && at(a.k_out) && at(a.cache.k) &&
            at(a.cache.v) && at(a.q_weight) && at(a.k_weight) && table(a.cos) && table(a.sin))
            break;
    }
    const int units = ch > 1 ? hw::cdiv(a.head_dim, 2 * ch) : 0;
    const int64_t tasks = (int64_t)a.T * p.heads;
    if (tasks == 0) return CLOVE_OK;
    if (units >= 1 && units <= 64 && tasks < (1 << 30)) {
        int lph = 4;
        while (lph < units) lph *= 2;
        if (a.dtype == CLOVE_DTYPE_FP16)
            ch == 8   ? rope::launch_units<CLOVE_DTYPE_FP16, 8>(p, lph, dev.num_cus, stream)
            : ch == 4 ? rope::launch_units<CLOVE_DTYPE_FP16, 4>(p, lph, dev.num_cus, stream)
                      : rope::launch_units<CLOVE_DTYPE_FP16, 2>(p, lph, dev.num_cus, stream);
        else
            ch == 8   ? rope::launch_units<CLOVE_DTYPE_BF16, 8>(p, lph, dev.num_cus, stream)
            : ch == 4 ? rope::launch_units<CLOVE_DTYPE_BF16, 4>(p, lph, dev.num_cus, stream)
                      : rope::launch_units<CLOVE_DTYPE_BF16, 2>(p, lph, dev.num_cus, stream);
        return check_launch();
    }
    const int64_t blocks = std::min<int64_t>(hw::cdiv64(tasks, 4), 64 * dev.num_cus);
    const auto kernel = a.dtype == CLOVE_DTYPE_FP16 ? rope::rope_any<CLOVE_DTYPE_FP16> : rope::rope_any<CLOVE_DTYPE_BF16>;
    CLOVE_LAUNCH(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return check_launch();
}

}  // namespace clove
