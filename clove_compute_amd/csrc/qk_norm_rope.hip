// Norms of queries and keys per head, position rotation and the cache write of
// keys and values, one pass over the fused QKV projection's rows.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w,  (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// in fp32 from the loaded element to the one rounding at the store.  Every
// element is read once and written once, a handful of flops each: HBM-bound
// for many tokens, launch-bound for one.
#include <algorithm>

#include "decode.hpp"

namespace clove {
namespace rope {

using namespace hw;

struct Params {
    RopeArgs a;
    int heads;  // q_heads + 2 kv_heads
};

// Where head `h` of token t goes: up to two places (a dense row and the cache).
template <typename P>
struct Places {
    P* dense;
    P* cached;
};
__device__ __forceinline__ Places<uint16_t> places(const RopeArgs& a, int t, int h) {
    Places<uint16_t> p{nullptr, nullptr};
    const int kh = h - a.q_heads, vh = kh - a.kv_heads;
    if (kh < 0) {
        p.dense = a.q_out + (int64_t)t * a.q_out_stride + (int64_t)h * a.head_dim;
        return p;
    }
    if (vh < 0 && a.k_out) p.dense = a.k_out + (int64_t)t * a.k_out_stride + (int64_t)kh * a.head_dim;
    if (a.cache.k) {
        const int slot = a.slots[t];
        const int page = slot / a.cache.page_size;
        if (slot >= 0 && page < a.cache.num_pages) {
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
        const Places<uint16_t> to = places(a, t, h);
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

}  // namespace rope

clove_status_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    const clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    rope::Params p{a, a.q_heads + 2 * a.kv_heads};
    const int64_t tasks = (int64_t)a.T * p.heads;
    const int64_t blocks = std::min<int64_t>(hw::cdiv64(tasks, 4), 64 * dev.num_cus);
    const auto kernel = a.dtype == CLOVE_DTYPE_FP16 ? rope::rope_any<CLOVE_DTYPE_FP16> : rope::rope_any<CLOVE_DTYPE_BF16>;
    CLOVE_LAUNCH(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return check_launch();
}

}  // namespace clove
