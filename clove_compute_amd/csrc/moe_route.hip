// The router of a sparse MLP block: scores of the experts, the choice by groups
// and of the top_k largest, their weights.
//
//   s = softmax(x) or sigmoid(x),  c = s + bias,  ids = the top_k largest c (x without a bias)
//
// s and c are 64 bits: of some hundred experts two often agree to 2^-24, and
// which of them comes first must not depend on an exponential's last bit.
#include <type_traits>

#include "moe.hpp"

namespace clove {
namespace route {

using namespace hw;

constexpr int WAVES = 4;  // tokens a workgroup
constexpr double NONE = -__builtin_inf();

// Reductions over the wave in the VALU: inside each row of 16 lanes by DPP (row_ror 8
// and 4, quad_perm 2301 and 1032), then across the rows by v_permlane16_swap and
// v_permlane32_swap.  Every lane has the result.
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t u = bitcast<uint64_t>(v);
    const unsigned lo = (unsigned)__builtin_amdgcn_mov_dpp((int)(unsigned)u, CTRL, 0xf, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_mov_dpp((int)(unsigned)(u >> 32), CTRL, 0xf, 0xf, false);
    return bitcast<double>((uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(v), CTRL, 0xf, 0xf, false));
}
template <bool FAR>
__device__ __forceinline__ void swap_rows(float v, float* a, float* b) {
    const unsigned u = bitcast<unsigned>(v);
    const auto s = FAR ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    *a = bitcast<float>(s[0]);
    *b = bitcast<float>(s[1]);
}
template <bool FAR>
__device__ __forceinline__ void swap_rows(double v, double* a, double* b) {
    const uint64_t u = bitcast<uint64_t>(v);
    float l0, l1, h0, h1;
    swap_rows<FAR>(bitcast<float>((unsigned)u), &l0, &l1);
    swap_rows<FAR>(bitcast<float>((unsigned)(u >> 32)), &h0, &h1);
    *a = bitcast<double>((uint64_t)bitcast<unsigned>(h0) << 32 | bitcast<unsigned>(l0));
    *b = bitcast<double>((uint64_t)bitcast<unsigned>(h1) << 32 | bitcast<unsigned>(l1));
}
template <class T, class F>
__device__ __forceinline__ T reduce(T v, F f) {
    v = f(v, dpp<0x128>(v));
    v = f(v, dpp<0x124>(v));
    v = f(v, dpp<0x4e>(v));
    v = f(v, dpp<0xb1>(v));
    T a, b;
    swap_rows<false>(v, &a, &b);
    v = f(a, b);
    swap_rows<true>(v, &a, &b);
    return f(a, b);
}
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }  // (never NaN)
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
template <class T>
__device__ __forceinline__ T wave_most(T v) {
    return reduce(v, [](T a, T b) { return most(a, b); });
}
__device__ __forceinline__ double wave_total(double v) {
    return reduce(v, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    const uint64_t u = bitcast<uint64_t>(v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, lane);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(u >> 32), lane);
    return bitcast<double>((uint64_t)hi << 32 | lo);
}

// The lowest lane of those with the largest value; -1 if that is -infinity.  Doubles by
// their fp32 roundings first, which keep the order: only where several lanes share the
// largest of them are the doubles compared, at more than twice the instructions.
__device__ __forceinline__ int best_lane(float v) {
    const float u = wave_most(v);
    return u > -__builtin_inff() ? __builtin_ctzll(__ballot(v == u)) : -1;
}
__device__ __forceinline__ int best_lane(double v) {
    const float f = (float)v, u = wave_most(f);
    if (!(u > -__builtin_inff())) return -1;
    const uint64_t m = __ballot(f == u);
    if ((m & (m - 1)) == 0) return __builtin_ctzll(m);
    const double w = wave_most(f == u ? v : NONE);
    return __builtin_ctzll(__ballot(f == u && v == w));
}

// Elements [0, n) of `V` adjacent ones at any alignment of their type; -infinity for the others.
template <int DT, int V>
__device__ __forceinline__ void load(float (&v)[V], const typename Elem<DT>::raw* p, int n) {
    using E = Elem<DT>;
    typedef typename E::raw raw;
    struct __attribute__((packed, aligned(sizeof(raw)))) Run {
        raw x[V];
    };
    if (n >= V) {
        const Run r = *reinterpret_cast<const Run*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = E::load(r.x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? E::load(p[i]) : -__builtin_inff();
    }
}

// One token a wave; lane l holds experts l V .. l V + V - 1, so that of equal values
// the lowest lane, and in it the lowest entry, is the lowest index.  C: what the choice
// goes by, the logits themselves (float) or score + bias (double).
//
// A round of the choice is the lanes' own best (kept up to date), one reduction, one
// ballot: some 40 instructions of one wave, which is the time (E = 64, top 6, 16384
// tokens: 16 waves a SIMD of 300 each).
template <int DT, int V, bool BIAS>
__global__ void __launch_bounds__(64 * WAVES) moe_route(const RouteArgs a, const FastDiv group, int t0) {
    typedef typename std::conditional<BIAS, double, float>::type C;
    constexpr C none = -__builtin_inff();
    __shared__ double lds[WAVES][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, N = a.experts, e0 = lane * V;
    const int64_t t = (int64_t)t0 + blockIdx.x * WAVES + wave;
    if (t >= a.T) return;
    const typename Elem<DT>::raw* row = static_cast<const typename Elem<DT>::raw*>(a.logits) + t * a.logits_stride;
    float x[V], bias[V];
    load<DT, V>(x, row + e0, N - e0);
    if constexpr (BIAS) load<CLOVE_DTYPE_FP32, V>(bias, a.bias + e0, N - e0);
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bool here = x[i] > -__builtin_inff();  // (false for NaN)
        if constexpr (BIAS) here = here && bias[i] > -__builtin_inff();
        x[i] = here ? x[i] : -__builtin_inff();
        top = most(top, x[i]);
    }
    const bool softmax = a.score == CLOVE_ROUTE_SOFTMAX;
    double s[V];
    if (softmax) {
        top = wave_most(top);
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = x[i] == top ? 1.0 : x[i] > -__builtin_inff() ? exp((double)x[i] - (double)top) : 0.0;
            if (!(x[i] > -__builtin_inff())) s[i] = 0.0;
            total += s[i];
        }
        const double inv = 1.0 / wave_total(total);  // (infinity if no expert is there: not used then)
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] *= inv;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = 1.0 / (1.0 + exp(-(double)x[i]));
    }
    C c[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (BIAS) c[i] = x[i] > -__builtin_inff() ? s[i] + (double)bias[i] : none;
        else c[i] = x[i];
    }
    if (a.groups > 1) {
        // `per` lanes to a group, a power of two: each the two largest of its share, then
        // the lanes' pairs merged
        const int n = group.d, per = 1 << (31 - __builtin_clz(64 / a.groups)), g = lane / per, sub = lane % per;
#pragma unroll
        for (int i = 0; i < V; ++i) lds[wave][e0 + i] = c[i] > none ? (BIAS ? (double)c[i] : s[i]) : NONE;
        asm volatile("" ::: "memory");  // (one wave's LDS accesses take effect in order)
        double first = NONE, second = NONE;
        if (g < a.groups) {
#pragma unroll 4
            for (int j = sub; j < n; j += per) {
                const double u = lds[wave][g * n + j];
                second = most(second, u > first ? first : u);
                first = most(first, u);
            }
        }
        for (int d = 1; d < per; d <<= 1) {
            const double f = __shfl_xor(first, d), u = __shfl_xor(second, d);
            second = most(most(second, u), f > first ? first : f);
            first = most(first, f);
        }
        // (one lane of each group stands for it)
        double v = sub != 0 || g >= a.groups ? NONE : a.group_top > 1 && second > NONE ? first + second : first;
        uint64_t kept = 0;
        for (int j = 0; j < a.top_groups; ++j) {
            const int l = best_lane(v);
            if (l < 0) break;
            kept |= (uint64_t)1 << (l / per);
            if (lane == l) v = NONE;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!((kept >> group.div(min(e0 + i, N - 1))) & 1)) c[i] = none;
    }
    int id = -1;
    double w = 0.0, sum = 0.0;
    C best = none;
    int at = 0;
    auto update = [&] {
        best = c[0];
        at = 0;
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (c[i] > best) best = c[i], at = i;
    };
    update();
    for (int j = 0; j < a.top_k; ++j) {
        const int l = best_lane(best);
        if (l < 0) break;
        const int i0 = __builtin_amdgcn_readlane(at, l);
        double mine = s[0];
#pragma unroll
        for (int i = 1; i < V; ++i) mine = i0 == i ? s[i] : mine;
        mine = lane_value(mine, l);
        sum += mine;
        if (lane == j) id = l * V + i0, w = mine;
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = lane == l && i0 == i ? none : c[i];
        update();
    }
    if (lane >= a.top_k) return;
    if (a.renormalize && sum > 0.0) w /= sum;
    a.ids[t * a.top_k + lane] = id;
    a.weights[t * a.top_k + lane] = (float)(w * (double)a.scale);
}

namespace {

template <int DT, bool BIAS>
clove_status_t run(const RouteArgs& a, hipStream_t stream) {
    const int v = cdiv(a.experts, 64);
    auto k = v <= 1 ? moe_route<DT, 1, BIAS> : v <= 2 ? moe_route<DT, 2, BIAS> : v <= 4 ? moe_route<DT, 4, BIAS>
             : v <= 8 ? moe_route<DT, 8, BIAS> : moe_route<DT, 16, BIAS>;
    // (a launch counts fewer than 2^32 threads)
    for (int64_t t = 0, most = (int64_t)1 << 25; t < a.T; t += most)
        CLOVE_LAUNCH(k, dim3((unsigned)cdiv64(min(most, a.T - t), WAVES)), dim3(64 * WAVES), 0, stream, a,
                     FastDiv(a.experts / a.groups), (int)t);
    return check_launch();
}
template <int DT>
clove_status_t run(const RouteArgs& a, hipStream_t stream) {
    return a.bias ? run<DT, true>(a, stream) : run<DT, false>(a, stream);
}

}  // namespace
}  // namespace route

clove_status_t launch_moe_route(const RouteArgs& a, hipStream_t stream) {
    using namespace route;
    DeviceInfo dev;
    if (const clove_status_t st = current_device_info(&dev); st != CLOVE_OK) return st;
    if (a.dtype == CLOVE_DTYPE_FP16) return run<CLOVE_DTYPE_FP16>(a, stream);
    if (a.dtype == CLOVE_DTYPE_BF16) return run<CLOVE_DTYPE_BF16>(a, stream);
    return run<CLOVE_DTYPE_FP32>(a, stream);
}

}  // namespace clove
