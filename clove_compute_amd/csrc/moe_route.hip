// The router of a sparse MLP block: scores of the experts, the choice by groups
// and of the top_k largest, their weights.
//
//   s = softmax(x) or sigmoid(x),  c = s + bias,  ids = the top_k largest c (x without a bias)
//
// s and c are 64 bits: of some hundred experts two often agree to 2^-24, and
// which of them comes first must not depend on an exponential's last bit.
#include <algorithm>
#include <cfloat>
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
// over each L = 16, 32 or 64 lanes
template <int L, class T, class F>
__device__ __forceinline__ T reduce(T v, F f) {
    v = f(v, dpp<0x128>(v));
    v = f(v, dpp<0x124>(v));
    v = f(v, dpp<0x4e>(v));
    v = f(v, dpp<0xb1>(v));
    T a, b;
    if constexpr (L >= 32) {
        swap_rows<false>(v, &a, &b);
        v = f(a, b);
    }
    if constexpr (L == 64) {
        swap_rows<true>(v, &a, &b);
        v = f(a, b);
    }
    return v;
}
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }  // (never NaN)
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
template <int L, class T>
__device__ __forceinline__ T lanes_most(T v) {
    return reduce<L>(v, [](T a, T b) { return most(a, b); });
}

// The bits of this lane's L lanes
template <int L>
__device__ __forceinline__ uint64_t own_lanes(uint64_t m) {
    if constexpr (L == 64) return m;
    return (m >> (threadIdx.x & 63 & ~(L - 1))) & (((uint64_t)1 << L) - 1);
}

// Of each L lanes the lowest with the largest value, -1 if that is -infinity.  Doubles by
// their fp32 roundings first, which keep the order: only where several lanes share the
// largest of them are the doubles compared, at more than twice the instructions.
template <int L>
__device__ __forceinline__ int best_lane(float v) {
    const float u = lanes_most<L>(v);
    return u > -__builtin_inff() ? __builtin_ctzll(own_lanes<L>(__ballot(v == u))) : -1;
}
template <int L>
__device__ __forceinline__ int best_lane(double v, float f) {
    const float u = lanes_most<L>(f);
    uint64_t m = own_lanes<L>(__ballot(f == u));
    if (__any((m & (m - 1)) != 0 && u > -__builtin_inff())) {
        const double w = lanes_most<L>(f == u ? v : NONE);
        m = own_lanes<L>(__ballot(f == u && v == w));
    }
    return u > -__builtin_inff() ? __builtin_ctzll(m) : -1;
}
template <int L>
__device__ __forceinline__ int best_lane(double v) {
    return best_lane<L>(v, (float)v);
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

// L lanes a token; its lane l holds experts l V .. l V + V - 1, so that of equal values
// the lowest lane, and in it the lowest entry, is the lowest index.  C: what the choice
// goes by, the logits themselves (float) or score + bias (double).
//
// A round of the choice is one reduction, one ballot, and the chosen lane's next best:
// some 30 instructions for all tokens of a wave, which is the time (E = 64, top 6, 16384
// tokens: 7.7 us with two tokens a wave, 12.0 with one, 27 with reductions through LDS;
// the 2.9 MB that it reads and writes take 0.6).  One token of 128 experts, top 8: 3.8 us, a
// launch, one load, eight rounds.
template <int DT, int V, int L, bool BIAS>
__global__ void __launch_bounds__(64 * WAVES) moe_route(const RouteArgs a, const FastDiv group, int t0) {
    typedef typename std::conditional<BIAS, double, float>::type C;
    constexpr C none = -__builtin_inff();
    __shared__ double values[WAVES][64 * V];  // of the groups' experts, then the chosen ones' scores
    __shared__ int chosen[WAVES][64 * V];
    const int lane = threadIdx.x & 63, l = lane % L, wave = threadIdx.x >> 6, N = a.experts, e0 = l * V;
    const int64_t t = (int64_t)t0 + (blockIdx.x * WAVES + wave) * (64 / L) + lane / L;
    const int64_t row = t < a.T ? t : a.T - 1;  // (past the last token: its row again, stored nowhere)
    double* mine = values[wave] + (lane - l) * V;  // this token's L V
    int* picks = chosen[wave] + (lane - l) * V;
    float x[V], bias[V];
    load<DT, V>(x, static_cast<const typename Elem<DT>::raw*>(a.logits) + row * a.logits_stride + e0, N - e0);
    if constexpr (BIAS) load<CLOVE_DTYPE_FP32, V>(bias, a.bias + e0, N - e0);
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bool here = x[i] > -__builtin_inff();  // (false for NaN)
        if constexpr (BIAS) here = here && bias[i] > -__builtin_inff();
        x[i] = here ? x[i] : -__builtin_inff();
        top = most(top, x[i]);
    }
    double s[V];
    if (a.score == CLOVE_ROUTE_SOFTMAX) {
        top = lanes_most<L>(top);
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = !(x[i] > -__builtin_inff()) ? 0.0 : x[i] == top ? 1.0 : exp((double)x[i] - (double)top);
            total += s[i];
        }
        total = reduce<L>(total, [](double u, double v) { return u + v; });
        const double inv = 1.0 / total;  // (infinity if no expert is there: not used then)
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
        const int n = group.d, per = 1 << (31 - __builtin_clz(L / a.groups)), g = l / per, sub = l % per;
#pragma unroll
        for (int i = 0; i < V; ++i) mine[e0 + i] = c[i] > none ? (BIAS ? (double)c[i] : s[i]) : NONE;
        asm volatile("" ::: "memory");  // (one wave's LDS accesses take effect in order)
        double first = NONE, second = NONE;
        if (g < a.groups) {
#pragma unroll 4
            for (int j = sub; j < n; j += per) {
                const double u = mine[g * n + j];
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
            // (two biases of fp32's lowest value add up to less than it: still more than none)
            const int at = best_lane<L>(v, v > NONE ? fmaxf((float)v, -FLT_MAX) : -__builtin_inff());
            if (at >= 0) kept |= (uint64_t)1 << (at / per);
            if (l == at) v = NONE;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!((kept >> group.div(min(e0 + i, N - 1))) & 1)) c[i] = none;
        asm volatile("" ::: "memory");
    }
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
    int found = 0;
    for (int j = 0; j < a.top_k; ++j) {
        const int won = best_lane<L>(best);
        if (!__any(won >= 0)) break;
        found += won >= 0;
        if (l == won) {
            double score = s[0];
#pragma unroll
            for (int i = 1; i < V; ++i) score = at == i ? s[i] : score;
            mine[j] = score;
            picks[j] = e0 + at;
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = at == i ? none : c[i];
            update();
        }
    }
    asm volatile("" ::: "memory");
    double sum = 0.0;
    if (a.renormalize)
        for (int j = 0; j < found; ++j) sum += mine[j];
    if (t >= a.T) return;
    for (int j = l; j < a.top_k; j += L) {
        double w = j < found ? mine[j] : 0.0;
        if (sum > 0.0) w /= sum;
        a.ids[t * a.top_k + j] = j < found ? picks[j] : -1;
        a.weights[t * a.top_k + j] = (float)(w * (double)a.scale);
    }
}

namespace {

template <int DT, int V, int L, bool BIAS>
clove_status_t launch(const RouteArgs& a, hipStream_t stream) {
    constexpr int TOKENS = WAVES * (64 / L);  // of a workgroup
    // (a launch counts fewer than 2^32 threads)
    for (int64_t t = 0, most = (int64_t)1 << 25; t < a.T; t += most)
        CLOVE_LAUNCH((moe_route<DT, V, L, BIAS>), dim3((unsigned)cdiv64(std::min(most, a.T - t), TOKENS)), dim3(64 * WAVES), 0, stream, a,
                     FastDiv(a.experts / a.groups), (int)t);
    return check_launch();
}

// Lanes a token: 16 for up to 32 experts, 32 for up to 128 (where there are as many as
// groups), else 64
template <int DT, bool BIAS>
clove_status_t run(const RouteArgs& a, hipStream_t stream) {
    const int n = a.experts;
    if (n <= 16) return launch<DT, 1, 16, BIAS>(a, stream);
    if (n <= 32 && a.groups <= 16) return launch<DT, 2, 16, BIAS>(a, stream);
    if (n <= 64 && a.groups <= 32) return launch<DT, 2, 32, BIAS>(a, stream);
    if (n <= 128 && a.groups <= 32) return launch<DT, 4, 32, BIAS>(a, stream);
    if (n <= 128) return launch<DT, 2, 64, BIAS>(a, stream);
    if (n <= 256) return launch<DT, 4, 64, BIAS>(a, stream);
    if (n <= 512) return launch<DT, 8, 64, BIAS>(a, stream);
    return launch<DT, 16, 64, BIAS>(a, stream);
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
