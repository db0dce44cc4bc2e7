// The router of a sparse MLP block: scores of the experts, the choice by groups
// and of the top_k largest, their weights.
//
//   s = softmax(x) or sigmoid(x),  c = s + bias,  ids = the top_k largest c (x without a bias)
//
// s and c are 64 bits: of some hundred experts two often agree to 2^-24, and
// which of them comes first must not depend on an exponential's last bit.
#include "moe.hpp"

namespace clove {
namespace route {

using namespace hw;

constexpr int WAVES = 4;      // tokens a workgroup
constexpr double NONE = -__builtin_inf();

// The larger value, of equal ones the lower index, over the wave.
__device__ __forceinline__ void wave_best(double& v, int& at) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const double u = __shfl_xor(v, d);
        const int b = __shfl_xor(at, d);
        if (u > v || (u == v && b < at)) {
            v = u;
            at = b;
        }
    }
}

// One token a wave; lane l holds experts l + 64 i, i < VPL.
template <int DT, int VPL>
__global__ void __launch_bounds__(64 * WAVES) moe_route(const RouteArgs a) {
    using E = Elem<DT>;
    __shared__ double lds[WAVES][64 * VPL];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * WAVES + wave, N = a.experts;
    if (t >= a.T) return;
    const typename E::raw* x = static_cast<const typename E::raw*>(a.logits) + (int64_t)t * a.logits_stride;
    double s[VPL], c[VPL];  // scores; what the choice goes by, NONE: not available
    double most = NONE;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 64 * i;
        const float f = e < N ? E::load(x[e]) : -__builtin_inff();
        const float b = a.bias && e < N ? a.bias[e] : 0.0f;
        const bool here = f > -__builtin_inff() && b > -__builtin_inff();  // (false for NaN)
        s[i] = here ? (double)f : NONE;
        c[i] = (double)b;
        most = s[i] > most ? s[i] : most;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const double u = __shfl_xor(most, d);
        most = u > most ? u : most;
    }
    double total = 0.0;
    const bool every_x = a.score == CLOVE_ROUTE_SOFTMAX;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const double f = s[i];
        const bool here = f > NONE;
        if (every_x) s[i] = !here ? 0.0 : f == most ? 1.0 : exp(f - most);
        else s[i] = here ? 1.0 / (1.0 + exp(-f)) : 0.0;
        total += s[i];
        c[i] = here ? (a.bias ? 0.0 : f) + c[i] : NONE;  // (the score joins a bias below)
    }
    if (every_x) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
#pragma unroll
        for (int i = 0; i < VPL; ++i) s[i] = total > 0.0 ? s[i] / total : 0.0;
    }
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] = c[i] > NONE ? s[i] + c[i] : NONE;
    }
    if (a.groups > 1) {
        // lane g: the value of group g
        const int n = N / a.groups;
#pragma unroll
        for (int i = 0; i < VPL; ++i) lds[wave][lane + 64 * i] = c[i] > NONE ? (a.bias ? c[i] : s[i]) : NONE;
        asm volatile("" ::: "memory");  // (one wave's LDS accesses take effect in order)
        double v = NONE;
        if (lane < a.groups) {
            double first = NONE, second = NONE;
            for (int j = 0; j < n; ++j) {
                const double u = lds[wave][lane * n + j];
                if (u > first) second = first, first = u;
                else if (u > second) second = u;
            }
            v = a.group_top > 1 && second > NONE ? first + second : first;
        }
        uint64_t kept = 0;
        for (int j = 0; j < a.top_groups; ++j) {
            double u = v;
            int g = lane;
            wave_best(u, g);
            if (!(u > NONE)) break;
            kept |= (uint64_t)1 << g;
            if (lane == g) v = NONE;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane + 64 * i;
            if (e < N && !((kept >> (e / n)) & 1)) c[i] = NONE;
        }
    }
    int id = -1;
    double w = 0.0, sum = 0.0;
    for (int j = 0; j < a.top_k; ++j) {
        double v = NONE, mine = 0.0;
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (c[i] > v) v = c[i], at = lane + 64 * i, mine = s[i];
        wave_best(v, at);
        if (!(v > NONE)) break;
        mine = __shfl(mine, at & 63);
        sum += mine;
        if (lane == j) id = at, w = mine;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (at == lane + 64 * i) c[i] = NONE;
    }
    if (lane >= a.top_k) return;
    if (a.renormalize && sum > 0.0) w /= sum;
    a.ids[(int64_t)t * a.top_k + lane] = id;
    a.weights[(int64_t)t * a.top_k + lane] = (float)(w * (double)a.scale);
}

namespace {

template <int DT>
clove_status_t run(const RouteArgs& a, hipStream_t stream) {
    const int v = cdiv(a.experts, 64);
    auto k = v <= 1 ? moe_route<DT, 1> : v <= 2 ? moe_route<DT, 2> : v <= 4 ? moe_route<DT, 4> : v <= 8 ? moe_route<DT, 8> : moe_route<DT, 16>;
    CLOVE_LAUNCH(k, dim3((unsigned)cdiv(a.T, WAVES)), dim3(64 * WAVES), 0, stream, a);
    return check_launch();
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
