// The norms before and after a block of a decoder with the residual between
// them, a row at a time:
//
//   u = x rsqrt(mean(x^2) + eps) w_post,  y = r + s g u,  h = y rsqrt(mean(y^2) + eps) w_pre
//
// A row stays in registers from its loads to its stores (every element is read
// and written once, in fp32 between), so an output may be its input: what is
// left is HBM for many tokens (8192 rows of 4096, fp16 with an fp32 stream, both
// norms and a gate, 470 MB: 79 to 83 us, 5.7 to 5.9 TB/s, where a copy reaches
// 5.1), and for one (a row of 2048: 2.4 us) a launch and two round trips.
#include <algorithm>

#include "moe.hpp"

namespace clove {
namespace norm {

using namespace hw;

constexpr int CH = 8;  // elements of a chunk: 16 bytes of 16-bit elements

// Elements [0, n) of a chunk at any alignment of its element type; the others 0.
template <int DT>
__device__ __forceinline__ void load(float (&v)[CH], const void* base, int64_t at, int n) {
    using E = Elem<DT>;
    const typename E::raw* p = static_cast<const typename E::raw*>(base) + at;
    if (n >= CH) {
        if constexpr (sizeof(typename E::raw) == 2) {
            const u32x4 w = *reinterpret_cast<const u32x4u*>(p);
#pragma unroll
            for (int i = 0; i < CH; ++i) v[i] = E::load((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4u*>(p), b = *reinterpret_cast<const u32x4u*>(p + 4);
#pragma unroll
            for (int i = 0; i < CH; ++i) v[i] = bitcast<float>(i < 4 ? a[i & 3] : b[i & 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < CH; ++i) v[i] = i < n ? E::load(p[i]) : 0.0f;
    }
}

template <int DT>
__device__ __forceinline__ void store(const float (&v)[CH], void* base, int64_t at, int n) {
    using E = Elem<DT>;
    typename E::raw* p = static_cast<typename E::raw*>(base) + at;
    if (n >= CH) {
        if constexpr (sizeof(typename E::raw) == 2) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (unsigned)E::store(v[2 * i]) | ((unsigned)E::store(v[2 * i + 1]) << 16);
            *reinterpret_cast<u32x4u*>(p) = w;
        } else {
            *reinterpret_cast<u32x4u*>(p) =
                u32x4{bitcast<unsigned>(v[0]), bitcast<unsigned>(v[1]), bitcast<unsigned>(v[2]), bitcast<unsigned>(v[3])};
            *reinterpret_cast<u32x4u*>(p + 4) =
                u32x4{bitcast<unsigned>(v[4]), bitcast<unsigned>(v[5]), bitcast<unsigned>(v[6]), bitcast<unsigned>(v[7])};
        }
    } else {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i < n) p[i] = E::store(v[i]);
    }
}

// The sum over the workgroup in a fixed order: each wave's, then the waves' in turn.
__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    lds_barrier();
    float s = lds[0];
    for (int w = 1; w < waves; ++w) s += lds[w];
    return s;
}

// 1 / sqrt(mean(y^2) + eps) for the row whose chunks the threads hold.  Squares past fp32, and a
// mean so small that fp32 lost part of them (below 2^-100, so with such an eps only), are taken
// of y 2^-80 or y 2^88 instead, which y becomes: the result fits what it became.  That is a
// branch of the whole workgroup (every thread has the same sum) that no usual row takes.
template <int CPT>
__device__ __forceinline__ float inverse_rms(float (&y)[CPT][CH], int D, float eps, float (*lds)[16]) {
    auto mean = [&](float* to) {
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
            for (int i = 0; i < CH; ++i) sum = fmaf(y[c][i], y[c][i], sum);
        return block_sum(sum, to) / (float)D;
    };
    float m = mean(lds[0]) + eps;
    if (__builtin_amdgcn_readfirstlane((m >= 0.0f && m < 0x1p-100f) || m == __builtin_inff())) {
        const float f = m < 1.0f ? 0x1p88f : 0x1p-80f;
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] *= f;
        m = mean(lds[1]) + eps * f * f;
    }
    return 1.0f / sqrtf(m);
}

// One row a workgroup, CPT chunks a thread (chunk c of the row: thread c % threads): as
// few as 1024 threads allow, so that a row's loads are all in flight at once and its sums
// are short.  A workgroup of its own per row, not a loop over rows: 8192 rows keep HBM busy
// by the workgroups that wait beside each other on a CU (four of 512 threads).
template <int DT, int RT, int CPT>
__global__ void __launch_bounds__(1024) block_norm(const BlockNormArgs a, int64_t t0) {
    __shared__ float lds[4][16];
    const int tid = threadIdx.x, NT = blockDim.x, D = a.D;
    const int64_t t = t0 + blockIdx.x;
    float y[CPT][CH];
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int d = (c * NT + tid) * CH;
        if (a.x) load<DT>(y[c], a.x, t * a.x_stride + d, D - d);
        else
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] = 0.0f;
    }
    float r = 1.0f;
    if (a.post_weight) r = inverse_rms(y, D, a.eps, lds);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int d = (c * NT + tid) * CH;
        float w[CH];
        if (a.post_weight) {
            load<DT>(w, a.post_weight, d, D - d);
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] = y[c][i] * r * w[i];
        }
        if (a.gate) {
            load<DT>(w, a.gate, t * a.gate_stride + d, D - d);
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] *= w[i];
        }
        if (a.residual) {
            load<RT>(w, a.residual, t * a.residual_stride + d, D - d);
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] = a.x ? fmaf(a.scale, y[c][i], w[i]) : w[i];
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] *= a.scale;
        }
        // (past the row's end: 0 again, whatever an infinite factor made of it)
        if (D - d < CH) {
#pragma unroll
            for (int i = 0; i < CH; ++i) y[c][i] = d + i < D ? y[c][i] : 0.0f;
        }
        if (a.y_out) store<RT>(y[c], a.y_out, t * a.y_out_stride + d, D - d);
    }
    if (!a.h_out) return;
    r = inverse_rms(y, D, a.eps, lds + 2);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int d = (c * NT + tid) * CH;
        float w[CH];
        if (a.pre_weight) {
            load<DT>(w, a.pre_weight, d, D - d);
#pragma unroll
            for (int i = 0; i < CH; ++i) w[i] = y[c][i] * r * w[i];
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i) w[i] = y[c][i] * r;
        }
        store<DT>(w, a.h_out, t * a.h_out_stride + d, D - d);
    }
}

namespace {

template <int DT, int RT>
clove_status_t run(const BlockNormArgs& a, hipStream_t stream) {
    const int chunks = cdiv(a.D, CH);
    const int cpt = cdiv(chunks, 1024) <= 1 ? 1 : cdiv(chunks, 1024) <= 2 ? 2 : 4;
    const int nt = 64 * cdiv(chunks, 64 * cpt);
    auto k = cpt == 1 ? block_norm<DT, RT, 1> : cpt == 2 ? block_norm<DT, RT, 2> : block_norm<DT, RT, 4>;
    // (a launch counts fewer than 2^32 threads)
    for (int64_t t = 0, most = ((int64_t)1 << 31) / nt; t < a.T; t += most)
        CLOVE_LAUNCH(k, dim3((unsigned)std::min(most, a.T - t)), dim3((unsigned)nt), 0, stream, a, t);
    return check_launch();
}

}  // namespace
}  // namespace norm

clove_status_t launch_block_norm(const BlockNormArgs& a, hipStream_t stream) {
    using namespace norm;
    DeviceInfo dev;
    if (const clove_status_t st = current_device_info(&dev); st != CLOVE_OK) return st;
    const bool wide = a.residual_dtype == CLOVE_DTYPE_FP32;
    if (a.dtype == CLOVE_DTYPE_FP16)
        return wide ? run<CLOVE_DTYPE_FP16, CLOVE_DTYPE_FP32>(a, stream) : run<CLOVE_DTYPE_FP16, CLOVE_DTYPE_FP16>(a, stream);
    return wide ? run<CLOVE_DTYPE_BF16, CLOVE_DTYPE_FP32>(a, stream) : run<CLOVE_DTYPE_BF16, CLOVE_DTYPE_BF16>(a, stream);
}

}  // namespace clove
