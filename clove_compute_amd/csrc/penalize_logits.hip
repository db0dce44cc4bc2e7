// Penalties for repeated tokens, biases and a grammar mask on logits.
//
//   x = logits[v];  seen: x > 0 ? x / r : x * r;  x -= f c + p [c > 0];
//   x += bias[v];  disallowed: -inf                          (fp32 throughout)
//
// A workgroup owns a slice of one row's vocabulary, 16 tokens a thread.  How
// often each token of the slice was produced comes from the row's history,
// counted in LDS (whole numbers: atomics give the same counts in any order), so
// nothing of the vocabulary's size is written to memory but the result.  HBM-bound
// for large batches: 256 rows of 128000 fp32 logits with masks and 8000 tokens of
// history each take 63.5 us (4.3 TB/s), 49 (5.3 TB/s, a copy's rate) without them.
// What is known before the counts -- logits, mask, the first ids -- is loaded
// ahead of them.  Every slice of a row reads its history anew (from L2), so slices
// are as long as leaves two workgroups per CU (at 8192 tokens instead of 16384 the
// above takes 66 us), and results pass the L2 by (68 us with ordinary stores).
#include <algorithm>

#include "decode.hpp"

namespace clove {
namespace logits {

using namespace hw;

constexpr int kPer = 16;  // tokens of a thread, in groups of adjacent ones

// A token's word in LDS.  PACKED: 15 bits of how often it was generated, bit 15
// for "in the prompt", and above them 1 + the last bias entry that names it,
// which holds for histories and lists of fewer than 32768 entries.  Otherwise
// the count has 31 bits under bit 31, and the entry a word of its own.
template <bool PACKED>
constexpr unsigned prompt_bit() { return PACKED ? 0x8000u : 0x80000000u; }

typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Adjacent elements in one 16-byte access at any alignment of their type
template <int DT>
struct Group {
    static constexpr int E = 8;
    u32x4 x;
    __device__ __forceinline__ void load(const uint16_t* p) { x = load_any16(reinterpret_cast<const unsigned char*>(p)); }
    __device__ __forceinline__ float get(int i) const { return Elem<DT>::load((uint16_t)(x[i / 2] >> (16 * (i & 1)))); }
};
template <>
struct Group<CLOVE_DTYPE_FP32> {
    static constexpr int E = 4;
    f32x4 x;
    __device__ __forceinline__ void load(const float* p) { x = *reinterpret_cast<const f32x4u*>(p); }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
};
template <int DT, int E>
__device__ __forceinline__ void store_group(typename Elem<DT>::raw* p, const float (&v)[E]) {
    if constexpr (DT == CLOVE_DTYPE_FP32) {
#pragma unroll
        for (int i = 0; i < E; i += 4)
            __builtin_nontemporal_store(f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]}, reinterpret_cast<f32x4u*>(p + i));
    } else {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (unsigned)Elem<DT>::store(v[2 * i]) | ((unsigned)Elem<DT>::store(v[2 * i + 1]) << 16);
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4u*>(p));
    }
}

template <int DI, int DO, bool PACKED>
__global__ void __launch_bounds__(1024) penalize(const LogitsArgs a, FastDiv slices) {
    using EI = Elem<DI>;
    using EO = Elem<DO>;
    constexpr unsigned kPrompt = prompt_bit<PACKED>(), kCount = kPrompt - 1;
    extern __shared__ __align__(16) unsigned words[];
    const int threads = blockDim.x, tid = threadIdx.x, slice = threads * kPer;
    const int b = slices.div(blockIdx.x), v0 = (blockIdx.x - b * slices.d) * slice;
    const int n = min(slice, a.vocab - v0);
    const typename EI::raw* in = static_cast<const typename EI::raw*>(a.logits) + b * a.logits_stride + v0;
    typename EO::raw* out = static_cast<typename EO::raw*>(a.out) + b * a.out_stride + v0;
    constexpr int E = Group<DI>::E, kGroups = kPer / E;
    Group<DI> x[kGroups];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const int at = (k * threads + tid) * E;
        if (at + E <= n) x[k].load(in + at);
    }
    // what else is known in advance: the mask of the thread's tokens, and the first
    // ids of the history, whatever its length is
    unsigned open[kGroups];
    const uint32_t* allowed = a.allowed ? a.allowed + b * a.allowed_stride : nullptr;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const int at = (k * threads + tid) * E;
        open[k] = allowed && at < n ? allowed[(v0 + at) >> 5] >> ((v0 + at) & 31) : 0xffu;
    }
    const int32_t* told = a.history + b * a.history_stride;
    i32x4 first = {};
    if (a.history && tid * 4 + 4 <= a.history_stride) first = *reinterpret_cast<const i32x4u*>(told + tid * 4);
    unsigned* const entry = words + slice;  // PACKED: not there
    const bool biased = a.bias_ids != nullptr, counted = a.history != nullptr || biased;
    if (counted) {
        u32x4* const w = reinterpret_cast<u32x4*>(words);
        for (int i = tid; i < slice * (PACKED ? 1 : 2) / 4; i += threads) w[i] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
    }
    if (biased) {
        const int m = (int)(a.bias_counts ? min((int64_t)max(a.bias_counts[b], 0), a.bias_stride) : a.bias_stride);
        const int32_t* ids = a.bias_ids + b * a.bias_stride;
        for (int i = tid; i < m; i += threads) {
            const unsigned at = (unsigned)ids[i] - (unsigned)v0;  // (an id below 0 is past every slice)
            if (at < (unsigned)n) PACKED ? atomicMax(&words[at], ((unsigned)i + 1u) << 16) : atomicMax(&entry[at], (unsigned)i + 1u);
        }
        if constexpr (PACKED) __syncthreads();  // the counts go below
    }
    if (a.history) {
        const int len = (int)min((int64_t)max(a.history_lens[b], 0), a.history_stride);
        const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
        auto count = [&](int id, int i) {
            const unsigned at = (unsigned)id - (unsigned)v0;
            if (at < (unsigned)n) i < prompt ? atomicOr(&words[at], kPrompt) : atomicAdd(&words[at], 1u);
        };
        int i = tid * 4;
        for (; i + 4 <= len; i += threads * 4) {
            const i32x4 id = i == tid * 4 ? first : *reinterpret_cast<const i32x4u*>(told + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) count(id[e], i + e);
        }
        for (; i < len; ++i) count(told[i], i);  // (the one thread that the last, shorter four fall to)
    }
    if (counted) __syncthreads();
    const float r = a.repetition ? a.repetition[b] : 1.0f;
    const float f = a.frequency ? a.frequency[b] : 0.0f, p = a.presence ? a.presence[b] : 0.0f;
    const float* bias = a.bias_values + b * a.bias_stride;
    auto result = [&](float l, unsigned word, unsigned e, unsigned open) {
        if constexpr (PACKED) e = word >> 16;
        if (word & (kPrompt | kCount)) {
            const unsigned c = word & kCount;
            if (a.repetition) l = l > 0.0f ? l / r : l * r;
            if (c) l = l - f * (float)c - p;
        }
        if (e) l += bias[e - 1u];
        return open ? l : -__builtin_inff();
    };
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const int at = (k * threads + tid) * E;
        if (at >= n) break;
        u32x4 w[E / 4] = {}, e[E / 4] = {};
        if (counted) {
#pragma unroll
            for (int i = 0; i < E / 4; ++i) {
                w[i] = *reinterpret_cast<const u32x4*>(words + at + 4 * i);
                if (!PACKED && biased) e[i] = *reinterpret_cast<const u32x4*>(entry + at + 4 * i);
            }
        }
        if (at + E <= n) {
            float y[E];
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = result(x[k].get(i), w[i / 4][i % 4], e[i / 4][i % 4], (open[k] >> i) & 1u);
            store_group<DO, E>(out + at, y);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (at + i < n) out[at + i] = EO::store(result(EI::load(in[at + i]), w[i / 4][i % 4], e[i / 4][i % 4], (open[k] >> i) & 1u));
        }
    }
}

typedef void (*Kernel)(const LogitsArgs, FastDiv);
template <int DI>
Kernel pick(int out, bool packed) {
    if (out == CLOVE_DTYPE_FP32)
        return packed ? (Kernel)penalize<DI, CLOVE_DTYPE_FP32, true> : (Kernel)penalize<DI, CLOVE_DTYPE_FP32, false>;
    return packed ? (Kernel)penalize<DI, DI, true> : (Kernel)penalize<DI, DI, false>;
}

}  // namespace logits

clove_status_t launch_penalize_logits(const LogitsArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    const bool counted = a.history || a.bias_ids;
    const bool packed = !(a.history && a.history_stride >= 32768) && !(a.bias_ids && a.bias_stride >= 32768);
    // the longest slices that still give two workgroups per CU
    int threads = packed ? 1024 : 512;
    while (threads > 256 && (int64_t)a.batch * hw::cdiv(a.vocab, threads * logits::kPer) < 2 * dev.num_cus) threads /= 2;
    const int slice = threads * logits::kPer, slices = hw::cdiv(a.vocab, slice);
    if ((int64_t)a.batch * slices > 0x7fffffff) return CLOVE_ERR_INVALID_DIM;
    const logits::Kernel kernel = a.dtype == CLOVE_DTYPE_FP16   ? logits::pick<CLOVE_DTYPE_FP16>(a.out_dtype, packed)
                                  : a.dtype == CLOVE_DTYPE_BF16 ? logits::pick<CLOVE_DTYPE_BF16>(a.out_dtype, packed)
                                                                : logits::pick<CLOVE_DTYPE_FP32>(a.out_dtype, packed);
    const int lds = counted ? slice * (packed ? 4 : 8) : 0;
    if ((st = ensure_lds(reinterpret_cast<const void*>(kernel), lds)) != CLOVE_OK) return st;
    CLOVE_LAUNCH(kernel, dim3((unsigned)(a.batch * slices)), dim3(threads), lds, stream, a, FastDiv(slices));
    return check_launch();
}

}  // namespace clove
