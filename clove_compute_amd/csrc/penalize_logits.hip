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
// history each take 53 us (5.1 TB/s), 48 (5.5 TB/s, a copy's rate) without them;
// bf16 logits to fp32 without a history 31 (6.3 TB/s).  What is known before the
// counts -- logits, mask, the first ids -- is loaded ahead of them, and results
// pass the L2 by.  Every slice of a row reads its history anew; a row's slices run
// on one XCD, whose L2 then has it (39 us with bf16 logits, masks and biases to
// fp32, 43 where they are spread over all XCDs; fp32 without masks 52 and 54).
#include <algorithm>

#include "decode.hpp"

namespace clove {
namespace logits {

using namespace hw;

constexpr int kPer = 16;  // tokens of a thread, in groups of adjacent ones
// loads of ids at once (32 x 32000 after 8191 tokens 9.9 us with one, 9.3 with two;
// 256 x 128000 after 8000 54 and 52; four win no more)
constexpr int kAhead = 2;

// A token's word in LDS.  PACKED: 15 bits of how often it was generated, bit 15
// for "in the prompt", and above them 1 + the last bias entry that names it,
// which holds for histories and lists of fewer than 32768 entries.  Otherwise
// the count has 31 bits under bit 31, and the entry a word of its own.
template <bool PACKED>
constexpr unsigned prompt_bit() { return PACKED ? 0x8000u : 0x80000000u; }

typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// E adjacent elements in one access, at any alignment of their type
template <int DT, int E>
struct Group {
    typedef unsigned any __attribute__((ext_vector_type(E / 2), aligned(2)));
    any x;
    __device__ __forceinline__ void load(const uint16_t* p) { x = *reinterpret_cast<const any*>(p); }
    __device__ __forceinline__ float get(int i) const { return Elem<DT>::load((uint16_t)(x[i / 2] >> (16 * (i & 1)))); }
};
template <int E>
struct Group<CLOVE_DTYPE_FP32, E> {
    f32x4 x;
    __device__ __forceinline__ void load(const float* p) { x = *reinterpret_cast<const f32x4u*>(p); }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
};
template <int DT, int E>
__device__ __forceinline__ void store_group(typename Elem<DT>::raw* p, const float (&v)[E]) {
    if constexpr (DT == CLOVE_DTYPE_FP32) {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4u*>(p));
    } else {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (unsigned)Elem<DT>::store(v[2 * i]) | ((unsigned)Elem<DT>::store(v[2 * i + 1]) << 16);
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4u*>(p));
    }
}

template <int DI, int DO, bool PACKED>
__global__ void __launch_bounds__(512) penalize(const LogitsArgs a, FastDiv slices, int apart) {
    using EI = Elem<DI>;
    using EO = Elem<DO>;
    constexpr unsigned kPrompt = prompt_bit<PACKED>(), kCount = kPrompt - 1;
    extern __shared__ __align__(16) unsigned words[];
    const int threads = blockDim.x, tid = threadIdx.x, slice = threads * kPer;
    // the slices of a row lie `apart` (8) workgroups apart: on one XCD, whose L2 has
    // its history after the first of them
    const int run = slices.div(blockIdx.x / apart), b = run * apart + blockIdx.x % apart, v0 = (blockIdx.x / apart - run * slices.d) * slice;
    if (b >= a.batch) return;
    const int n = min(slice, a.vocab - v0);
    const typename EI::raw* in = static_cast<const typename EI::raw*>(a.logits) + b * a.logits_stride + v0;
    typename EO::raw* out = static_cast<typename EO::raw*>(a.out) + b * a.out_stride + v0;
    // so many that a result is 16 bytes: a wave's store is whole lines (with 8 of
    // bf16 in two stores of fp32, 256 x 128000 without a history take 49 us, not 31)
    constexpr int E = DO == CLOVE_DTYPE_FP32 ? 4 : 8, kGroups = kPer / E;
    Group<DI, E> x[kGroups];
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
        open[k] = allowed && at < n ? allowed[(v0 + at) >> 5] : 0xffffffffu;  // (shifted below: here it would be awaited)
    }
    const int32_t* told = a.history + b * a.history_stride;
    i32x4 first = {};
    if (a.history && tid * 4 + 4 <= a.history_stride) first = *reinterpret_cast<const i32x4u*>(told + tid * 4);
    const bool biased = a.bias_ids != nullptr, counted = a.history != nullptr || biased;
    const int32_t* named = a.bias_ids + b * a.bias_stride;
    int id[kAhead] = {};
    if (biased && tid < a.bias_stride) id[0] = named[tid];
    const int len = a.history ? (int)min((int64_t)max(a.history_lens[b], 0), a.history_stride) : 0;
    const int prompt = a.history && a.prompt_lens ? a.prompt_lens[b] : 0;
    const int entries = !biased ? 0 : (int)(a.bias_counts ? min((int64_t)max(a.bias_counts[b], 0), a.bias_stride) : a.bias_stride);
    const float r = a.repetition ? a.repetition[b] : 1.0f;
    const float f = a.frequency ? a.frequency[b] : 0.0f, p = a.presence ? a.presence[b] : 0.0f;
    unsigned* const entry = words + slice;  // PACKED: not there
    if (counted) {
        u32x4* const w = reinterpret_cast<u32x4*>(words);
        for (int i = tid; i < slice * (PACKED ? 1 : 2) / 4; i += threads) w[i] = u32x4{0u, 0u, 0u, 0u};
    }
    // the ids that follow the first ones, kAhead loads at a time, and the history's
    // last one to three (the thread's is looked at behind its others)
    // (unsigned: steps past the longest length, 2^31 - 1, do not turn negative)
    const unsigned whole = len & ~3, step = 4 * threads;
    const int last = tid < len - (int)whole ? told[whole + tid] : -1;
    i32x4 ids[kAhead];
    ids[0] = first;
    auto load = [&](unsigned i0, int u0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u >= u0 && i0 + u * step < whole) ids[u] = *reinterpret_cast<const i32x4u*>(told + i0 + u * step);
    };
    load(4 * tid, 1);
    if (counted) __syncthreads();
    if (biased) {
        for (unsigned i0 = tid; i0 < (unsigned)entries; i0 += kAhead * threads) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if ((u > 0 || i0 > (unsigned)tid) && i0 + u * threads < (unsigned)entries) id[u] = named[i0 + u * threads];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const unsigned i = i0 + u * threads;
                const unsigned at = (unsigned)id[u] - (unsigned)v0;  // (an id below 0 is past every slice)
                if (i < (unsigned)entries && at < (unsigned)n) PACKED ? atomicMax(&words[at], (i + 1u) << 16) : atomicMax(&entry[at], i + 1u);
            }
        }
        if constexpr (PACKED) __syncthreads();  // the counts go below
    }
    auto count = [&](int id, int i) {
        const unsigned at = (unsigned)id - (unsigned)v0;
        if (at < (unsigned)n) i < prompt ? atomicOr(&words[at], kPrompt) : atomicAdd(&words[at], 1u);
    };
    for (unsigned i0 = 4 * tid; i0 < whole; i0 += kAhead * step) {
        if (i0 > 4u * tid) load(i0, 0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u * step < whole) {
#pragma unroll
                for (int e = 0; e < 4; ++e) count(ids[u][e], (int)(i0 + u * step) + e);
            }
        }
    }
    if (tid < len - (int)whole) count(last, (int)whole + tid);
    if (counted) __syncthreads();
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
        const unsigned bits = open[k] >> ((v0 + at) & 31);
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
            for (int i = 0; i < E; ++i) y[i] = result(x[k].get(i), w[i / 4][i % 4], e[i / 4][i % 4], (bits >> i) & 1u);
            store_group<DO, E>(out + at, y);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (at + i < n) out[at + i] = EO::store(result(EI::load(in[at + i]), w[i / 4][i % 4], e[i / 4][i % 4], (bits >> i) & 1u));
        }
    }
}

typedef void (*Kernel)(const LogitsArgs, FastDiv, int);
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
    // Counting, slices of 8192 tokens: each reads the row's history, but more of them
    // fill the CUs better (256 x 128000 and 64 x 152064 after 8000 and 4000 tokens: 53
    // and 16 us, with 16384 52 and 18, with 4096 57 and 17.5).  Otherwise, and with
    // fewer than two workgroups per CU, of 4096 (256 x 128000 47.6 and 49 us).
    int threads = counted ? 512 : 256;
    if ((int64_t)a.batch * hw::cdiv(a.vocab, threads * logits::kPer) < 2 * dev.num_cus) threads = 256;
    const int slice = threads * logits::kPer, slices = hw::cdiv(a.vocab, slice);
    const int apart = a.batch >= 8 ? 8 : 1;
    const int64_t grid = (int64_t)hw::cdiv(a.batch, apart) * apart * slices;
    if (grid > 0x7fffffff) return CLOVE_ERR_INVALID_DIM;
    const logits::Kernel kernel = a.dtype == CLOVE_DTYPE_FP16   ? logits::pick<CLOVE_DTYPE_FP16>(a.out_dtype, packed)
                                  : a.dtype == CLOVE_DTYPE_BF16 ? logits::pick<CLOVE_DTYPE_BF16>(a.out_dtype, packed)
                                                                : logits::pick<CLOVE_DTYPE_FP32>(a.out_dtype, packed);
    const int lds = counted ? slice * (packed ? 4 : 8) : 0;
    if ((st = ensure_lds(reinterpret_cast<const void*>(kernel), lds)) != CLOVE_OK) return st;
    CLOVE_LAUNCH(kernel, dim3((unsigned)grid), dim3(threads), lds, stream, a, FastDiv(slices), apart);
    return check_launch();
}

}  // namespace clove
