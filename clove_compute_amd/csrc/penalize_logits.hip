// Penalties for repeated tokens, biases and a grammar mask on logits.
//
//   x = logits[v];  seen: x > 0 ? x / r : x * r;  x -= f c + p [c > 0];
//   x += bias[v];  disallowed: -inf                          (fp32 throughout)
//
// A workgroup owns a slice of one row's vocabulary.  How often each token of
// the slice was produced comes from the row's history, counted in LDS (whole
// numbers: atomics give the same counts in any order), so nothing of the
// vocabulary's size is written to memory but the result.
#include <algorithm>

#include "decode.hpp"

namespace clove {
namespace logits {

using namespace hw;

constexpr int kThreads = 256;

// LDS words of a token: count of the generated part, with the top bit for "in
// the history at all"; and, with biases, 1 + the last list entry that names it.
constexpr unsigned kSeen = 0x80000000u;

template <int DI, int DO>
__global__ void __launch_bounds__(kThreads) penalize(const LogitsArgs a, int slice, int slices) {
    using EI = Elem<DI>;
    using EO = Elem<DO>;
    extern __shared__ unsigned lds[];
    const int b = blockIdx.x / slices, v0 = (blockIdx.x - b * slices) * slice;
    const int n = min(slice, a.vocab - v0);
    unsigned* const count = lds;
    unsigned* const last = lds + slice;
    const bool biased = a.bias_ids != nullptr;
    const int words = biased ? 2 * slice : slice;
    for (int i = threadIdx.x; i < words; i += kThreads) lds[i] = 0u;
    __syncthreads();
    if (a.history) {
        const int len = (int)min((int64_t)max(a.history_lens[b], 0), a.history_stride);
        const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
        const int32_t* ids = a.history + b * a.history_stride;
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const unsigned at = (unsigned)ids[i] - (unsigned)v0;
            if (at < (unsigned)n && ids[i] >= 0) {
                atomicOr(&count[at], kSeen);
                if (i >= prompt) atomicAdd(&count[at], 1u);
            }
        }
    }
    if (biased) {
        const int m = (int)(a.bias_counts ? min((int64_t)max(a.bias_counts[b], 0), a.bias_stride) : a.bias_stride);
        const int32_t* ids = a.bias_ids + b * a.bias_stride;
        for (int i = threadIdx.x; i < m; i += kThreads) {
            const unsigned at = (unsigned)ids[i] - (unsigned)v0;
            if (at < (unsigned)n && ids[i] >= 0) atomicMax(&last[at], (unsigned)i + 1u);
        }
    }
    __syncthreads();
    const float r = a.repetition ? a.repetition[b] : 1.0f;
    const float f = a.frequency ? a.frequency[b] : 0.0f, p = a.presence ? a.presence[b] : 0.0f;
    const typename EI::raw* in = static_cast<const typename EI::raw*>(a.logits) + b * a.logits_stride + v0;
    typename EO::raw* out = static_cast<typename EO::raw*>(a.out) + b * a.out_stride + v0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        float x = EI::load(in[i]);
        const unsigned seen = count[i], c = seen & ~kSeen;
        if (seen) {
            if (a.repetition) x = x > 0.0f ? x / r : x * r;
            if (c) x = x - f * (float)c - p;
        }
        if (biased && last[i]) x += a.bias_values[b * a.bias_stride + (last[i] - 1u)];
        if (a.allowed && !((a.allowed[b * a.allowed_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31)) & 1u))
            x = -__builtin_inff();
        out[i] = EO::store(x);
    }
}

typedef void (*Kernel)(const LogitsArgs, int, int);
template <int DI>
Kernel pick(int out) {
    return out == CLOVE_DTYPE_FP32 ? (Kernel)penalize<DI, CLOVE_DTYPE_FP32> : (Kernel)penalize<DI, DI>;
}

}  // namespace logits

clove_status_t launch_penalize_logits(const LogitsArgs& a, hipStream_t stream) {
    const int slice = 4096;
    const int slices = hw::cdiv(a.vocab, slice);
    if ((int64_t)a.batch * slices > 0x7fffffff) return CLOVE_ERR_INVALID_DIM;
    const logits::Kernel kernel = a.dtype == CLOVE_DTYPE_FP16   ? logits::pick<CLOVE_DTYPE_FP16>(a.out_dtype)
                                  : a.dtype == CLOVE_DTYPE_BF16 ? logits::pick<CLOVE_DTYPE_BF16>(a.out_dtype)
                                                                : logits::pick<CLOVE_DTYPE_FP32>(a.out_dtype);
    CLOVE_LAUNCH(kernel, dim3((unsigned)(a.batch * slices)), dim3(logits::kThreads),
                 (a.bias_ids ? 2 : 1) * slice * sizeof(unsigned), stream, a, slice, slices);
    return check_launch();
}

}  // namespace clove
