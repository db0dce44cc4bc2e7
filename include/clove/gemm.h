// C++ drop-in for the Clove Compute GEMM API on MI355X.
//
// Same namespace, function names, argument order and default arguments as the
// reference header include/clove/kernels/gemm.cuh:41-101, with hipStream_t in
// place of cudaStream_t.  Every call forwards to the C ABI in <clove/gemm_c.h>;
// a non-OK status is reported the reference's way (include/clove/common.cuh:11-21):
// print file:line and the error, then exit(EXIT_FAILURE).  <clove/common.h>
// brings the rest of the reference's common header: CLOVE_CHECK_CUDA /
// CLOVE_CHECK_LAST / CLOVE_SYNC_CHECK, cdiv, DType, dtype_size, CudaType.
#pragma once

#include <clove/common.h>
#include <clove/gemm_c.h>

#include <hip/hip_fp16.h>
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>

namespace clove {

// include/clove/kernels/gemm.cuh:13-31: the FP16 GEMM's tile configuration,
// same member names.  The values describe this library's large-shape FP16
// kernel on gfx950: a 256x256x64 workgroup tile of four 64-wide waves, each
// wave a 128x128 tile of 16x16x32 fp16 MFMAs (fp32 accumulation).  Nothing in
// the library reads these; they are informational, as in the reference.
struct GemmConfig {
    static constexpr int BM = 256;  // workgroup tile M
    static constexpr int BN = 256;  // workgroup tile N
    static constexpr int BK = 64;   // workgroup tile K (one LDS stage)

    static constexpr int WM = 128;  // wave tile M
    static constexpr int WN = 128;  // wave tile N

    static constexpr int TM = 8;    // MFMA tiles per wave along M (WM / WMMA_M)
    static constexpr int TN = 8;    // MFMA tiles per wave along N (WN / WMMA_N)

    static constexpr int NUM_THREADS = 256;  // 4 waves of 64 lanes

    // matrix-core instruction shape (v_mfma_f32_16x16x32_f16); the reference
    // names it after WMMA
    static constexpr int WMMA_M = 16;
    static constexpr int WMMA_N = 16;
    static constexpr int WMMA_K = 32;
};

// include/clove/kernels/gemm.cuh:72
constexpr int INT4_GROUP_SIZE = CLOVE_INT4_GROUP_SIZE;

namespace detail {
inline void check(clove_status_t status, const char* file, int line) {
    if (status != CLOVE_OK) {
        std::fprintf(stderr, "clove error at %s:%d: %s\n", file, line,
                     clove_status_string(status));
        std::exit(EXIT_FAILURE);
    }
}
}  // namespace detail

#define CLOVE_CHECK_STATUS(call) ::clove::detail::check((call), __FILE__, __LINE__)

// include/clove/kernels/gemm.cuh:41-49
inline void gemm_fp16(const half* A, const half* B, half* C, int M, int N, int K,
                      float alpha = 1.0f, float beta = 0.0f, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_fp16(A, B, C, M, N, K, alpha, beta, stream));
}

// include/clove/kernels/gemm.cuh:57-65
inline void gemm_int8(const int8_t* A_q, const int8_t* B_q, half* C, int M, int N, int K,
                      float A_scale, int8_t A_zero, float B_scale, int8_t B_zero,
                      hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_int8(A_q, B_q, C, M, N, K, A_scale, A_zero, B_scale,
                                       B_zero, stream));
}

// include/clove/kernels/gemm.cuh:77-87
inline void gemm_int4(const uint8_t* A_q, const half* A_scale, const half* A_zero,
                      const uint8_t* B_q, const half* B_scale, const half* B_zero, half* C,
                      int M, int N, int K, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_int4(A_q, A_scale, A_zero, B_q, B_scale, B_zero, C, M, N,
                                       K, stream));
}

// include/clove/kernels/gemm.cuh:93-101
inline void gemm_fp16_batched(const half* A, const half* B, half* C, int batch, int M, int N,
                              int K, float alpha = 1.0f, float beta = 0.0f,
                              hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(
        clove_gemm_fp16_batched(A, B, C, batch, M, N, K, alpha, beta, stream));
}

// include/clove/kernels/activations.cuh:25-31
inline void swiglu(const half* gate, const half* up, half* output, int size,
                   hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_swiglu(gate, up, output, size, stream));
}

// include/clove/kernels/activations.cuh:37-46 (declared, never defined, in the
// reference)
inline void swiglu_fused(const half* input, const half* W_gate, const half* W_up, half* output,
                         int batch_seq, int hidden_dim, int intermediate_dim,
                         hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_swiglu_fused(input, W_gate, W_up, output, batch_seq, hidden_dim,
                                          intermediate_dim, stream));
}

// Extensions (no reference counterpart; see <clove/gemm_c.h>).
inline void gemm_int8_rowcol(const int8_t* A_q, const int8_t* B_q, const half* A_scale,
                             const half* B_scale, half* C, int M, int N, int K,
                             int8_t A_zero = 0, int8_t B_zero = 0, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_int8_rowcol(A_q, B_q, A_scale, B_scale, C, M, N, K, A_zero,
                                              B_zero, stream));
}

inline void gemm_int8_ex(const int8_t* A_q, const int8_t* B_q, half* C, int M, int N, int K,
                         float A_scale, int8_t A_zero, float B_scale, int8_t B_zero,
                         clove_int8_mode_t mode, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_int8_ex(A_q, B_q, C, M, N, K, A_scale, A_zero, B_scale,
                                          B_zero, (int)mode, stream));
}

inline void gemm_int4_ex(const uint8_t* A_q, const half* A_scale, const half* A_zero,
                         const uint8_t* B_q, const half* B_scale, const half* B_zero, half* C,
                         int M, int N, int K, clove_int4_mode_t mode, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_gemm_int4_ex(A_q, A_scale, A_zero, B_q, B_scale, B_zero, C, M, N,
                                          K, mode, stream));
}

inline void gemm_w4a16(const half* X, const uint8_t* W_q, const half* W_scale,
                       const half* W_zero, half* Y, int T, int O, int K, float alpha = 1.0f,
                       float beta = 0.0f, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(
        clove_gemm_w4a16(X, W_q, W_scale, W_zero, Y, T, O, K, alpha, beta, stream));
}

inline void w4a16_swiglu(const half* X, const uint8_t* W_q, const half* W_scale,
                         const half* W_zero, half* H, int T, int I, int K,
                         hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_w4a16_swiglu(X, W_q, W_scale, W_zero, H, T, I, K, stream));
}

// The decode step around the linear layers (see <clove/gemm_c.h> for each
// formula; rows are dense unless a stride is given).
inline void qk_norm_rope(const void* qkv, int64_t qkv_stride, const void* q_weight, const void* k_weight, float eps,
                         const float* rope_cos, const float* rope_sin, int max_position, const int32_t* positions,
                         void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride,
                         const clove_kv_cache_t* cache, const int32_t* slots, int T, int q_heads, int kv_heads,
                         int head_dim, int rot_dim, bool interleaved, clove_dtype_t dtype, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_qk_norm_rope(qkv, qkv_stride, q_weight, k_weight, eps, rope_cos, rope_sin, max_position,
                                          positions, q_out, q_out_stride, k_out, k_out_stride, cache, slots, T, q_heads,
                                          kv_heads, head_dim, rot_dim, interleaved ? 1 : 0, (int)dtype, stream));
}

inline void paged_attention(const void* q, int64_t q_stride, const clove_kv_cache_t& cache, const int32_t* block_table,
                            int64_t table_stride, const int32_t* context_lens, void* out, int64_t out_stride, int batch,
                            int q_heads, int max_context, float scale, float softcap = 0.0f, int window = 0,
                            float* weights = nullptr, int64_t weights_stride = 0, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_paged_attention(q, q_stride, &cache, block_table, table_stride, context_lens, out,
                                             out_stride, weights, weights_stride, batch, q_heads, max_context, scale,
                                             softcap, window, stream));
}

inline void cache_evict(const clove_kv_cache_t& cache, const int32_t* block_table, int64_t table_stride,
                        const int32_t* context_lens, const float* weights, int64_t weights_stride,
                        const int32_t* positions, int64_t positions_stride, float* weights_out,
                        int64_t weights_out_stride, int32_t* positions_out, int64_t positions_out_stride,
                        int32_t* lens_out, int batch, int max_context, int budget, int sinks, int recent,
                        hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_cache_evict(&cache, block_table, table_stride, context_lens, weights, weights_stride,
                                         positions, positions_stride, weights_out, weights_out_stride, positions_out,
                                         positions_out_stride, lens_out, batch, max_context, budget, sinks, recent,
                                         stream));
}

inline void penalize_logits(const void* logits, int64_t logits_stride, clove_dtype_t dtype, void* out,
                            int64_t out_stride, clove_dtype_t out_dtype, int batch, int vocab, const int32_t* history,
                            int64_t history_stride, const int32_t* history_lens, const int32_t* prompt_lens,
                            const float* repetition, const float* presence, const float* frequency,
                            const int32_t* bias_ids = nullptr, const float* bias_values = nullptr,
                            int64_t bias_stride = 0, const int32_t* bias_counts = nullptr,
                            const uint32_t* allowed = nullptr, int64_t allowed_stride = 0, hipStream_t stream = 0) {
    CLOVE_CHECK_STATUS(clove_penalize_logits(logits, logits_stride, (int)dtype, out, out_stride, (int)out_dtype, batch,
                                             vocab, history, history_stride, history_lens, prompt_lens, repetition,
                                             presence, frequency, bias_ids, bias_values, bias_stride, bias_counts,
                                             allowed, allowed_stride, stream));
}

}  // namespace clove
