/*
 * clove_gemm C ABI -- MI355X (gfx950) GEMM hot path of Clove Compute.
 *
 * Plain C: raw device pointers, int dimensions, a status code.  Every entry
 * point is asynchronous on `stream` (a hipStream_t; NULL = the default stream),
 * does not synchronise the host, and validates its arguments before touching
 * the GPU.  Half-precision buffers are IEEE binary16 (passed as void*).
 * All matrices are dense row-major.  Output buffers must not overlap inputs.
 *
 * Each declaration names the reference interface it replaces (paths relative
 * to the Clove Compute source tree).  The C++ spellings with the reference's
 * names, argument order and defaults live in <clove/gemm.h>.
 *
 * Scratch: split-K launches keep a per-(device, stream) scratch buffer that
 * the library allocates on first use (hipMalloc) and keeps until
 * clove_release_scratch() or process exit.  Calls on different streams never
 * share scratch; calls on one stream are ordered by the stream.  A call that
 * needs more scratch than the stream holds allocates a larger buffer (twice
 * the size or more) and keeps the old one until clove_release_scratch(), so
 * that calls of other host threads on the same stream that already took it
 * stay valid; no call synchronises a stream.  Host threads may issue calls on
 * one stream at once: those that use the library's scratch queue all of their
 * launches before another thread's begins.  (A bound workspace is the caller's:
 * one for each thread and stream.)
 */
#ifndef CLOVE_GEMM_C_H
#define CLOVE_GEMM_C_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum clove_status {
    CLOVE_OK = 0,
    CLOVE_ERR_NULL_POINTER = 1,   /* a required pointer is NULL */
    CLOVE_ERR_INVALID_DIM = 2,    /* a dimension is negative */
    CLOVE_ERR_INVALID_ARG = 3,    /* odd K for INT4, bad mode, misaligned half pointer */
    CLOVE_ERR_ALIASING = 4,       /* the output overlaps an input */
    CLOVE_ERR_OUT_OF_MEMORY = 5,  /* scratch allocation failed */
    CLOVE_ERR_LAUNCH = 6,         /* the HIP runtime rejected a launch */
    CLOVE_ERR_NO_DEVICE = 7,      /* no usable HIP device */
    CLOVE_ERR_WORKSPACE = 8,      /* the bound workspace is too small for the call */
    CLOVE_ERR_SCRATCH_LIMIT = 9   /* clove_gemm_fp16_noalloc: the call needs more scratch
                                     than CLOVE_NOALLOC_SCRATCH_BYTES */
} clove_status_t;

/* INT4 arithmetic selected by clove_gemm_int4_ex. */
typedef enum clove_int4_mode {
    /* per-128-group (q - zero) * scale on both operands, int32 partials per group
     * (the layout and scales the reference API declares) */
    CLOVE_INT4_GROUPWISE = 0,
    /* the reference kernel's arithmetic: q - 8, zeros ignored, whole-K integer
     * sum scaled by the last group's scales, B stride floor(N/2)
     * (src/kernels/gemm_int4.cu:45-193) */
    CLOVE_INT4_REFERENCE_LITERAL = 1
} clove_int4_mode_t;

/* include/clove/kernels/gemm.cuh:72 (INT4_GROUP_SIZE) */
#define CLOVE_INT4_GROUP_SIZE 128

/* Human-readable name of a status code (static storage). */
const char* clove_status_string(clove_status_t status);

/* ABI revision of this header; bumped on any signature change. */
int clove_abi_version(void);

/*
 * C = alpha * A @ B + beta * C.  A [M,K], B [K,N], C [M,N], fp16; fp32
 * accumulation and fp32 epilogue, fp16 round-to-nearest-even output.
 * beta == 0 never reads C.  M == 0 or N == 0 is a no-op; K == 0 gives beta*C.
 * Replaces clove::gemm_fp16 (include/clove/kernels/gemm.cuh:41-49,
 * src/kernels/gemm_fp16.cu:277-305).
 */
clove_status_t clove_gemm_fp16(const void* A, const void* B, void* C,
                               int M, int N, int K, float alpha, float beta,
                               void* stream);

/*
 * Batched clove_gemm_fp16 with contiguous batches: A [batch,M,K],
 * B [batch,K,N], C [batch,M,N].
 * Replaces clove::gemm_fp16_batched (include/clove/kernels/gemm.cuh:93-101,
 * src/kernels/gemm_fp16.cu:366-383).
 */
clove_status_t clove_gemm_fp16_batched(const void* A, const void* B, void* C,
                                       int batch, int M, int N, int K,
                                       float alpha, float beta, void* stream);

/*
 * W8A8 with per-tensor scale and zero point:
 *   acc = sum_k (A_q[m,k] - A_zero) * (B_q[k,n] - B_zero)      (int32, exact)
 *   C   = fp16( float(acc) * (A_scale * B_scale) )
 * A_q [M,K], B_q [K,N] int8; C [M,N] fp16.
 * Replaces clove::gemm_int8 (include/clove/kernels/gemm.cuh:57-65,
 * src/kernels/gemm_int8.cu:119-137).
 */
clove_status_t clove_gemm_int8(const int8_t* A_q, const int8_t* B_q, void* C,
                               int M, int N, int K,
                               float A_scale, int8_t A_zero,
                               float B_scale, int8_t B_zero, void* stream);

/* INT8 arithmetic modes of clove_gemm_int8_ex */
typedef enum {
    /* acc = sum over k < K only (clove_gemm_int8) */
    CLOVE_INT8_EXACT = 0,
    /* the reference kernel's accumulator at any K: it walks K in 32-wide tiles,
     * loads 0 for k >= K and subtracts the zero points from those zeros too, so
     * acc = exact + (32*ceil(K/32) - K) * A_zero * B_zero
     * (src/kernels/gemm_int8.cu:43, 52-54, 63-64, 89-93); equal to
     * CLOVE_INT8_EXACT when K % 32 == 0 or a zero point is 0 */
    CLOVE_INT8_REFERENCE_LITERAL = 1
} clove_int8_mode_t;

/*
 * clove_gemm_int8 with a choice of arithmetic mode (clove_int8_mode_t).
 * Extension of clove::gemm_int8 (include/clove/kernels/gemm.cuh:57-65).
 */
clove_status_t clove_gemm_int8_ex(const int8_t* A_q, const int8_t* B_q, void* C,
                                  int M, int N, int K,
                                  float A_scale, int8_t A_zero,
                                  float B_scale, int8_t B_zero, int mode, void* stream);

/*
 * W8A8 with fp16 per-row scales A_scale [M] (tokens) and per-column scales
 * B_scale [N] (output channels): C = fp16(float(acc) * (A_scale[m]*B_scale[n])).
 * With broadcast scales it equals clove_gemm_int8 bit for bit.  Extension of
 * clove::gemm_int8 (include/clove/kernels/gemm.cuh:57-65), which is per-tensor.
 */
clove_status_t clove_gemm_int8_rowcol(const int8_t* A_q, const int8_t* B_q,
                                      const void* A_scale, const void* B_scale,
                                      void* C, int M, int N, int K,
                                      int8_t A_zero, int8_t B_zero, void* stream);

/*
 * Test hook: the raw int32 accumulators [M,N] of the INT8 kernels (same kernels,
 * integer epilogue).  No reference counterpart: it exposes the bit-exact
 * accumulator the reference's gemm_int8_kernel keeps in registers
 * (src/kernels/gemm_int8.cu:37, :87-96).
 */
clove_status_t clove_gemm_int8_acc32(const int8_t* A_q, const int8_t* B_q,
                                     int32_t* acc, int M, int N, int K,
                                     int8_t A_zero, int8_t B_zero, void* stream);

/*
 * Packed INT4 x INT4 GEMM, group-wise (CLOVE_INT4_GROUPWISE):
 *   A_q [M, K/2]        two nibbles per byte, even k in the high nibble
 *   A_scale, A_zero     [M, ceil(K/128)] fp16
 *   B_q [K, ceil(N/2)]  two nibbles per byte along N, even n in the high nibble
 *   B_scale, B_zero     [ceil(K/128), N] fp16
 *   C [M,N] fp16 = sum_g A_scale[m,g]*B_scale[g,n] *
 *                  sum_{k in g} (qA - zA[m,g]) * (qB - zB[g,n])
 * Zero points are integer offsets stored as fp16 (non-integers round to nearest
 * even).  K must be even.  For even N the byte layout is the reference's.
 * Replaces clove::gemm_int4 (include/clove/kernels/gemm.cuh:77-87,
 * src/kernels/gemm_int4.cu:195-216).
 */
clove_status_t clove_gemm_int4(const uint8_t* A_q, const void* A_scale,
                               const void* A_zero, const uint8_t* B_q,
                               const void* B_scale, const void* B_zero, void* C,
                               int M, int N, int K, void* stream);

/*
 * Test hook: the per-group int32 partial sums of the group-wise INT4 GEMM,
 *   P[(m * N + n) * G + g] = sum_{k in group g} (qA[m,k] - zA[m,g]) * (qB[k,n] - zB[g,n])
 * (G = K / 128), the exact integers the int8-MFMA kernel folds into its fp32
 * accumulators (same pre-pass, same kernel, no fold), so that they can be
 * checked bit for bit.  No reference counterpart: the reference's
 * gemm_int4_kernel never forms per-group partials (src/kernels/gemm_int4.cu:
 * 137-190 sums every k before scaling).  Operands as clove_gemm_int4 (no
 * scales).  Domain: K a multiple of 256, A_q 16-byte aligned, P 4-byte aligned
 * (else CLOVE_ERR_INVALID_ARG); a partial whose row or column zero point lies
 * outside [-112, 127] is INT32_MIN.
 */
clove_status_t clove_gemm_int4_group_acc32(const uint8_t* A_q, const void* A_zero,
                                           const uint8_t* B_q, const void* B_zero,
                                           int32_t* P, int M, int N, int K, void* stream);

/* clove_gemm_int4 with an explicit arithmetic mode (see clove_int4_mode_t).
 * In CLOVE_INT4_REFERENCE_LITERAL mode B_q is [K, floor(N/2)] as in the
 * reference and the zero pointers may be NULL (never read). */
clove_status_t clove_gemm_int4_ex(const uint8_t* A_q, const void* A_scale,
                                  const void* A_zero, const uint8_t* B_q,
                                  const void* B_scale, const void* B_zero,
                                  void* C, int M, int N, int K,
                                  clove_int4_mode_t mode, void* stream);

/*
 * W4A16 linear layer: fp16 activations x group-128 INT4 weights.
 *   Y[t,o] = alpha * sum_k X[t,k] * (qW(o,k) - W_zero[o,g]) * W_scale[o,g]
 *            + beta * Y[t,o]
 * X [T,K] fp16, W_q [O, K/2] (gemm_int4's A layout), W_scale/W_zero [O, K/128]
 * fp16, Y [T,O] fp16.  beta = 1 is the residual add of the reference's o_proj
 * and down_proj (src/runtime/inference.cu:165-168, :191-194).  K even.
 * No reference entry point takes fp16 activations with INT4 weights; this is
 * the linear-layer call (src/runtime/inference.cu:139-194) on INT4 weights.
 */
clove_status_t clove_gemm_w4a16(const void* X, const uint8_t* W_q,
                                const void* W_scale, const void* W_zero, void* Y,
                                int T, int O, int K, float alpha, float beta,
                                void* stream);

/*
 * SwiGLU: output[i] = fp16(silu(gate[i]) * up[i]), silu(x) = x / (1 + exp(-x))
 * in fp32.  Replaces clove::swiglu (include/clove/kernels/activations.cuh:25-31,
 * src/kernels/activations.cu:76-134).  `output` may be `gate` or `up` (in place).
 */
clove_status_t clove_swiglu(const void* gate, const void* up, void* output, int size,
                            void* stream);

/*
 * Fused gate/up projections and SwiGLU on FP16 weights:
 *   output[t,i] = swiglu(fp16(input @ W_gate)[t,i], fp16(input @ W_up)[t,i])
 * input [batch_seq, hidden_dim], W_gate / W_up [hidden_dim, intermediate_dim]
 * (gemm_fp16's B layout), output [batch_seq, intermediate_dim], all fp16.
 * Replaces clove::swiglu_fused, declared in include/clove/kernels/
 * activations.cuh:37-46 and never defined there.  Where gemm_fp16 would run
 * each projection on its GEMV or skinny MFMA kernel (aligned operands, the
 * decode and small-batch shapes), one launch that writes neither projection
 * to memory: each output tile's gate and up sums are formed side by side in
 * the k order of those kernels, so the result equals gemm_fp16 x 2 followed
 * by clove_swiglu bit for bit, and the epilogue applies SwiGLU to their fp16
 * values.  Where gemm_fp16 takes its 256x256 tile (large prefill), exactly
 * those two calls and clove_swiglu, the up projection in a library buffer of
 * batch_seq x intermediate_dim fp16 (bit-identical by construction).  Other
 * shapes (unaligned operands, or hidden_dim % 64 != 0 beyond 4 rows): one
 * direct kernel with the reference naive kernel's fp32 k-order arithmetic for
 * both projections, within the FP16 tolerance of the two-call result.
 */
clove_status_t clove_swiglu_fused(const void* input, const void* W_gate, const void* W_up,
                                  void* output, int batch_seq, int hidden_dim,
                                  int intermediate_dim, void* stream);

/*
 * Fused MLP gate/up projections and SwiGLU on group-128 INT4 weights:
 *   H[t,i] = swiglu(gate[t,i], up[t,i]),
 *   gate = fp16(X @ dequant(W[0:I])^T),  up = fp16(X @ dequant(W[I:2I])^T)
 * X [T,K] fp16; W_q [2I, K/2] in gemm_int4's A layout with the I gate rows
 * first and the I up rows after them; W_scale / W_zero [2I, K/128] fp16;
 * H [T,I] fp16.  K even.  The reference MLP's gate and up gemm_fp16 calls and
 * its swiglu (src/runtime/inference.cu:172-186) in one pass that writes
 * neither projection to memory (when K % 128 == 0 and X, W_q are 16-byte
 * aligned, or T <= 4; other shapes run the two W4A16 layers and SwiGLU).
 */
clove_status_t clove_w4a16_swiglu(const void* X, const uint8_t* W_q, const void* W_scale,
                                  const void* W_zero, void* H, int T, int I, int K,
                                  void* stream);

/* ------------------------------------------------------------------------
 * The decode step around the linear layers.  No reference counterpart is
 * replaced (the reference declares a paged_attention in include/clove/kernels/
 * attention.cuh:85-100 and never defines it).  Element type `dtype`: see
 * clove_dtype_t; every sum, norm and softmax statistic is fp32 and a result is
 * rounded once (what a softmax weight keeps: clove_paged_attention).  Row strides count elements.  All of these take their scratch
 * as the GEMMs do (library buffers, a bound workspace, or a size query).
 * ------------------------------------------------------------------------ */
typedef enum clove_dtype {
    CLOVE_DTYPE_FP16 = 0,
    CLOVE_DTYPE_BF16 = 1,
    CLOVE_DTYPE_FP32 = 2 /* logits only */
} clove_dtype_t;

/* Largest head_dim and max_context of these operators. */
#define CLOVE_MAX_HEAD_DIM 1024
#define CLOVE_MAX_CONTEXT (1 << 30)

/* The key-value cache of one layer, in pages.  Key (page, head, row) starts at
 * element page * page_stride + (head * page_size + row) * head_dim of `k`, its
 * value at the same element of `v`; page_stride 0 means dense pages
 * (kv_heads * page_size * head_dim).  Slot s is row s % page_size of page
 * s / page_size.  dtype is FP16 or BF16. */
typedef struct clove_kv_cache {
    void* k;
    void* v;
    int64_t page_stride;
    int num_pages;
    int page_size;
    int kv_heads;
    int head_dim;
    int dtype;
} clove_kv_cache_t;

/*
 * Norms of queries and keys for each head, the position rotation, and the
 * write into the cache, in one pass over the fused QKV projection's output:
 *   qkv row t (qkv_stride elements apart): q_heads queries, kv_heads keys, then
 *   kv_heads values of head_dim elements each
 *   x = a query or key;  y = x / sqrt(mean(x^2) + eps) * weight, where its
 *   weight (q_weight, k_weight [head_dim], `dtype`) is not NULL, else y = x
 *   first rot_dim elements rotated by c, s = rope_cos/rope_sin[positions[t], i]
 *   (fp32 [max_position, rot_dim / 2]): (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
 *   with (a, b) = (i, i + rot_dim / 2), or (2i, 2i + 1) where `interleaved`
 * Queries go to q_out [T, q_heads, head_dim] (rows q_out_stride apart); keys to
 * k_out likewise (NULL: not wanted); keys and values to slot slots[t] of
 * `cache` (NULL: not wanted).  A slot outside the cache (a negative one marks a
 * padding token) is not written; two tokens of one call must not name the same
 * slot.  A position outside [0, max_position) makes that token's q and k NaN
 * (rot_dim > 0).  q_out / k_out may be the queries / keys of qkv themselves
 * (same rows; of several the same stride), else outputs must not overlap inputs.
 * rot_dim is even and at most head_dim; with rot_dim 0 the tables and positions
 * are not read.  T == 0 is a no-op.
 */
clove_status_t clove_qk_norm_rope(const void* qkv, int64_t qkv_stride, const void* q_weight,
                                  const void* k_weight, float eps, const float* rope_cos,
                                  const float* rope_sin, int max_position, const int32_t* positions,
                                  void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride,
                                  const clove_kv_cache_t* cache, const int32_t* slots, int T,
                                  int q_heads, int kv_heads, int head_dim, int rot_dim,
                                  int interleaved, int dtype, void* stream);

/*
 * Attention of one new token per sequence over the paged cache.  Query head h
 * of sequence b reads KV head h / (q_heads / kv_heads).  Key j of sequence b is
 * row j % page_size of page block_table[b * table_stride + j / page_size];
 * with n = context_lens[b] (taken as at most max_context, at least 0) it sees
 * the keys j in [window > 0 ? max(0, n - window) : 0, n) whose page lies in
 * [0, num_pages), a page outside it being absent:
 *   s_j = scale * q . k_j   (softcap > 0: softcap * tanh(s_j / softcap))
 *   p = softmax(s),  out = sum_j p_j v_j      (a query that sees no key: 0)
 * and, where `weights` (fp32, rows weights_stride apart) is not NULL,
 *   weights[b, j] += sum over the heads of p_j      for every key it sees.
 * q, out [batch, q_heads, head_dim] (rows q_stride / out_stride apart) are the
 * cache's dtype.  Cache rows that no key names are not used, whatever they hold.
 * An infinite value makes its element of the result infinite (values of both
 * signs, or a weight of 0, make it NaN).  The weights enter the sum over the
 * values with 24 bits from a BF16 cache and 22 from an FP16 one, whose weights
 * are held to 2^-40 of the largest; below 2^-126 of it they are 0.
 * max_context bounds the lengths on the host: it is at most table_stride *
 * page_size (and weights_stride), and a row of the table has ceil(max_context /
 * page_size) entries, of which those past the length may be anything.  The work
 * is shared out on the device by the lengths themselves, so a recorded call may
 * be replayed with others; with more than about 7900 sequences x KV heads x 16
 * query heads of one, long sequences are not split.  Sums run in a fixed order: a call gives the same
 * bits every time.  With `weights` the call takes a buffer of batch * q_heads *
 * max_context floats of scratch.
 */
clove_status_t clove_paged_attention(const void* q, int64_t q_stride, const clove_kv_cache_t* cache,
                                     const int32_t* block_table, int64_t table_stride,
                                     const int32_t* context_lens, void* out, int64_t out_stride,
                                     float* weights, int64_t weights_stride, int batch, int q_heads,
                                     int max_context, float scale, float softcap, int window,
                                     void* stream);

/*
 * Eviction from the cache by accumulated attention weight: cuts every sequence
 * longer than `budget` down to it, in place.  Of the n = context_lens[b] tokens
 * (at most max_context) those are kept first whose position (positions[b, i],
 * of the token in slot i) is < sinks or > newest - recent (newest: the largest
 * of them), then those of the largest weights[b, i]; at equal weight (-0 equals
 * 0, NaN is below everything) the lower slot stays.  Kept tokens below slot
 * `budget` do not move; the j-th kept one past it moves into the j-th slot
 * below it that is free: its K and V rows of every head, its weight and its
 * position.  Keys hold their rotation, so attention without a window does not
 * depend on their order.
 *   lens_out[b]            min(n, budget)
 *   weights_out[b, i], positions_out[b, i]   of the slots as they are then; 0
 *                          and -1 for lens_out[b] <= i < max_context
 * Each output may be its input (same rows; of several the same stride).  A row
 * whose page lies outside the cache is not copied.  Sequences must not share
 * pages, or have a page twice.  A second call with the same inputs moves the same
 * rows again and changes nothing.
 */
clove_status_t clove_cache_evict(const clove_kv_cache_t* cache, const int32_t* block_table,
                                 int64_t table_stride, const int32_t* context_lens,
                                 const float* weights, int64_t weights_stride,
                                 const int32_t* positions, int64_t positions_stride,
                                 float* weights_out, int64_t weights_out_stride,
                                 int32_t* positions_out, int64_t positions_out_stride,
                                 int32_t* lens_out, int batch, int max_context, int budget,
                                 int sinks, int recent, void* stream);

/*
 * Penalties for repeated tokens, biases and a grammar mask on logits, fp32:
 *   x = logits[b, v]
 *   v anywhere in history[b, 0 : history_lens[b]]:  x = x > 0 ? x / r : x * r
 *   c = how often v is in history[b, prompt_lens[b] : history_lens[b]]
 *   x -= frequency[b] * c;  c > 0: x -= presence[b]
 *   v in bias_ids[b, 0 : bias_counts[b]]:  x += its bias_values (the last entry
 *   for v counts)
 *   bit v % 32 of allowed[b, v / 32] clear:  x = -infinity
 *   out[b, v] = x
 * r = repetition[b].  Any of repetition, presence, frequency [batch], history,
 * bias_ids and allowed may be NULL: that part is left out (prompt_lens NULL: no
 * prompt, everything was generated; bias_counts NULL: all bias_stride entries).
 * Rows of history and of the bias lists are history_stride / bias_stride entries
 * long, any of which may be read; lengths are taken as at least 0 and at most
 * that.  Ids outside [0, vocab) are ignored.  logits are `dtype` (FP16, BF16 or
 * FP32), out is `out_dtype` (the same, or FP32), rows logits_stride / out_stride
 * elements apart; out may be logits itself where dtype and (of several rows)
 * stride agree.
 */
clove_status_t clove_penalize_logits(const void* logits, int64_t logits_stride, int dtype, void* out,
                                     int64_t out_stride, int out_dtype, int batch, int vocab,
                                     const int32_t* history, int64_t history_stride,
                                     const int32_t* history_lens, const int32_t* prompt_lens,
                                     const float* repetition, const float* presence,
                                     const float* frequency, const int32_t* bias_ids,
                                     const float* bias_values, int64_t bias_stride,
                                     const int32_t* bias_counts, const uint32_t* allowed,
                                     int64_t allowed_stride, void* stream);

/* ------------------------------------------------------------------------
 * A sparse MLP block around the linear layers: the norms before and after a
 * block with its residual, the router, and the products of the experts it
 * chose.  No reference counterpart.  Element types, strides, rounding and
 * scratch as for the decode step above; only the products take scratch.
 * ------------------------------------------------------------------------ */

/* Largest D of clove_block_norm, experts and top_k of the others. */
#define CLOVE_MAX_NORM_DIM 32768
#define CLOVE_MAX_EXPERTS 1024
#define CLOVE_MAX_TOP_K 64

/*
 * What a block gave joins the residual stream, and the next block's input
 * leaves it, in one pass:
 *   u = x / sqrt(mean(x^2) + eps) * post_weight, where post_weight is not
 *       NULL, else u = x
 *   y = residual + scale * gate * u
 *   h = y / sqrt(mean(y^2) + eps) * pre_weight
 * x, gate, the weights and h are `dtype` (FP16 or BF16), residual and y are
 * residual_dtype (the same, or FP32).  h comes from the fp32 y, not from the
 * rounded one; squares that leave fp32 are taken of scaled rows, so a finite row
 * of any size has its norm.  gate is one row for all tokens (gate_stride 0) or a
 * row for each, NULL: 1; pre_weight NULL: 1; x NULL: y = residual (a stack's
 * first norm; post_weight, gate and scale are not used); residual NULL: 0 (not
 * both).
 * y_out or h_out may be NULL: not wanted.
 * Rows [T, D], strides in elements.  y_out may be residual, y_out or h_out may
 * be x or gate (same rows and type; of several rows the same stride); else
 * outputs overlap neither inputs nor each other.  T == 0 or D == 0 is a no-op.
 */
clove_status_t clove_block_norm(const void* x, int64_t x_stride, const void* residual,
                                int64_t residual_stride, const void* post_weight, const void* gate,
                                int64_t gate_stride, float scale, const void* pre_weight, void* y_out,
                                int64_t y_out_stride, void* h_out, int64_t h_out_stride, int T, int D,
                                float eps, int dtype, int residual_dtype, void* stream);

typedef enum clove_route_score {
    CLOVE_ROUTE_SOFTMAX = 0, /* exp(x_e) / the sum of it over the token's available experts */
    CLOVE_ROUTE_SIGMOID = 1  /* 1 / (1 + exp(-x_e)) */
} clove_route_score_t;

/*
 * The experts of each token and their weights, from the router's logits
 * [T, experts] (`dtype`: FP16, BF16 or FP32; rows logits_stride apart):
 *   s_e = score of x_e;  c_e = s_e + bias_e (bias [experts] fp32, NULL: none)
 *   groups > 1: the experts are that many equal runs; the value of a run is the
 *   sum of its group_top (1 or 2) largest c, and only those of the top_groups
 *   largest values are left
 *   ids[t, 0 : top_k]  = the experts of the largest c (without a bias: of the
 *   largest x), largest first
 *   weights[t, j]      = scale * s of that expert, where `renormalize` divided
 *   by the sum of the chosen ones' (a sum of 0 divides nothing)
 * Equal values go to the lowest index.  s, c and the sums are 64 bits: only
 * the weights (fp32) are rounded.  An expert whose logit or bias is NaN or
 * -infinity is not available; a place for which no expert is left has id -1
 * and weight 0.  +infinity counts as the limit (softmax: shared equally among
 * those that have it).
 */
clove_status_t clove_moe_route(const void* logits, int64_t logits_stride, int dtype, const float* bias,
                               int score, int groups, int top_groups, int group_top, int top_k,
                               int renormalize, float scale, int32_t* ids, float* weights, int T,
                               int experts, void* stream);

/*
 * clove_w4a16_swiglu with weights of its own for every (token, place) pair
 * p = t * top_k + j, those of expert e = expert_ids[p]:
 *   H[p, i] = fp16(silu(g) * u),  g = X[t] . dequant(W[e, i]),
 *                                 u = X[t] . dequant(W[e, I + i])
 * X [T, K] fp16, expert_ids [T, top_k], W_q [experts, 2 I, K / 2] in gemm_int4's
 * A layout (of each expert the I gate rows, then the I up rows), W_scale /
 * W_zero [experts, 2 I, ceil(K / 128)] fp16, H [T top_k, I] fp16.  g and u stay
 * fp32 (no rounding before SwiGLU).  A pair whose id lies outside [0, experts)
 * (a padding token, an expert of another device) has no product and its row of
 * H is left as it is; an expert may come twice in a row.  K is even.  Which
 * kernel runs goes by the sizes, the alignments and the device's number of CUs
 * alone, and a row's bits do not depend on what other tokens chose.  Fastest
 * with K % 32 == 0 and 16-byte aligned X and W_q.
 * Zero points round to the nearest integer, as clove_gemm_w4a16's; q - z is
 * exact up to 2048 in magnitude and rounded to fp16 past that.
 * Scratch: 4 bytes a pair, at most 2 MB (more pairs than 2^19, or an X of 2^31
 * bytes, go in parts), and up to 64 MB of fp32 products where K is split.  2^31
 * tiles of 32 rows by 32 pairs and more, or one token's X of 2^31 bytes (here a
 * row, below top_k rows), are CLOVE_ERR_INVALID_DIM.
 */
clove_status_t clove_moe_w4a16_swiglu(const void* X, const int32_t* expert_ids, const uint8_t* W_q,
                                      const void* W_scale, const void* W_zero, void* H, int T, int top_k,
                                      int experts, int I, int K, void* stream);

/*
 * clove_gemm_w4a16 with weights of its own for every pair, summed over the
 * token's places:
 *   Y[t, o] = alpha * sum_j weights[t, j] * (H[p] . dequant(W[e, o]))
 *             + beta * Y[t, o],   p = t * top_k + j, e = expert_ids[p]
 * H [T top_k, K] fp16, expert_ids [T, top_k], weights [T, top_k] fp32 (NULL: 1),
 * W_q [experts, O, K / 2], W_scale / W_zero [experts, O, ceil(K / 128)] fp16,
 * Y [T, O] fp16, rounded once.  The row of H and the weight of a pair without a
 * product (see above) are not used; a token without any gets beta * Y.
 * beta == 0 never reads Y.  K is even.  The rest as above, but for the scratch:
 * the pairs' fp32 products besides, T top_k O * 4 bytes up to 512 MB (with more,
 * as many outputs at a time as fit there; at least 256), which library scratch
 * rounds up to a power of two.
 */
clove_status_t clove_moe_w4a16(const void* H, const int32_t* expert_ids, const float* weights,
                               const uint8_t* W_q, const void* W_scale, const void* W_zero, void* Y, int T,
                               int top_k, int experts, int O, int K, float alpha, float beta, void* stream);

/* Caller-owned workspace (no reference counterpart: the reference allocates no
 * scratch).  Per host thread, three modes:
 *
 *  - library scratch (the default): the per-(device, stream) buffers above;
 *  - a bound workspace, clove_workspace_bind(ptr, bytes): calls on this thread
 *    take their split-K partials, completion counters and intermediates from
 *    [ptr, ptr + bytes) and allocate nothing.  With at least the queried size
 *    a call's results are bit for bit those with library scratch.  A call
 *    that needs more returns CLOVE_ERR_WORKSPACE and launches nothing, unless
 *    it has an ordinary plan that takes none, which it then runs (the same
 *    sums, fp32 ones in another order): FP16 products up to K = 1024 and INT8
 *    up to K = 2048 on the skinny kernel without their K split, and with any K
 *    where operands are unaligned or K is not a whole number of K tiles and
 *    64 x 64 tiles cover the CUs; W4A16 with fewer than 16 groups (20 with up
 *    to 32 tokens), or with up to 32 tokens on wide layers or within the
 *    streaming kernel's reach; w4a16_swiglu at 3 or 4 tokens; INT4 with
 *    K % 128 != 0.  The same calls run that way when the library's scratch
 *    cannot grow: during a stream capture, where they do not try to, or when
 *    memory is short; every other call allocates, or returns
 *    CLOVE_ERR_OUT_OF_MEMORY.  (No kernel uses private
 *    scratch either, which the library build checks.)  ptr must be 256-byte aligned
 *    and bytes >= CLOVE_WORKSPACE_MIN_BYTES; the first CLOVE_WORKSPACE_MIN_BYTES
 *    (the counters) must be zero before the first call, and every call leaves
 *    them zero.  Calls that may run at the same time on the device (other
 *    streams, other threads) must not share a workspace.
 *    clove_workspace_bind(NULL, 0) returns to library scratch;
 *  - a size query: between clove_workspace_query_begin() and
 *    clove_workspace_query_end(), calls on this thread validate their
 *    arguments and plan their launches but launch nothing and allocate
 *    nothing; query_end returns the largest workspace any of them needs
 *    (0 if none needs one) and restores the previous mode.  A query plans
 *    with the pointers it is given (alignment selects kernels), so pass the
 *    ones the real call will use. */
#define CLOVE_WORKSPACE_MIN_BYTES ((size_t)65536)
clove_status_t clove_workspace_bind(void* ptr, size_t bytes);
clove_status_t clove_workspace_query_begin(void);
size_t clove_workspace_query_end(void);

/*
 * clove_gemm_fp16 for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * No reference counterpart.  Same arguments, kernels, split plans and results
 * (bit for bit) as clove_gemm_fp16; it calls no hipMalloc / hipFree and no
 * allocating library routine.  Its split-K partials and completion counters
 * live in a fixed device array of CLOVE_NOALLOC_SCRATCH_BYTES per GPU (the
 * library's static device memory, held until the process ends); a call that
 * would need more returns CLOVE_ERR_SCRATCH_LIMIT and launches nothing.
 * Every shape with M <= 512 and N, K <= 8192 whose operands are 16-byte
 * aligned, with N % 8 == 0 and K % 64 == 0, fits, as does every shape on the
 * 256x256 tile (its K split needs at most 64 MiB of partials).  The first call on a device clears the array's counters
 * with one small kernel on `stream`.  Every call on a GPU shares that GPU's
 * array: calls that may overlap on one GPU (other streams, other host
 * threads) race and must be serialised by the caller.  Inside a workspace
 * size query it validates and plans as clove_gemm_fp16, returns
 * CLOVE_ERR_SCRATCH_LIMIT for a call the array cannot hold, and leaves the
 * query's size as it was (the array is not the caller's workspace).
 */
#define CLOVE_NOALLOC_SCRATCH_BYTES ((size_t)65 << 20)
clove_status_t clove_gemm_fp16_noalloc(const void* A, const void* B, void* C,
                                       int M, int N, int K, float alpha, float beta,
                                       void* stream);

/* Frees the scratch buffers held for the current device (all streams),
 * including the SwiGLU intermediates and buffers replaced by larger ones.
 * Synchronises the device first; no other call may be using the library on
 * this device meanwhile.  No reference counterpart. */
clove_status_t clove_release_scratch(void);

#ifdef __cplusplus
}
#endif

#endif /* CLOVE_GEMM_C_H */
