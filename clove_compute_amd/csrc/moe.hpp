// Operators of a sparse MLP block: the norms before and after a block with its
// residual, the router, the products of the chosen experts.  Shared by the C ABI
// layer (capi.hip) and their kernels; not installed.
#pragma once

#include "decode.hpp"

namespace clove {

struct BlockNormArgs {
    const void* x = nullptr;  // null: nothing joins the residual
    int64_t x_stride = 0;
    const void* residual = nullptr;  // null: zero
    int64_t residual_stride = 0;
    const void* post_weight = nullptr;  // [D] or null: x is not normed
    const void* gate = nullptr;         // null: 1
    int64_t gate_stride = 0;            // 0: one row for all
    float scale = 1.0f;
    const void* pre_weight = nullptr;  // [D] or null: 1
    void* y_out = nullptr;             // null: not wanted
    int64_t y_out_stride = 0;
    void* h_out = nullptr;  // null: not wanted
    int64_t h_out_stride = 0;
    int T = 0, D = 0;
    float eps = 0.0f;
    int dtype = 0, residual_dtype = 0;
};
clove_status_t launch_block_norm(const BlockNormArgs& a, hipStream_t stream);

struct RouteArgs {
    const void* logits = nullptr;
    int64_t logits_stride = 0;
    int dtype = 0;
    const float* bias = nullptr;
    int score = 0, groups = 1, top_groups = 1, group_top = 1, top_k = 1;
    bool renormalize = false;
    float scale = 1.0f;
    int32_t* ids = nullptr;
    float* weights = nullptr;
    int T = 0, experts = 0;
};
clove_status_t launch_moe_route(const RouteArgs& a, hipStream_t stream);

// Products of pairs (token, place): pair p = t top_k + j with the weights of
// expert ids[p], none where that lies outside [0, experts).
struct MoeArgs {
    const uint16_t* X = nullptr;  // SwiGLU: [T, K]; else [T top_k, K]
    const int32_t* ids = nullptr;
    const float* weights = nullptr;  // [T top_k] or null: 1 (not SwiGLU)
    const uint8_t* W = nullptr;      // [experts, rows, K / 2], SwiGLU: 2 O rows, gate first
    const uint16_t* scale = nullptr;
    const uint16_t* zero = nullptr;
    uint16_t* Y = nullptr;  // SwiGLU: [T top_k, O]; else [T, O]
    int T = 0, top_k = 0, experts = 0, O = 0, K = 0;
    float alpha = 1.0f, beta = 0.0f;
};
clove_status_t launch_moe_w4a16(const MoeArgs& a, bool swiglu, hipStream_t stream);

}  // namespace clove
