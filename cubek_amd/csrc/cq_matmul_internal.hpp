// What the objects of libcubek_matmul_hip.so share: the arguments of a product, of the routing and of the weighted sum.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/cubek_matmul.h"

namespace cq {

// Threads of a launch along one dimension.
constexpr uint64_t kLaunchThreads = 1ull << 32;

// y[p] = epilogue(x[row(p)] * dequantize(W[e])^T) for the positions p of expert e; a product without experts is one expert that has all
// positions.
struct MatmulArgs {
    const char* words;   // stored codes, row r of expert e at words + e * expert_bytes + r * row_bytes
    const char* scales;  // typed param_dtype
    const char* x;       // [tokens, cols], typed dtype
    char* y;             // [positions, out_cols], typed y_dtype
    const char* bias;    // [experts, wide], typed bias_dtype; or NULL
    const char* residual;    // like y; or NULL
    const int32_t* offsets;  // [experts + 1]; or NULL: one expert
    const int32_t* row_of;   // [positions]; or NULL: row p
    int dtype, y_dtype, param_dtype, bias_dtype;
    uint32_t bits;    // bits per value
    uint32_t native;  // 0: fields of the U32 store and i8 bytes; 1 e4m3, 2 e5m2, 3 e2m1x2
    uint32_t wide;    // rows of W
    uint32_t out_cols;  // columns of y: wide, or half of it where gated
    uint32_t cols;      // columns of W
    uint32_t experts, tokens, positions;
    uint64_t row_bytes, expert_bytes;
    uint32_t block_rows, block_cols;  // 0, 0: one scale per tensor
    uint64_t scale_row, scale_col, scale_expert;  // strides of the scales, in elements
    uint64_t x_stride, y_stride, residual_stride, bias_stride, bias_expert;  // in elements
    uint32_t activation, gated;
    void* workspace;
    uint64_t workspace_bytes;
};
// Tiles that a launch has to hold for any offsets: every expert may end in a tile that is not full.
inline uint64_t most_tiles(const MatmulArgs& a, uint32_t size_log2) {
    const uint64_t full = (static_cast<uint64_t>(a.positions) + (1u << size_log2) - 1u) >> size_log2;
    return a.offsets ? full + (a.experts < a.positions ? a.experts : a.positions) : full;
}

hipError_t launch_matmul_general(hipStream_t s, const MatmulArgs& a);

struct RouteArgs {
    const char* logits;
    int dtype;
    uint64_t stride_token, stride_expert;
    float* weights;
    int32_t *experts, *offsets, *rows, *slots;
    uint32_t tokens, num_experts, chosen;
    uint32_t sigmoid, normalize;
    uint32_t vector_logits;  // a lane's logits are contiguous and on a boundary of their own size, up to 16 bytes
    void* workspace;
};
uint64_t route_workspace_bytes(uint64_t tokens, uint64_t experts, uint64_t chosen);
hipError_t launch_route(hipStream_t s, const RouteArgs& a);

struct CombineArgs {
    const char* h;
    const int32_t* slots;
    const float* weights;
    const char* residual;
    char* y;
    int h_dtype, y_dtype;
    uint32_t tokens, chosen, cols, positions;
    uint64_t h_stride, y_stride, residual_stride;
};
hipError_t launch_combine(hipStream_t s, const CombineArgs& a);

}  // namespace cq
