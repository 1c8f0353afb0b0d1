/* cubek_matmul.h — C ABI of libcubek_matmul_hip.so: products of many tokens with quantized weights on MI355X (gfx950), the same
 * grouped by expert, and the routing around them.
 *
 * It stands beside cubek_quant.h, whose tensors, schemes and status codes it uses: cq_quantize makes the weights,
 * cq_gemv_quantized multiplies up to sixteen vectors with them, the products here take any number of tokens and what stands behind a
 * product (bias, activation, gate, residual) in the same launches.  The reference multiplies quantized operands in its matmul crate
 * (MatmulInputHandle::Quantized, crates/cubek-matmul/src/base.rs:309-317), without an epilogue and without groups.
 *
 * As everywhere in this library: device pointers, strides in elements, the caller owns every buffer, calls only enqueue kernels on
 * the caller's stream (no allocation, synchronisation or memset: they can be captured into a HIP graph) and validate before
 * they launch.  Results do not depend on anything but the arguments: no atomics on floats, no order that changes from call to call. */
#ifndef CUBEK_MATMUL_H
#define CUBEK_MATMUL_H

#include "cubek_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum cq_activation {
    CQ_ACT_IDENTITY = 0,
    CQ_ACT_RELU = 1,      /* max(v, 0), NaN stays NaN                                    */
    CQ_ACT_SILU = 2,      /* v / (1 + exp(-v))                                           */
    CQ_ACT_GELU = 3,      /* v * (1 + erf(v / sqrt 2)) / 2                               */
    CQ_ACT_GELU_TANH = 4  /* v * (1 + tanh(sqrt(2 / pi) (v + 0.044715 v^3))) / 2         */
} cq_activation;

/* What stands behind a product, in f32 before the one rounding to the type of y:
 *   v[n] = sum_k x[k] * W[n, k] + bias[n]
 *   y[n] = act(v[n]) + residual[n]                  plain: y has as many columns as W has rows
 *   y[n] = act(v[n]) * v[N + n] + residual[n]       gated: W has 2 N rows, the gate's in front of the others
 *   bias     : NULL or [rows of W] ([experts, rows of W] for cq_experts_quantized), typed like x or f32 (by its elem_size), any strides
 *   residual : NULL or the shape of y, typed like y, its last dimension contiguous; may be y itself
 * Every field not used is 0. */
typedef struct cq_epilogue {
    uint32_t activation; /* cq_activation */
    uint32_t gated;      /* 0 or 1 */
    const cq_tensor* bias;
    const cq_tensor* residual;
} cq_epilogue;

/* y = epilogue(x * dequantize(W)^T) for any number of tokens.
 *   values : U32-store [rows, cols / num_quants] or native-store [rows, cols] ([rows, cols / 2] for e2m1), rows may be pitched
 *   params : scales typed scheme->param, [1] per tensor or [rows / block_rows, cols / block_cols] for blocks over the last one or
 *            two dimensions, any strides
 *   x      : [tokens, cols] typed `dtype` (or [cols]: one token), its last dimension contiguous; x and params start on a multiple of their
 *            elements' size (CQ_ERR_INVALID_ARGUMENT)
 *   y      : [tokens, N] typed `y_dtype` (or [N]), its last dimension contiguous; N as in cq_epilogue
 *   epilogue : NULL for the bare product
 *   workspace : optional device scratch of cq_matmul_workspace_bytes() bytes, 16-byte aligned; lets products of few tokens and
 *            few rows spread their columns over the GPU.  Without it they are right, and slower.
 * Every weight enters as the value cq_dequantize would store for `dtype`, F(F(scale) * F(code)); sums are f32, their order
 * depends on the shapes, on strides and alignment, and on whether the workspace has the bytes that were asked for: not on the values.  No tokens: nothing is launched.  No columns: sums of nothing. */
cq_status cq_matmul_quantized(cq_stream_t stream, const cq_tensor* values, const cq_tensor* params, const cq_scheme* scheme,
                              const cq_tensor* x, const cq_tensor* y, cq_dtype dtype, cq_dtype y_dtype,
                              const cq_epilogue* epilogue, void* workspace, size_t workspace_bytes);
size_t cq_matmul_workspace_bytes(const cq_tensor* values, const cq_scheme* scheme, const cq_tensor* x, cq_dtype dtype,
                                 const cq_epilogue* epilogue);

/* The same product with a weight of its own for every group of rows of y ("positions"): y[p] = epilogue(x[rows[p]] *
 * dequantize(W[e])^T) for the positions p of expert e, offsets[e] <= p < offsets[e + 1].
 *   values  : [experts, rows, ...], params [experts, rows / block_rows, cols / block_cols] or [1]; otherwise as above
 *   x       : [tokens, cols]
 *   offsets : i32 [experts + 1] in device memory, contiguous, ascending from 0 to at most the positions.  What they hold is not known to the
 *             host: values outside are taken as the nearest inside, and positions of no expert are left unwritten.
 *   rows    : i32 [positions] in device memory, contiguous, or NULL: position p takes row p of x, which then has as many rows as y.  A row
 *             outside of x is taken as the nearest inside.
 *   y       : [positions, N]
 *   workspace : as above, of cq_experts_workspace_bytes() bytes */
cq_status cq_experts_quantized(cq_stream_t stream, const cq_tensor* values, const cq_tensor* params, const cq_scheme* scheme,
                               const cq_tensor* x, const cq_tensor* offsets, const cq_tensor* rows, const cq_tensor* y,
                               cq_dtype dtype, cq_dtype y_dtype, const cq_epilogue* epilogue, void* workspace,
                               size_t workspace_bytes);
size_t cq_experts_workspace_bytes(const cq_tensor* values, const cq_scheme* scheme, const cq_tensor* y, cq_dtype dtype,
                                  const cq_epilogue* epilogue);

typedef enum cq_score {
    CQ_SCORE_SOFTMAX = 0, /* over all experts of the token */
    CQ_SCORE_SIGMOID = 1
} cq_score;

#define CQ_MAX_EXPERTS 1024
#define CQ_MAX_CHOSEN 64

/* Each token's experts by its logits, and the positions of the pairs (token, choice) sorted by expert, tokens of an expert
 * ascending: what cq_experts_quantized and cq_combine take.
 *   logits  : [tokens, experts] typed `dtype`, any strides; at most CQ_MAX_EXPERTS
 *   weights : f32 [tokens, chosen], experts : i32 [tokens, chosen], by falling logit; equal ones (+0 and -0 too) by rising
 *             expert.  NaN counts as -infinity.  1 <= chosen <= min(experts, CQ_MAX_CHOSEN).
 *   offsets : i32 [experts + 1]; rows : i32 [tokens * chosen], the token of each position; slots : i32 [tokens, chosen], the position of
 *             each pair.  All outputs contiguous.
 *   normalize : a token's weights are divided by their sum (0 stays 0), also where sigmoids are too small for f32 themselves: down to logits of
 *             -709.78, past which, as masks of a type's lowest value are, they count 0.  A token whose logits are all -infinity gets weights of 0.
 *   workspace : cq_route_workspace_bytes() bytes of device memory, 16-byte aligned (0 for few tokens)
 * tokens <= 2^28 - 64 and tokens * chosen < 2^31.  No tokens: the offsets are set to 0. */
cq_status cq_route(cq_stream_t stream, const cq_tensor* logits, const cq_tensor* weights, const cq_tensor* experts,
                   const cq_tensor* offsets, const cq_tensor* rows, const cq_tensor* slots, cq_dtype dtype, cq_score score,
                   uint32_t normalize, void* workspace, size_t workspace_bytes);
size_t cq_route_workspace_bytes(uint64_t tokens, uint64_t experts, uint64_t chosen);

/* y[t] = residual[t] + sum_j weights[t, j] * h[slots[t, j]], in f32 from j = 0 on, rounded once.
 *   h : [positions, cols] typed `h_dtype`; slots i32, weights f32 [tokens, chosen], contiguous; y, residual (NULL: none; may be y)
 *   [tokens, cols] typed `y_dtype`; last dimensions contiguous.  A slot outside of h adds nothing, whatever its weight. */
cq_status cq_combine(cq_stream_t stream, const cq_tensor* h, const cq_tensor* slots, const cq_tensor* weights,
                     const cq_tensor* residual, const cq_tensor* y, cq_dtype h_dtype, cq_dtype y_dtype);

/* hipError_t of the most recent failed HIP call of this library on the calling thread (0 if none). */
int cq_matmul_last_hip_error(void);

#ifdef __cplusplus
}
#endif
#endif /* CUBEK_MATMUL_H */
