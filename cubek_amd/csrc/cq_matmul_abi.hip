// C ABI of libcubek_matmul_hip.so (include/cubek_matmul.h): argument checks, the choice of a kernel, launches.
#include "cq_abi_checks.hpp"
#include "cq_matmul_tiles.hpp"

namespace {

thread_local int g_last_hip_error = 0;

cq_status hip_status(hipError_t e) {
    if (e == hipSuccess) return CQ_OK;
    g_last_hip_error = static_cast<int>(e);
    return CQ_ERR_HIP;
}

// The launchers read hipGetLastError() after each launch: an error that earlier HIP calls of the caller left would be taken for theirs.
void drop_stale_hip_error() { (void)hipGetLastError(); }

constexpr uint64_t kMostRouted = (cq::kLaunchThreads / 1024 - 1) * 64;  // tokens of a routing: 64 of them are a workgroup of 1024 threads

// The weights of a product: [rows, stored columns], or [experts, rows, stored columns].
cq_status read_weights(const cq_tensor* values, const cq_tensor* params, const cq_scheme* scheme, bool experts, cq::MatmulArgs* a) {
    const bool native = scheme->store == CQ_STORE_NATIVE;
    const uint32_t lead = experts ? 1u : 0u;
    if (!tensor_ok(values)) return CQ_ERR_INVALID_ARGUMENT;
    if (values->rank != 2 + lead || values->elem_size != (native ? 1u : 4u)) return CQ_ERR_SHAPE_MISMATCH;
    const uint64_t* const shape = values->shape + lead;
    a->bits = cq_value_size_bits(scheme->value);
    const uint64_t nq = cq_scheme_num_quants(scheme);
    if (shape[0] > kMostExtent || shape[1] > kMostExtent / nq || (experts && values->shape[0] > kMostExtent)) return CQ_ERR_TOO_LARGE;
    if (shape[1] > 1 && values->strides[lead + 1] != 1) return CQ_ERR_NON_CONTIGUOUS;
    a->words = static_cast<const char*>(values->ptr);
    a->wide = static_cast<uint32_t>(shape[0]);
    a->cols = static_cast<uint32_t>(shape[1] * nq);
    a->experts = experts ? static_cast<uint32_t>(values->shape[0]) : 1u;
    a->row_bytes = stride_of(values, lead) * values->elem_size;
    a->expert_bytes = experts ? stride_of(values, 0) * values->elem_size : 0;
    // i8 bytes are the 8-bit fields of the U32 store, and e2m1 nibbles lie alike in both stores
    if (scheme->value == CQ_VALUE_E2M1_OCP)
        a->native = 3;
    else if (native)
        a->native = scheme->value == CQ_VALUE_E4M3 ? 1u : scheme->value == CQ_VALUE_E5M2 ? 2u : scheme->value == CQ_VALUE_E2M1 ? 3u : 0u;
    a->param_dtype = scheme->param == CQ_PARAM_F32 ? CQ_F32 : (scheme->param == CQ_PARAM_F16 ? CQ_F16 : CQ_BF16);
    if (!params) return CQ_OK;  // a question about sizes
    if (!tensor_ok(params) || !aligned(params->ptr, dtype_size(a->param_dtype))) return CQ_ERR_INVALID_ARGUMENT;
    if (params->elem_size != dtype_size(a->param_dtype)) return CQ_ERR_SHAPE_MISMATCH;
    a->scales = static_cast<const char*>(params->ptr);
    if (scheme->level == CQ_LEVEL_TENSOR) {
        for (uint32_t d = 0; d < params->rank; d++)
            if (params->shape[d] < 1) return CQ_ERR_SHAPE_MISMATCH;
        return CQ_OK;
    }
    const uint32_t rank = scheme->block_rank;
    if (params->rank != values->rank || rank > values->rank) return CQ_ERR_SHAPE_MISMATCH;
    a->block_cols = scheme->block[rank - 1];
    a->block_rows = rank >= 2 ? scheme->block[rank - 2] : 1;
    if (rank == 3 && scheme->block[0] != 1) return CQ_ERR_SHAPE_MISMATCH;  // a scale belongs to one expert
    if (a->wide % a->block_rows || a->cols % a->block_cols || params->shape[lead] != a->wide / a->block_rows ||
        params->shape[lead + 1] != a->cols / a->block_cols || (experts && params->shape[0] != a->experts))
        return CQ_ERR_SHAPE_MISMATCH;
    a->scale_row = stride_of(params, lead);
    a->scale_col = stride_of(params, lead + 1);
    a->scale_expert = experts ? stride_of(params, 0) : 0;
    return CQ_OK;
}

cq_status read_epilogue(const cq_epilogue* epi, const cq_tensor* y, bool experts, cq::MatmulArgs* a) {
    a->out_cols = a->wide;
    if (!epi) return CQ_OK;
    if (epi->activation > CQ_ACT_GELU_TANH || epi->gated > 1) return CQ_ERR_INVALID_ARGUMENT;
    a->activation = epi->activation;
    a->gated = epi->gated;
    if (a->gated) {
        if (a->wide % 2) return CQ_ERR_SHAPE_MISMATCH;
        a->out_cols = a->wide / 2;
    }
    if (!y) return CQ_OK;  // a question about sizes
    if (const cq_tensor* b = epi->bias) {
        if (!tensor_ok(b)) return CQ_ERR_INVALID_ARGUMENT;
        const uint32_t lead = experts ? 1u : 0u;
        if (b->rank != 1 + lead || (experts && b->shape[0] != a->experts) || b->shape[lead] != a->wide ||
            (b->elem_size != 4 && b->elem_size != dtype_size(a->dtype)))
            return CQ_ERR_SHAPE_MISMATCH;
        a->bias = static_cast<const char*>(b->ptr);
        a->bias_dtype = b->elem_size == 4 ? CQ_F32 : a->dtype;
        a->bias_stride = b->strides[lead];
        a->bias_expert = experts ? b->strides[0] : 0;
    }
    if (const cq_tensor* r = epi->residual) {
        if (!tensor_ok(r)) return CQ_ERR_INVALID_ARGUMENT;
        if (r->rank != y->rank || r->elem_size != y->elem_size) return CQ_ERR_SHAPE_MISMATCH;
        for (uint32_t d = 0; d < y->rank; d++)
            if (r->shape[d] != y->shape[d]) return CQ_ERR_SHAPE_MISMATCH;
        if (r->shape[r->rank - 1] > 1 && r->strides[r->rank - 1] != 1) return CQ_ERR_NON_CONTIGUOUS;
        a->residual = static_cast<const char*>(r->ptr);
        a->residual_stride = r->rank == 2 ? r->strides[0] : 0;
    }
    return CQ_OK;
}

// x: [tokens, cols], y: [positions, out_cols]; or both without their first dimension
cq_status read_activations(const cq_tensor* x, const cq_tensor* y, cq_dtype dtype, cq_dtype y_dtype, bool experts, cq::MatmulArgs* a) {
    if (!tensor_ok(x) || !tensor_ok(y) || !aligned(x->ptr, dtype_size(dtype))) return CQ_ERR_INVALID_ARGUMENT;
    if (x->rank > 2 || y->rank != x->rank || (experts && x->rank != 2) || x->elem_size != dtype_size(dtype) || y->elem_size != dtype_size(y_dtype))
        return CQ_ERR_SHAPE_MISMATCH;
    const uint32_t last = x->rank - 1;
    const uint64_t tokens = last ? x->shape[0] : 1, positions = last ? y->shape[0] : 1;
    if (x->shape[last] != a->cols) return CQ_ERR_SHAPE_MISMATCH;
    if (tokens > kMostExtent || positions > kMostExtent) return CQ_ERR_TOO_LARGE;
    if ((a->cols > 1 && x->strides[last] != 1) || (y->shape[last] > 1 && y->strides[last] != 1)) return CQ_ERR_NON_CONTIGUOUS;
    a->x = static_cast<const char*>(x->ptr);
    a->y = static_cast<char*>(y->ptr);
    a->dtype = dtype;
    a->y_dtype = y_dtype;
    a->tokens = static_cast<uint32_t>(tokens);
    a->positions = static_cast<uint32_t>(positions);
    a->x_stride = last ? stride_of(x, 0) : 0;
    a->y_stride = last ? y->strides[0] : 0;
    return CQ_OK;
}

cq_status launch(cq_stream_t stream, cq::MatmulArgs& a) {
    return hip_status(cq::tiles_take(a) ? cq::launch_matmul_tiles(stream, a) : cq::launch_matmul_general(stream, a));
}

// What the product with these sizes would share its columns by, if it had the room; 0 where it does not share them.
size_t workspace_for(cq::MatmulArgs& a, cq_dtype dtype, const cq_scheme* scheme, uint64_t cols) {
    if (a.positions == 0 || a.out_cols == 0 || a.experts == 0 || cols != a.cols || a.positions > kMostExtent) return 0;
    a.dtype = dtype;
    if (scheme->level == CQ_LEVEL_BLOCK) a.block_cols = scheme->block[scheme->block_rank - 1], a.block_rows = 1;
    return cq::tiles_take(a) ? cq::room_of(a, cq::choice_within(a, ~0ull)) : 0;
}

}  // namespace

extern "C" {

size_t cq_matmul_workspace_bytes(const cq_tensor* values, const cq_scheme* scheme, const cq_tensor* x, cq_dtype dtype, const cq_epilogue* epilogue) {
    cq::MatmulArgs a{};
    if (check_scheme(scheme) != CQ_OK || read_weights(values, nullptr, scheme, false, &a) != CQ_OK || !tensor_ok(x) || !valid_dtype(dtype) ||
        read_epilogue(epilogue, nullptr, false, &a) != CQ_OK)
        return 0;
    a.positions = a.tokens = static_cast<uint32_t>(x->rank == 1 ? 1 : x->shape[0]);
    return workspace_for(a, dtype, scheme, x->shape[x->rank - 1]);
}

cq_status cq_matmul_quantized(cq_stream_t stream, const cq_tensor* values, const cq_tensor* params, const cq_scheme* scheme, const cq_tensor* x,
                              const cq_tensor* y, cq_dtype dtype, cq_dtype y_dtype, const cq_epilogue* epilogue, void* workspace,
                              size_t workspace_bytes) {
    cq::MatmulArgs a{};
    cq_status st = check_scheme(scheme);
    if (st != CQ_OK) return st;
    if (!valid_dtype(dtype) || !valid_dtype(y_dtype) || !params) return CQ_ERR_INVALID_ARGUMENT;
    if ((st = read_weights(values, params, scheme, false, &a)) != CQ_OK) return st;
    if ((st = read_activations(x, y, dtype, y_dtype, false, &a)) != CQ_OK) return st;
    if ((st = read_epilogue(epilogue, y, false, &a)) != CQ_OK) return st;
    if (a.positions != a.tokens || y->shape[y->rank - 1] != a.out_cols) return CQ_ERR_SHAPE_MISMATCH;
    if (a.positions == 0 || a.out_cols == 0) return CQ_OK;
    a.workspace = aligned(workspace, 16) ? workspace : nullptr;
    a.workspace_bytes = a.workspace ? workspace_bytes : 0;
    drop_stale_hip_error();
    return launch(stream, a);
}

size_t cq_experts_workspace_bytes(const cq_tensor* values, const cq_scheme* scheme, const cq_tensor* y, cq_dtype dtype, const cq_epilogue* epilogue) {
    cq::MatmulArgs a{};
    if (check_scheme(scheme) != CQ_OK || read_weights(values, nullptr, scheme, true, &a) != CQ_OK || !tensor_ok(y) || !valid_dtype(dtype) ||
        read_epilogue(epilogue, nullptr, true, &a) != CQ_OK || y->rank != 2)
        return 0;
    const int32_t offsets = 0;
    a.positions = a.tokens = static_cast<uint32_t>(y->shape[0]);
    a.offsets = &offsets;  // not read: only that there are some
    return workspace_for(a, dtype, scheme, a.cols);
}

cq_status cq_experts_quantized(cq_stream_t stream, const cq_tensor* values, const cq_tensor* params, const cq_scheme* scheme, const cq_tensor* x,
                               const cq_tensor* offsets, const cq_tensor* rows, const cq_tensor* y, cq_dtype dtype, cq_dtype y_dtype,
                               const cq_epilogue* epilogue, void* workspace, size_t workspace_bytes) {
    cq::MatmulArgs a{};
    cq_status st = check_scheme(scheme);
    if (st != CQ_OK) return st;
    if (!valid_dtype(dtype) || !valid_dtype(y_dtype) || !params) return CQ_ERR_INVALID_ARGUMENT;
    if ((st = read_weights(values, params, scheme, true, &a)) != CQ_OK) return st;
    if ((st = read_activations(x, y, dtype, y_dtype, true, &a)) != CQ_OK) return st;
    if ((st = read_epilogue(epilogue, y, true, &a)) != CQ_OK) return st;
    if (y->shape[1] != a.out_cols || (!rows && a.positions != a.tokens)) return CQ_ERR_SHAPE_MISMATCH;
    if ((st = read_indexes(offsets, a.experts + 1ull, &a.offsets)) != CQ_OK) return st;
    if (rows && (st = read_indexes(rows, a.positions, &a.row_of)) != CQ_OK) return st;
    if (a.positions == 0 || a.out_cols == 0 || a.experts == 0) return CQ_OK;
    if (a.tokens == 0) return CQ_ERR_SHAPE_MISMATCH;  // positions without a row to take
    a.workspace = aligned(workspace, 16) ? workspace : nullptr;
    a.workspace_bytes = a.workspace ? workspace_bytes : 0;
    drop_stale_hip_error();
    return launch(stream, a);
}

size_t cq_route_workspace_bytes(uint64_t tokens, uint64_t experts, uint64_t chosen) {
    if (experts > CQ_MAX_EXPERTS || chosen > CQ_MAX_CHOSEN || chosen > experts || tokens > kMostRouted) return 0;
    return cq::route_workspace_bytes(tokens, experts, chosen);
}

cq_status cq_route(cq_stream_t stream, const cq_tensor* logits, const cq_tensor* weights, const cq_tensor* experts, const cq_tensor* offsets,
                   const cq_tensor* rows, const cq_tensor* slots, cq_dtype dtype, cq_score score, uint32_t normalize, void* workspace,
                   size_t workspace_bytes) {
    if (!tensor_ok(logits) || !tensor_ok(weights) || !tensor_ok(experts) || !tensor_ok(offsets) || !tensor_ok(rows) || !tensor_ok(slots) ||
        !valid_dtype(dtype) || (score != CQ_SCORE_SOFTMAX && score != CQ_SCORE_SIGMOID) || normalize > 1)
        return CQ_ERR_INVALID_ARGUMENT;
    if (logits->rank != 2 || logits->elem_size != dtype_size(dtype) || weights->rank != 2) return CQ_ERR_SHAPE_MISMATCH;
    const uint64_t tokens = logits->shape[0], num = logits->shape[1], chosen = weights->shape[1];
    if (num > CQ_MAX_EXPERTS || chosen > CQ_MAX_CHOSEN || tokens > kMostRouted || tokens * chosen > kMostExtent) return CQ_ERR_TOO_LARGE;
    if (chosen < 1 || chosen > num) return CQ_ERR_INVALID_ARGUMENT;
    for (const cq_tensor* t : {weights, experts, slots}) {
        if (t->rank != 2 || t->elem_size != 4 || t->shape[0] != tokens || t->shape[1] != chosen) return CQ_ERR_SHAPE_MISMATCH;
        if (!is_contiguous(t)) return CQ_ERR_NON_CONTIGUOUS;
        if (!aligned(t->ptr, 4)) return CQ_ERR_INVALID_ARGUMENT;
    }
    cq::RouteArgs a{};
    const int32_t *to_offsets, *to_rows;
    cq_status st = read_indexes(offsets, num + 1, &to_offsets);
    if (st != CQ_OK || (st = read_indexes(rows, tokens * chosen, &to_rows)) != CQ_OK) return st;
    a.logits = static_cast<const char*>(logits->ptr);
    a.dtype = dtype;
    a.stride_token = logits->strides[0];
    a.stride_expert = logits->strides[1];
    a.weights = static_cast<float*>(weights->ptr);
    a.experts = static_cast<int32_t*>(experts->ptr);
    a.offsets = const_cast<int32_t*>(to_offsets);
    a.rows = const_cast<int32_t*>(to_rows);
    a.slots = static_cast<int32_t*>(slots->ptr);
    a.tokens = static_cast<uint32_t>(tokens);
    a.num_experts = static_cast<uint32_t>(num);
    a.chosen = static_cast<uint32_t>(chosen);
    a.sigmoid = score == CQ_SCORE_SIGMOID;
    a.normalize = normalize;
    a.workspace = workspace;
    if (const uint64_t need = cq::route_workspace_bytes(tokens, num, chosen))
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) return CQ_ERR_WORKSPACE_TOO_SMALL;
    drop_stale_hip_error();
    return hip_status(cq::launch_route(stream, a));
}

cq_status cq_combine(cq_stream_t stream, const cq_tensor* h, const cq_tensor* slots, const cq_tensor* weights, const cq_tensor* residual,
                     const cq_tensor* y, cq_dtype h_dtype, cq_dtype y_dtype) {
    if (!tensor_ok(h) || !tensor_ok(slots) || !tensor_ok(weights) || !tensor_ok(y) || (residual && !tensor_ok(residual)) || !valid_dtype(h_dtype) ||
        !valid_dtype(y_dtype))
        return CQ_ERR_INVALID_ARGUMENT;
    if (h->rank != 2 || slots->rank != 2 || weights->rank != 2 || y->rank != 2 || h->elem_size != dtype_size(h_dtype) ||
        y->elem_size != dtype_size(y_dtype) || slots->elem_size != 4 || weights->elem_size != 4 || h->shape[1] != y->shape[1])
        return CQ_ERR_SHAPE_MISMATCH;
    const uint64_t tokens = y->shape[0], chosen = slots->shape[1];
    if (slots->shape[0] != tokens || weights->shape[0] != tokens || weights->shape[1] != chosen) return CQ_ERR_SHAPE_MISMATCH;
    if (residual && (residual->rank != 2 || residual->elem_size != y->elem_size || residual->shape[0] != tokens || residual->shape[1] != y->shape[1]))
        return CQ_ERR_SHAPE_MISMATCH;
    if (tokens > kMostExtent || y->shape[1] > kMostExtent || h->shape[0] > kMostExtent || chosen > kMostExtent) return CQ_ERR_TOO_LARGE;
    for (const cq_tensor* t : {h, y, residual})
        if (t && t->shape[1] > 1 && t->strides[1] != 1) return CQ_ERR_NON_CONTIGUOUS;
    if (!is_contiguous(slots) || !is_contiguous(weights)) return CQ_ERR_NON_CONTIGUOUS;
    cq::CombineArgs a{};
    a.h = static_cast<const char*>(h->ptr);
    a.slots = static_cast<const int32_t*>(slots->ptr);
    a.weights = static_cast<const float*>(weights->ptr);
    a.residual = residual ? static_cast<const char*>(residual->ptr) : nullptr;
    a.y = static_cast<char*>(y->ptr);
    a.h_dtype = h_dtype;
    a.y_dtype = y_dtype;
    a.tokens = static_cast<uint32_t>(tokens);
    a.chosen = static_cast<uint32_t>(chosen);
    a.cols = static_cast<uint32_t>(y->shape[1]);
    a.positions = static_cast<uint32_t>(h->shape[0]);
    a.h_stride = h->strides[0];
    a.y_stride = y->strides[0];
    a.residual_stride = residual ? residual->strides[0] : 0;
    if (a.tokens == 0 || a.cols == 0) return CQ_OK;
    drop_stale_hip_error();
    return hip_status(cq::launch_combine(stream, a));
}

int cq_matmul_last_hip_error(void) { return g_last_hip_error; }

}  // extern "C"
