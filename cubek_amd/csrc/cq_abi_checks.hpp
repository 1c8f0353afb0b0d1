// Checks of arguments that the C ABIs of products (cq_matmul_abi.hip) and attention (cq_attention_abi.hip) share.
#pragma once

#include <stdint.h>

#include "../../include/cubek_quant.h"

namespace {

constexpr uint64_t kMostExtent = 0x7fffffffull;  // rows, columns, positions and tokens are 32-bit numbers in the kernels

uint32_t dtype_size(int dtype) { return dtype == CQ_F32 ? 4u : 2u; }
bool valid_dtype(int dtype) { return dtype == CQ_F32 || dtype == CQ_F16 || dtype == CQ_BF16; }
bool has_elements(const cq_tensor* t) {
    for (uint32_t d = 0; d < t->rank; d++)
        if (t->shape[d] == 0) return false;
    return true;
}

// A tensor without elements may come without an address.
bool tensor_ok(const cq_tensor* t) {
    return t && t->shape && t->strides && t->rank >= 1 && t->rank <= CQ_MAX_RANK && (t->ptr || !has_elements(t));
}
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

bool is_contiguous(const cq_tensor* t) {
    if (!has_elements(t)) return true;
    uint64_t expect = 1;
    for (int d = static_cast<int>(t->rank) - 1; d >= 0; d--) {
        if (t->shape[d] != 1 && t->strides[d] != expect) return false;
        expect *= t->shape[d];
    }
    return true;
}

// The stride of dimension d; one entry counts as 0, whatever the tensor says, and keeps no product from a kernel by its alignment.
uint64_t stride_of(const cq_tensor* t, uint32_t d) { return t->shape[d] > 1 ? t->strides[d] : 0; }

cq_status check_scheme(const cq_scheme* s) {
    if (!s) return CQ_ERR_INVALID_ARGUMENT;
    if (cq_value_size_bits(s->value) == 0 || s->param > CQ_PARAM_BF16 || s->store > CQ_STORE_NATIVE || s->level > CQ_LEVEL_BLOCK || s->reserved != 0)
        return CQ_ERR_INVALID_ARGUMENT;
    if (s->mode != CQ_MODE_SYMMETRIC) return CQ_ERR_UNSUPPORTED_SCHEME;
    if (s->level == CQ_LEVEL_BLOCK) {
        if (s->block_rank < 1 || s->block_rank > CQ_MAX_BLOCK_DIMS) return CQ_ERR_INVALID_ARGUMENT;
        for (uint32_t i = 0; i < s->block_rank; i++)
            if (s->block[i] == 0) return CQ_ERR_INVALID_ARGUMENT;
    }
    // the native store holds i8, e4m3, e5m2 bytes or e2m1 pairs (crates/cubek-quant/src/quantize.rs:196-219)
    if (s->store == CQ_STORE_NATIVE && (s->value == CQ_VALUE_Q4F || s->value == CQ_VALUE_Q4S || s->value == CQ_VALUE_Q2F || s->value == CQ_VALUE_Q2S))
        return CQ_ERR_UNSUPPORTED_SCHEME;
    return CQ_OK;
}

// An i32 tensor [n], contiguous.
cq_status read_indexes(const cq_tensor* t, uint64_t n, const int32_t** out) {
    if (!tensor_ok(t) || !aligned(t->ptr, 4)) return CQ_ERR_INVALID_ARGUMENT;
    if (t->rank != 1 || t->elem_size != 4 || t->shape[0] != n) return CQ_ERR_SHAPE_MISMATCH;
    if (!is_contiguous(t)) return CQ_ERR_NON_CONTIGUOUS;
    *out = static_cast<const int32_t*>(t->ptr);
    return CQ_OK;
}

}  // namespace
