// One query against some keys of its sequence by a wave, in f32, whatever the cache holds: what attention_general_kernel is made of, and the kernels on
// the matrix cores fall back to where entries that are not numbers lie among keys that not every row sees.
#pragma once

#include "cq_attention_internal.hpp"
#include "cq_device.hpp"

namespace cq {
namespace {

// Entry d of a row: its code as a number (of floats, the entry).
__device__ __forceinline__ float code_at(const CacheArgs& c, int dtype, const char* row, uint32_t d) {
    switch (c.code) {
        case kCacheInt8: return static_cast<float>(reinterpret_cast<const int8_t*>(row)[d]);
        case kCacheE4M3: return __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(row[d]), 0);
        case kCacheE5M2: return __builtin_amdgcn_cvt_f32_bf8(static_cast<uint8_t>(row[d]), 0);
        case kCacheFloat: return load_dtype(dtype, row, d);
        default: {
            const uint32_t nibble = static_cast<uint8_t>(row[d / 2u]) >> (4u * (d & 1u)) & 15u;
            if (c.code == kCacheInt4) return static_cast<float>(static_cast<int32_t>(nibble ^ 8u) - 8);
            const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(nibble, 1.0f, 0);
            return v[0];
        }
    }
}

__device__ __forceinline__ const char* row_of(const CacheSide& side, uint64_t page, uint64_t place, uint32_t head) {
    return side.base + page * side.page + head * side.head + place * side.slot;
}
__device__ __forceinline__ float scale_at(const CacheArgs& c, const CacheSide& side, uint64_t page, uint64_t place, uint32_t head, uint32_t block) {
    if (c.code == kCacheFloat) return 1.0f;
    return load_dtype(c.param_dtype, side.scales, page * side.scale_page + head * side.scale_head + place * side.scale_slot + block * side.scale_block);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// The keys first, first + stride ... (64 of them at a time) up to `last`: a lane a key for the scores, with `query` in LDS; a lane the entries lane, lane + 64
// ... for the values, with `weights` (64 floats of the wave) in LDS.
template <uint32_t kEntries>
__device__ __forceinline__ void attend_row(const AttentionArgs& a, const Sequence& s, uint32_t kv_head, int32_t position, float slope, const float* query,
                                           float* weights, int64_t first, int64_t stride, int64_t last, float* top_out, float* sum_out, float* acc) {
    const uint32_t lane = threadIdx.x & 63u, dim = a.cache.dim;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kEntries; i++) acc[i] = 0.0f;
    for (int64_t base = first; base <= last; base += stride) {
        const int32_t here = static_cast<int32_t>(min(static_cast<int64_t>(64), last - base + 1));
        float t = -INFINITY;
        if (static_cast<int32_t>(lane) < here) {
            const uint32_t j = static_cast<uint32_t>(base) + lane;
            const uint64_t page = page_of(a, s, j / a.cache.page_size), place = j % a.cache.page_size;
            const char* const row = row_of(a.cache.keys, page, place, kv_head);
            t = 0.0f;
            for (uint32_t d0 = 0, b = 0; d0 < dim; d0 += a.cache.block, b++) {
                float of_block = 0.0f;
                for (uint32_t d = d0; d < d0 + a.cache.block; d++) of_block = __builtin_fmaf(query[d], code_at(a.cache, a.dtype, row, d), of_block);
                t = __builtin_fmaf(of_block, scale_at(a.cache, a.cache.keys, page, place, kv_head, b), t);
            }
            t *= a.scale;
            if (a.cap > 0.0f) t = a.cap * tanhf(t / a.cap);
            t -= slope * static_cast<float>(abs(position - static_cast<int32_t>(j)));
        }
        const float before = top;
        top = fmaxf(top, wave_max(t));
        const float zero = top == -INFINITY ? 0.0f : top;  // nothing but -infinity so far
        const float weight = static_cast<int32_t>(lane) < here ? expf(t - zero) : 0.0f, shrink = expf(before - zero);
        sum = __builtin_fmaf(sum, shrink, wave_sum(weight));
        weights[lane] = weight;
#pragma unroll
        for (uint32_t i = 0; i < kEntries; i++) acc[i] *= shrink;
        __builtin_amdgcn_wave_barrier();
        for (int32_t k = 0; k < here; k++) {
            const uint32_t j = static_cast<uint32_t>(base) + static_cast<uint32_t>(k);
            const uint64_t page = page_of(a, s, j / a.cache.page_size), place = j % a.cache.page_size;
            const char* const row = row_of(a.cache.values, page, place, kv_head);
            const float w = weights[k];
#pragma unroll
            for (uint32_t i = 0; i < kEntries; i++) {
                const uint32_t d = i * 64u + lane;
                if (d < dim) acc[i] = __builtin_fmaf(w, code_at(a.cache, a.dtype, row, d) * scale_at(a.cache, a.cache.values, page, place, kv_head, d / a.cache.block), acc[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    *top_out = top, *sum_out = sum;
}

}  // namespace
}  // namespace cq
