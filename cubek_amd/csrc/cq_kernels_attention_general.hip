// Attention over pages for everything that the matrix cores do not take: f32 queries, heads of any size up to 512, any block, page size and
// alignment.
//
// A workgroup takes one query.  Its four waves take 64 keys at a time in turn: a lane a key for the scores (its row against the query in LDS),
// a lane eight entries of the result for the values; running maximum, sum and result are each wave's own and meet in LDS at the end.  Everything is
// f32.  Bound by vector instructions, one value of the cache an element load, a conversion and an FMA: nothing is shared between queries.
#include <hip/hip_runtime.h>

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

constexpr uint32_t kEntries = CQ_MAX_HEAD_DIM / 64;

__global__ __launch_bounds__(256) void attention_general_kernel(AttentionArgs a, uint32_t token0) {
    __shared__ float query[CQ_MAX_HEAD_DIM], weights[4][64], part[4][CQ_MAX_HEAD_DIM], part_max[4], part_sum[4];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t token = token0 + blockIdx.x, head = blockIdx.y, kv_head = head / a.group, dim = a.cache.dim;
    const Sequence s = sequence_of(a, last_at_or_below(a.seqs, token, [&](uint32_t i) { return static_cast<int64_t>(a.offsets[i]) <= 0 ? 0ull : static_cast<uint64_t>(a.offsets[i]); }));
    if (token < s.first || token >= s.last) return;
    const int32_t position = s.position + static_cast<int32_t>(token - s.first);
    const Seen seen = seen_from(a, s, position);
    for (uint32_t d = threadIdx.x; d < dim; d += 256) query[d] = load_dtype(a.dtype, a.q, token * a.q_token + head * a.q_head + d);
    __syncthreads();

    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    float top = -INFINITY, sum = 0.0f, acc[kEntries] = {};
    for (int64_t base = seen.low + static_cast<int64_t>(wave) * 64; base <= seen.high; base += 256) {
        const int32_t here = static_cast<int32_t>(min(static_cast<int64_t>(64), seen.high - base + 1));
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
        weights[wave][lane] = weight;
#pragma unroll
        for (uint32_t i = 0; i < kEntries; i++) acc[i] *= shrink;
        __builtin_amdgcn_wave_barrier();
        for (int32_t k = 0; k < here; k++) {
            const uint32_t j = static_cast<uint32_t>(base) + static_cast<uint32_t>(k);
            const uint64_t page = page_of(a, s, j / a.cache.page_size), place = j % a.cache.page_size;
            const char* const row = row_of(a.cache.values, page, place, kv_head);
            const float w = weights[wave][k];
#pragma unroll
            for (uint32_t i = 0; i < kEntries; i++) {
                const uint32_t d = i * 64u + lane;
                if (d < dim) acc[i] = __builtin_fmaf(w, code_at(a.cache, a.dtype, row, d) * scale_at(a.cache, a.cache.values, page, place, kv_head, d / a.cache.block), acc[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) part_max[wave] = top, part_sum[wave] = sum;
#pragma unroll
    for (uint32_t i = 0; i < kEntries; i++) part[wave][i * 64u + lane] = acc[i];
    __syncthreads();
    const float most = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
    float share[4], total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        share[w] = part_max[w] == -INFINITY ? 0.0f : expf(part_max[w] - most);
        total = __builtin_fmaf(part_sum[w], share[w], total);
    }
    for (uint32_t d = threadIdx.x; d < dim; d += 256) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++)
            if (part_max[w] != -INFINITY) v = __builtin_fmaf(part[w][d], share[w], v);
        store_dtype(a.dtype, a.y, token * a.y_token + head * a.y_head + d, total != 0.0f ? v / total : 0.0f);
    }
}

}  // namespace

hipError_t launch_attention_general(hipStream_t s, const AttentionArgs& a) {
    constexpr uint32_t kPiece = static_cast<uint32_t>(kLaunchThreads / 256 - 1);
    for (uint64_t token = 0; token < a.tokens; token += kPiece) {
        const uint32_t n = a.tokens - token < kPiece ? static_cast<uint32_t>(a.tokens - token) : kPiece;
        hipLaunchKernelGGL(attention_general_kernel, dim3(n, a.heads), dim3(256), 0, s, a, static_cast<uint32_t>(token));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cq
