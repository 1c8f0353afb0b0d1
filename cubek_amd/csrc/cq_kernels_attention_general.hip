// Attention over pages for everything that the matrix cores do not take: f32 queries, heads of any size up to 512, any block, page size and
// alignment.
//
// A workgroup takes one query.  Its four waves take 64 keys at a time in turn: a lane a key for the scores (its row against the query in LDS),
// a lane eight entries of the result for the values; running maximum, sum and result are each wave's own and meet in LDS at the end.  Everything is
// f32.  Bound by vector instructions, one value of the cache an element load, a conversion and an FMA: nothing is shared between queries (64 single tokens over
// 257 to 8191 keys of 8 heads of i8, four queries a head: 10.4 ms, where the matrix cores take 0.12).
#include <hip/hip_runtime.h>

#include "cq_attention_rows.hpp"

namespace cq {
namespace {

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

    float top, sum, acc[kEntries];
    attend_row<kEntries>(a, s, kv_head, position, a.slopes ? a.slopes[head] : 0.0f, query, weights[wave], seen.low + static_cast<int64_t>(wave) * 64, 256, seen.high, &top, &sum, acc);
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
