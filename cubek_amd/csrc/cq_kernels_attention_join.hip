// The results of several splits of the keys, joined: y = sum_s w_s part_s / sum_s w_s with w_s = sum_s exp2(largest score_s - the largest of all).
//
// A wave a row (token, head): a lane holds largest score and sum of its split, then four entries of the result, splits behind one another with eight loads
// on their way.  Bound by a launch and two rounds from L2 where rows are few; the parts are then asked for together with the sums (kEarly).  Of many rows, bound
// by the parts' bytes, only what has a share is read.  A row that is whole in one part (sum below zero) is in y already.
#include <hip/hip_runtime.h>

#include "cq_attention_tiles.hpp"

namespace cq {
namespace {

constexpr uint32_t kAtOnce = 8;      // parts on their way
constexpr uint64_t kFewRows = 4096;  // a wave each for half of what the GPU holds at once

template <bool kEarly>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, Split split, uint32_t row0) {
    const uint32_t lane = threadIdx.x & 63u, row = row0 + blockIdx.x * 4u + (threadIdx.x >> 6);
    if (row >= a.tokens * a.heads) return;
    const uint32_t token = row / a.heads, head = row % a.heads;
    const auto whole = [](float sum) { return __builtin_bit_cast(int32_t, __builtin_amdgcn_readfirstlane(f32_bits(sum))) == static_cast<int32_t>(f32_bits(kWhole)); };
    // every lane stays, as the others read its share
    const uint32_t d = min(lane * 4u, a.cache.dim - 4u);
    const float* const parts = split.parts + static_cast<uint64_t>(row) * split.splits * a.cache.dim + d;
    f32x4 of[kAtOnce];
    uint32_t most_part = split.splits - 1u;
    const auto load = [&](uint32_t p0) {
#pragma unroll
        for (uint32_t p = 0; p < kAtOnce; p++) of[p] = *reinterpret_cast<const f32x4*>(parts + static_cast<uint64_t>(min(p0 + p, most_part)) * a.cache.dim);
    };
    if constexpr (kEarly) load(0);
    const float* const stats = split.stats + 2ull * row * split.splits;
    const bool mine = lane < split.splits;
    const float top = mine ? stats[2 * lane] : -INFINITY, sum = mine ? stats[2 * lane + 1] : 0.0f;
    if constexpr (!kEarly)
        if (whole(sum)) return;
    // whether the token is anybody's, looked up while the parts are on their way: of one that is not, they are not numbers of ours
    const Sequence s = sequence_of(a, last_at_or_below(a.seqs, token, [&](uint32_t i) { return static_cast<uint64_t>(max(a.offsets[i], 0)); }));
    float most = top;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
    const float weight = top == -INFINITY ? 0.0f : sum * __builtin_amdgcn_exp2f(top - most);
    float all = weight;
#pragma unroll
    for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d, 64);
    const float share = all == 0.0f ? 0.0f : weight / all;
    const uint32_t used = 64u - static_cast<uint32_t>(__builtin_clzll(__builtin_amdgcn_ballot_w64(mine && share != 0.0f) | 1ull));  // parts up to the last that has a share
    if constexpr (!kEarly) most_part = used - 1u, load(0);
    f32x4 v = {};
    for (uint32_t p0 = 0;;) {
#pragma unroll
        for (uint32_t p = 0; p < kAtOnce; p++) {
            const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(f32_bits(share), min(p0 + p, 63u)));
            if (p0 + p < used && by != 0.0f) v = __builtin_elementwise_fma(of[p], f32x4{by, by, by, by}, v);  // a part without keys may hold anything
        }
        p0 += kAtOnce;
        if (p0 >= used) break;
        load(p0);
    }
    if (token < s.first || token >= s.last || lane * 4u >= a.cache.dim || (kEarly && whole(sum))) return;
    const uint64_t at = (token * a.y_token + head * a.y_head + d) * 2u;
    const u32x2 w = a.dtype == CQ_BF16 ? u32x2{pair_of<true>(v[0], v[1]), pair_of<true>(v[2], v[3])} : u32x2{pair_of<false>(v[0], v[1]), pair_of<false>(v[2], v[3])};
    *reinterpret_cast<u32x2*>(a.y + at) = w;
}

}  // namespace

hipError_t launch_attention_join(hipStream_t s, const AttentionArgs& a, const Split& split) {
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.heads;
    constexpr uint64_t kPiece = (kLaunchThreads / 256 - 1) * 4;
    for (uint64_t row = 0; row < rows; row += kPiece) {
        const uint64_t n = rows - row < kPiece ? rows - row : kPiece;
        const dim3 grid(static_cast<uint32_t>((n + 3) / 4));
        if (rows <= kFewRows)
            hipLaunchKernelGGL(attention_join_kernel<true>, grid, dim3(256), 0, s, a, split, static_cast<uint32_t>(row));
        else
            hipLaunchKernelGGL(attention_join_kernel<false>, grid, dim3(256), 0, s, a, split, static_cast<uint32_t>(row));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cq
