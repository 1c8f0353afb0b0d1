// The results of several splits of the keys, joined: y = sum_s w_s part_s / sum_s w_s with w_s = sum_s exp2(largest score_s - the largest of all).
//
// A wave a row (token, head): a lane holds largest score and sum of its split, then four entries of the result, splits behind one another with eight loads
// on their way.  Of few rows, bound by a launch and two rounds from L2, the first eight are asked for together with the sums (kEarly); many are bound by the parts'
// bytes, and only what has a share is read.  A row that is whole in one part (kWhole) is in y already.
#include <hip/hip_runtime.h>

#include "cq_attention_tiles.hpp"

namespace cq {
namespace {

constexpr uint32_t kAtOnce = 8;      // parts on their way
constexpr uint64_t kFewRows = 4096;  // a wave each for half of what the GPU holds at once

// The shares of a row's parts, a lane each.
struct Joined {
    float share;
    uint32_t used;  // parts up to the last that has a share
    bool whole;     // in y already
    __device__ __forceinline__ Joined(const AttentionArgs& a, const Split& split, uint32_t row, uint32_t lane) {
        const float* const stats = split.stats + 2ull * row * split.splits;
        const bool mine = lane < split.splits;
        const float top = mine ? stats[2 * lane] : -INFINITY, sum = mine ? stats[2 * lane + 1] : 0.0f;
        whole = __builtin_amdgcn_readfirstlane(f32_bits(sum)) == f32_bits(kWhole);
        float most = top;
#pragma unroll
        for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        // A part that has seen no key has a sum of zero; one whose scores are all not numbers has a sum that is none over a largest score of -infinity
        const float weight = sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f(top == -INFINITY ? 0.0f : top - most);
        float all = weight;
#pragma unroll
        for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d, 64);
        share = all == 0.0f ? 0.0f : weight / all;
        used = 64u - static_cast<uint32_t>(__builtin_clzll(__builtin_amdgcn_ballot_w64(mine && share != 0.0f) | 1ull));
    }
    __device__ __forceinline__ float share_of(uint32_t part) const { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(f32_bits(share), min(part, 63u))); }
};

// Whether a token is anybody's: of one that is not, the parts are not numbers of ours and y stays as it is.
__device__ __forceinline__ bool of_a_sequence(const AttentionArgs& a, uint32_t token) {
    const Sequence s = sequence_of(a, last_at_or_below(a.seqs, token, [&](uint32_t i) { return static_cast<uint64_t>(max(a.offsets[i], 0)); }));
    return token >= s.first && token < s.last;
}

__device__ __forceinline__ void store_row(const AttentionArgs& a, uint32_t token, uint32_t head, uint32_t lane, uint32_t d, f32x4 v) {
    if (lane * 4u >= a.cache.dim) return;
    const u32x2 w = a.dtype == CQ_BF16 ? u32x2{pair_of<true>(v[0], v[1]), pair_of<true>(v[2], v[3])} : u32x2{pair_of<false>(v[0], v[1]), pair_of<false>(v[2], v[3])};
    *reinterpret_cast<u32x2*>(a.y + (token * a.y_token + head * a.y_head + d) * 2u) = w;
}

template <bool kEarly>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, Split split, uint32_t row0) {
    const uint32_t lane = threadIdx.x & 63u, row = row0 + blockIdx.x * 4u + (threadIdx.x >> 6);
    if (row >= a.tokens * a.heads) return;
    const uint32_t token = row / a.heads, head = row % a.heads, d = min(lane * 4u, a.cache.dim - 4u);
    const float* const parts = split.parts + static_cast<uint64_t>(row) * split.splits * a.cache.dim + d;
    f32x4 of[kAtOnce];
    const auto load = [&](uint32_t p0, uint32_t last) {
#pragma unroll
        for (uint32_t p = 0; p < kAtOnce; p++) of[p] = *reinterpret_cast<const f32x4*>(parts + static_cast<uint64_t>(min(p0 + p, last)) * a.cache.dim);
    };
    if constexpr (kEarly) load(0, split.splits - 1u);
    // every lane stays until the end, as the others read its share
    const Joined joined(a, split, row, lane);
    if (joined.whole) return;
    f32x4 v = {};
    for (uint32_t p0 = 0; p0 < joined.used; p0 += kAtOnce) {
        if (!kEarly || p0 != 0) load(p0, joined.used - 1u);
#pragma unroll
        for (uint32_t p = 0; p < kAtOnce; p++) {
            const float by = joined.share_of(p0 + p);
            if (p0 + p < joined.used && by != 0.0f) v = __builtin_elementwise_fma(of[p], f32x4{by, by, by, by}, v);  // a part without a share may hold anything
        }
    }
    if (of_a_sequence(a, token)) store_row(a, token, head, lane, d, v);
}

// The same with four waves a row, every fourth part a wave's, all of them on their way at once: for few rows of many parts (64 rows of 64 parts: 7.6 us with a
// wave a row, 4.5 with four; 2048 rows of 7: 4.7 and 9.6).
constexpr uint32_t kWide = 4;
__global__ __launch_bounds__(64 * kWide) void attention_join_wide_kernel(AttentionArgs a, Split split) {
    __shared__ f32x4 handed[kWide - 1][64];
    constexpr uint32_t kMine = 64 / kWide;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x, token = row / a.heads, head = row % a.heads;
    const uint32_t d = min(lane * 4u, a.cache.dim - 4u);
    const float* const parts = split.parts + static_cast<uint64_t>(row) * split.splits * a.cache.dim + d;
    f32x4 of[kMine];
#pragma unroll
    for (uint32_t p = 0; p < kMine; p++) of[p] = *reinterpret_cast<const f32x4*>(parts + static_cast<uint64_t>(min(p * kWide + wave, split.splits - 1u)) * a.cache.dim);
    const Joined joined(a, split, row, lane);
    f32x4 v = {};
#pragma unroll
    for (uint32_t p = 0; p < kMine; p++) {
        const float by = joined.share_of(p * kWide + wave);
        if (p * kWide + wave < joined.used && by != 0.0f) v = __builtin_elementwise_fma(of[p], f32x4{by, by, by, by}, v);
    }
    if (wave != 0) handed[wave - 1u][lane] = v;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (uint32_t w = 0; w < kWide - 1; w++) v += handed[w][lane];
    if (!joined.whole && of_a_sequence(a, token)) store_row(a, token, head, lane, d, v);
}

}  // namespace

hipError_t launch_attention_join(hipStream_t s, const AttentionArgs& a, const Split& split) {
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.heads;
    if (rows <= kFewRows / kWide && split.splits > 2 * kAtOnce) {
        hipLaunchKernelGGL(attention_join_wide_kernel, dim3(static_cast<uint32_t>(rows)), dim3(64 * kWide), 0, s, a, split);
        return hipGetLastError();
    }
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
