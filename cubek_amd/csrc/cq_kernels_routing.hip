// The choice of experts for every token, the positions of the pairs (token, choice) sorted by expert, and the weighted sum of the
// experts' results.
//
// Choice: a wave takes a token, lane l its experts l * kR .. l * kR + kR - 1.  Logits become whole numbers of the same order,
// so that a round of the choice is a maximum over a lane's own, a maximum over the wave and a ballot: the lowest lane that has it, and there the
// lowest of its experts.  A chosen one is struck off.  Softmax in f32 with the largest logit subtracted.
//
// Positions: the choices of 64 tokens are a 64-bit mask per expert (a token takes an expert once), so a pair's rank among its
// expert's is a count of bits: no sort, and an order that no atomic can change.  Few tokens: one workgroup does everything in one
// launch.  More: a launch for the choices that also leaves every chunk's count per expert, and one in which every chunk adds up what
// lies in front of it.
#include <hip/hip_runtime.h>

#include "cq_matmul_epilogue.hpp"

namespace cq {
namespace {

// Whole numbers in the order of the floats: +0 and -0 alike, NaN as -infinity, 0 below everything.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (!(v == v)) v = -__builtin_inff();
    const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}

// The choice for one token by one wave: lane j < chosen holds the j-th expert and its weight.
template <int kR>
__device__ __forceinline__ void choose(const RouteArgs& a, uint32_t token, uint32_t lane, uint32_t* expert, float* weight) {
    float logit[kR];
    uint32_t key[kR];
#pragma unroll
    for (int r = 0; r < kR; r++) {
        const uint32_t e = lane * kR + r;
        const bool there = e < a.num_experts;
        logit[r] = there ? load_float(a.dtype, a.logits, token * a.stride_token + e * a.stride_expert) : -__builtin_inff();
        if (!(logit[r] == logit[r])) logit[r] = -__builtin_inff();
        key[r] = there ? ordered(logit[r]) : 0u;
    }
    uint32_t mine = 0;
    float mine_logit = -__builtin_inff(), largest = 0.0f;
    for (uint32_t j = 0; j < a.chosen; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int r = 1; r < kR; r++) best = max(best, key[r]);
        const uint32_t top = wave_max(best);
        const uint32_t from = static_cast<uint32_t>(__builtin_ctzll(__builtin_amdgcn_ballot_w64(best == top)));
        uint32_t at = 0;  // the lowest of the lane's experts that has the maximum
        float value = 0.0f;
#pragma unroll
        for (int r = kR - 1; r >= 0; r--)
            if (key[r] == best) at = r, value = logit[r];
#pragma unroll
        for (int r = 0; r < kR; r++)
            if (lane == from && at == static_cast<uint32_t>(r)) key[r] = 0u;
        const uint32_t e = from * kR + __builtin_amdgcn_readlane(at, from);
        const float l = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, value), from));
        if (j == 0) largest = l;
        if (lane == j) mine = e, mine_logit = l;
    }
    const auto score = [&](float l) {
        if (a.sigmoid) return l == -__builtin_inff() ? 0.0f : 1.0f / (1.0f + expf(-l));
        // the largest itself scores 1 also where it is infinite; a token without any finite logit scores nothing
        return l == -__builtin_inff() ? 0.0f : (l == largest ? 1.0f : expf(l - largest));
    };
    float w = lane < a.chosen ? score(mine_logit) : 0.0f;
    float divisor = 1.0f;
    if (a.normalize) {
        divisor = wave_sum(w);
    } else if (!a.sigmoid) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kR; r++) sum += score(logit[r]);
        divisor = wave_sum(sum);
    }
    *expert = mine;
    *weight = divisor > 0.0f ? w / divisor : 0.0f;
}

// Sums of `count[e]` over the experts in front of e, for every e, in place, by the first wave; returns with everybody past a barrier.
// count has num + 1 places; the last one becomes the total.
__device__ __forceinline__ void scan_experts(uint32_t* count, uint32_t num) {
    if (threadIdx.x < 64) {
        uint32_t carry = 0;
        for (uint32_t e0 = 0; e0 <= num; e0 += 64) {
            const uint32_t e = e0 + threadIdx.x, own = e < num ? count[e] : 0u;
            uint32_t sum = own;
#pragma unroll
            for (uint32_t d = 1; d < 64; d *= 2) {
                const uint32_t below = __shfl_up(sum, d);
                sum += threadIdx.x >= d ? below : 0u;
            }
            if (e <= num) count[e] = carry + sum - own;
            carry += __builtin_amdgcn_readlane(sum, 63);
        }
    }
    __syncthreads();
}

constexpr uint32_t kWords = 4;              // masks of 64 tokens that a workgroup holds
constexpr uint32_t kChunk = 64 * kWords;    // tokens of one launch alone
constexpr uint32_t kSmallThreads = 1024;

// Few tokens: everything by one workgroup.
template <int kR>
__global__ __launch_bounds__(kSmallThreads) void route_small_kernel(RouteArgs a) {
    __shared__ unsigned long long mask[kWords][64 * kR];
    __shared__ uint32_t before[64 * kR + 1];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t i = threadIdx.x; i < kWords * 64 * kR; i += kSmallThreads) mask[0][i] = 0;
    __syncthreads();
    for (uint32_t t = wave; t < a.tokens; t += kSmallThreads / 64) {
        uint32_t e;
        float w;
        choose<kR>(a, t, lane, &e, &w);
        if (lane < a.chosen) {
            a.weights[t * a.chosen + lane] = w;
            a.experts[t * a.chosen + lane] = static_cast<int32_t>(e);
            atomicOr(&mask[t / 64][e], 1ull << (t % 64));
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.num_experts; e += kSmallThreads) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) n += __popcll(mask[i][e]);
        before[e] = n;
    }
    __syncthreads();
    scan_experts(before, a.num_experts);
    for (uint32_t e = threadIdx.x; e <= a.num_experts; e += kSmallThreads) a.offsets[e] = static_cast<int32_t>(before[e]);
    for (uint32_t i = threadIdx.x; i < a.tokens * a.chosen; i += kSmallThreads) {
        const uint32_t t = i / a.chosen, e = static_cast<uint32_t>(a.experts[i]);  // written by this workgroup, in front of the barriers
        uint32_t slot = before[e] + __popcll(mask[t / 64][e] & ((1ull << (t % 64)) - 1ull));
        for (uint32_t k = 0; k < t / 64; k++) slot += __popcll(mask[k][e]);
        a.slots[i] = static_cast<int32_t>(slot);
        a.rows[slot] = static_cast<int32_t>(t);
    }
}

// Many tokens, first launch: the choices of a chunk of 64 tokens by 16 waves, and its mask per expert into the workspace
// [chunk][expert].
template <int kR>
__global__ __launch_bounds__(kSmallThreads) void route_choose_kernel(RouteArgs a, unsigned long long* __restrict__ masks) {
    __shared__ unsigned long long mask[64 * kR];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t i = threadIdx.x; i < 64 * kR; i += kSmallThreads) mask[i] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * 64u;
    for (uint32_t t = wave; t < 64 && first + t < a.tokens; t += kSmallThreads / 64) {
        uint32_t e;
        float w;
        choose<kR>(a, first + t, lane, &e, &w);
        if (lane < a.chosen) {
            const uint32_t i = (first + t) * a.chosen + lane;
            a.weights[i] = w;
            a.experts[i] = static_cast<int32_t>(e);
            atomicOr(&mask[e], 1ull << t);
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.num_experts; e += kSmallThreads) masks[static_cast<uint64_t>(blockIdx.x) * a.num_experts + e] = mask[e];
}

// Second launch: a workgroup counts, per expert, the pairs of all chunks and of those in front of its own, and places its chunks'.
__global__ __launch_bounds__(kSmallThreads) void route_place_kernel(RouteArgs a, const unsigned long long* __restrict__ masks, uint32_t chunks,
                                                                    uint32_t chunks_each) {
    __shared__ uint32_t total[CQ_MAX_EXPERTS + 1], before[CQ_MAX_EXPERTS];
    const uint32_t first = blockIdx.x * chunks_each, last = min(chunks, first + chunks_each);
    for (uint32_t e = threadIdx.x; e < a.num_experts; e += kSmallThreads) total[e] = before[e] = 0;
    __syncthreads();
    for (uint64_t i = threadIdx.x; i < static_cast<uint64_t>(chunks) * a.num_experts; i += kSmallThreads) {
        const uint32_t chunk = static_cast<uint32_t>(i / a.num_experts), e = static_cast<uint32_t>(i % a.num_experts);
        const uint32_t n = __popcll(masks[i]);
        if (n == 0) continue;
        atomicAdd(&total[e], n);
        if (chunk < first) atomicAdd(&before[e], n);
    }
    __syncthreads();
    scan_experts(total, a.num_experts);
    if (blockIdx.x == 0)
        for (uint32_t e = threadIdx.x; e <= a.num_experts; e += kSmallThreads) a.offsets[e] = static_cast<int32_t>(total[e]);
    const uint32_t pairs = (min(a.tokens, last * 64u) - first * 64u) * a.chosen;
    for (uint32_t i = threadIdx.x; i < pairs; i += kSmallThreads) {
        const uint32_t pair = first * 64u * a.chosen + i, t = pair / a.chosen, e = static_cast<uint32_t>(a.experts[pair]);
        uint32_t slot = total[e] + before[e];
        for (uint32_t c = first; c < t / 64u; c++) slot += __popcll(masks[static_cast<uint64_t>(c) * a.num_experts + e]);
        slot += __popcll(masks[static_cast<uint64_t>(t / 64u) * a.num_experts + e] & ((1ull << (t % 64u)) - 1ull));
        a.slots[pair] = static_cast<int32_t>(slot);
        a.rows[slot] = static_cast<int32_t>(t);
    }
}

template <int kR>
hipError_t route(hipStream_t s, const RouteArgs& a) {
    if (a.tokens <= kChunk) {
        hipLaunchKernelGGL(route_small_kernel<kR>, dim3(1), dim3(kSmallThreads), 0, s, a);
        return hipGetLastError();
    }
    auto* const masks = static_cast<unsigned long long*>(a.workspace);
    const uint32_t chunks = (a.tokens + 63) / 64, each = (chunks + 255) / 256;
    hipLaunchKernelGGL(route_choose_kernel<kR>, dim3(chunks), dim3(kSmallThreads), 0, s, a, masks);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(route_place_kernel, dim3((chunks + each - 1) / each), dim3(kSmallThreads), 0, s, a, static_cast<const unsigned long long*>(masks), chunks, each);
    return hipGetLastError();
}

// A thread makes one value of y.
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    const uint32_t n = blockIdx.x * 256u + threadIdx.x;
    if (n >= a.cols) return;
    for (uint32_t t = blockIdx.y; t < a.tokens; t += gridDim.y) {
        float sum = 0.0f;
        for (uint32_t j = 0; j < a.chosen; j++) {
            const uint64_t pair = static_cast<uint64_t>(t) * a.chosen + j;
            const uint32_t slot = static_cast<uint32_t>(a.slots[pair]);
            if (slot < a.positions) sum = __builtin_fmaf(a.weights[pair], load_float(a.h_dtype, a.h, slot * a.h_stride + n), sum);
        }
        if (a.residual) sum += load_float(a.y_dtype, a.residual, t * a.residual_stride + n);
        store_float(a.y_dtype, a.y, t * a.y_stride + n, sum);
    }
}

}  // namespace

uint64_t route_workspace_bytes(uint64_t tokens, uint64_t experts, uint64_t) {
    return tokens <= kChunk ? 0 : (tokens + 63) / 64 * experts * 8;
}

hipError_t launch_route(hipStream_t s, const RouteArgs& a) {
    if (a.num_experts <= 64) return route<1>(s, a);
    if (a.num_experts <= 128) return route<2>(s, a);
    if (a.num_experts <= 256) return route<4>(s, a);
    if (a.num_experts <= 512) return route<8>(s, a);
    return route<16>(s, a);
}

hipError_t launch_combine(hipStream_t s, const CombineArgs& a) {
    hipLaunchKernelGGL(combine_kernel, dim3((a.cols + 255) / 256, a.tokens < 65535 ? a.tokens : 65535), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace cq
