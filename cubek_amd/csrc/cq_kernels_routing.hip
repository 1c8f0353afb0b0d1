// The choice of experts for every token, the positions of the pairs (token, choice) sorted by expert, and the weighted sum of the
// experts' results.
//
// Choice: 16 lanes take a token of up to 128 experts, a wave one of more; lane l its experts l * kR .. l * kR + kR - 1.  Logits become
// whole numbers of the same order, so that a round of the choice is a maximum over a lane's own, a maximum over the lanes by DPP and a ballot: the
// lowest lane that has it, and there the lowest of its experts, which is struck off.  Softmax in f32 with the largest logit subtracted.  Bound by these
// instructions, about 15 per token and choice for 128 experts (a wave per token with shuffles through LDS took four times as long).
//
// Positions: the choices of 64 tokens are a 64-bit mask per expert (a token takes an expert once), so a pair's rank among its
// expert's is a count of bits: no sort, and an order that no atomic can change.  Few tokens: one workgroup does everything in one
// launch.  More: a launch for the choices that also leaves every chunk's mask and count per expert, and one in which every workgroup adds up the
// counts that lie in front of its chunks.
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

template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xf, 0xf, true));
}

// Over kLanes lanes, to all of them: two neighbours, four, eight (the half row mirrored), sixteen (the row mirrored), and from row to row.
template <int kLanes, class F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, F f) {
    v = f(v, dpp<0xB1>(v));
    v = f(v, dpp<0x4E>(v));
    v = f(v, dpp<0x141>(v));
    v = f(v, dpp<0x140>(v));
    if constexpr (kLanes == 64) {
        const uint32_t rows[4] = {static_cast<uint32_t>(__builtin_amdgcn_readlane(v, 0)), static_cast<uint32_t>(__builtin_amdgcn_readlane(v, 16)),
                                  static_cast<uint32_t>(__builtin_amdgcn_readlane(v, 32)), static_cast<uint32_t>(__builtin_amdgcn_readlane(v, 48))};
        v = f(f(rows[0], rows[1]), f(rows[2], rows[3]));
    }
    return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t max_over_lanes(uint32_t v) {
    return over_lanes<kLanes>(v, [](uint32_t x, uint32_t y) { return max(x, y); });
}
template <int kLanes>
__device__ __forceinline__ float sum_over_lanes(float v) {
    return __builtin_bit_cast(float, over_lanes<kLanes>(__builtin_bit_cast(uint32_t, v), [](uint32_t x, uint32_t y) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y));
    }));
}

// A lane's kR logits, from expert `first` on; NaN as -infinity, and so what lies past the last expert.
template <int kR>
__device__ __forceinline__ void load_logits(const RouteArgs& a, uint32_t token, uint32_t first, float* logit) {
    const uint64_t at = token * a.stride_token + first * a.stride_expert;
    const bool whole = a.vector_logits && first + kR <= a.num_experts;  // contiguous, a lane's on a boundary of their own size, up to 16 bytes
    if (whole && a.dtype == CQ_F32) {
        typedef float vec __attribute__((ext_vector_type(kR >= 4 ? 4 : kR)));
        constexpr int kN = sizeof(vec) / 4;
#pragma unroll
        for (int q = 0; q < kR / kN; q++) {
            const vec v = reinterpret_cast<const vec*>(a.logits + at * 4)[q];
#pragma unroll
            for (int r = 0; r < kN; r++) logit[q * kN + r] = kN == 1 ? reinterpret_cast<const float*>(&v)[0] : v[r];
        }
    } else if (whole) {
        typedef uint16_t vec __attribute__((ext_vector_type(kR >= 8 ? 8 : kR)));
        constexpr int kN = sizeof(vec) / 2;
#pragma unroll
        for (int q = 0; q < kR / kN; q++) {
            const vec v = reinterpret_cast<const vec*>(a.logits + at * 2)[q];
#pragma unroll
            for (int r = 0; r < kN; r++) {
                const uint16_t bits = kN == 1 ? reinterpret_cast<const uint16_t*>(&v)[0] : v[r];
                logit[q * kN + r] = a.dtype == CQ_BF16 ? __builtin_bit_cast(float, static_cast<uint32_t>(bits) << 16) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < kR; r++) logit[r] = first + r < a.num_experts ? load_float(a.dtype, a.logits, at + r * a.stride_expert) : -__builtin_inff();
    }
#pragma unroll
    for (int r = 0; r < kR; r++)
        if (!(logit[r] == logit[r])) logit[r] = -__builtin_inff();
}

// The choice for one token by kLanes lanes, of which this one is `lane`: weights and experts are stored, and `chosen(expert)` is called once for each
// choice, by the lane that holds it.  Choices are at most as many as the lanes.  Tokens past the last go through the motions (`there`).
template <int kLanes, int kR, class F>
__device__ __forceinline__ void choose(const RouteArgs& a, uint32_t token, uint32_t lane, bool there, F chosen) {
    float logit[kR];
    uint32_t key[kR];
    load_logits<kR>(a, token, lane * kR, logit);
#pragma unroll
    for (int r = 0; r < kR; r++) key[r] = lane * kR + r < a.num_experts ? ordered(logit[r]) : 0u;
    const uint32_t group = (threadIdx.x & 63u) & ~(kLanes - 1u);  // the first of the token's lanes in its wave
    float mine = -__builtin_inff(), largest = 0.0f;
    for (uint32_t j = 0; j < a.chosen; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int r = 1; r < kR; r++) best = max(best, key[r]);
        const uint32_t top = max_over_lanes<kLanes>(best);
        const uint64_t have = __builtin_amdgcn_ballot_w64(best == top);
        const uint32_t from = kLanes == 64 ? static_cast<uint32_t>(__builtin_ctzll(have)) : static_cast<uint32_t>(__builtin_ctz(static_cast<uint32_t>(have >> group) & 0xffffu));
        // the logit again, from its number
        const float l = __builtin_bit_cast(float, top & 0x80000000u ? top & 0x7fffffffu : ~top);
        if (j == 0) largest = l;
        if (lane == j) mine = l;
        uint32_t at = 0;
        bool left = lane == from;
#pragma unroll
        for (int r = 0; r < kR; r++) {
            const bool hit = left && key[r] == top;
            at = hit ? static_cast<uint32_t>(r) : at;
            key[r] = hit ? 0u : key[r];
            left = left && !hit;
        }
        if (lane == from && there) {
            a.experts[token * a.chosen + j] = static_cast<int32_t>(lane * kR + at);
            chosen(lane * kR + at);
        }
    }
    // Sigmoids of a token that are all below 1/2 are divided by their sum as multiples of exp(largest), so that small ones keep their quotients where
    // exp(-l) leaves the range of f32.  From -709.7827 down it leaves that of 64 bits: masks of a type's lowest value weigh nothing, as those of -infinity do.
    const bool small = a.sigmoid && a.normalize && largest < 0.0f;
    const auto score = [&](float l) {
        if (a.sigmoid) {
            float s = 1.0f / (1.0f + expf(-l));
            if (small) s = l <= -709.7827f ? 0.0f : expf(l - largest) / (1.0f + expf(l));
            return s;
        }
        // the largest itself scores 1 also where it is infinite; a token without any finite logit scores nothing
        return l == -__builtin_inff() ? 0.0f : (l == largest ? 1.0f : expf(l - largest));
    };
    const float w = lane < a.chosen ? score(mine) : 0.0f;
    float divisor = 1.0f;
    if (a.normalize) {
        divisor = sum_over_lanes<kLanes>(w);
    } else if (!a.sigmoid) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kR; r++) sum += score(logit[r]);
        divisor = sum_over_lanes<kLanes>(sum);
    }
    if (lane < a.chosen && there) a.weights[token * a.chosen + lane] = divisor > 0.0f ? w / divisor : 0.0f;
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
constexpr uint32_t kThreads = 1024;

// A chunk's counts, of a byte each, come four at a time.
__host__ __device__ inline uint32_t counts_pitch(uint32_t experts) { return (experts + 3u) & ~3u; }

// Few tokens: everything by one workgroup.
template <int kLanes, int kR>
__global__ __launch_bounds__(kThreads) void route_small_kernel(RouteArgs a) {
    __shared__ unsigned long long mask[kWords][kLanes * kR];
    __shared__ uint32_t before[kLanes * kR + 1];
    for (uint32_t i = threadIdx.x; i < kWords * kLanes * kR; i += kThreads) mask[0][i] = 0;
    __syncthreads();
    for (uint32_t t = threadIdx.x / kLanes; t < (a.tokens + 64u / kLanes - 1u) / (64u / kLanes) * (64u / kLanes); t += kThreads / kLanes)  // whole waves
        choose<kLanes, kR>(a, min(t, a.tokens - 1u), threadIdx.x % kLanes, t < a.tokens, [&](uint32_t e) { atomicOr(&mask[t / 64][e], 1ull << (t % 64)); });
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.num_experts; e += kThreads) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) n += __popcll(mask[i][e]);
        before[e] = n;
    }
    __syncthreads();
    scan_experts(before, a.num_experts);
    for (uint32_t e = threadIdx.x; e <= a.num_experts; e += kThreads) a.offsets[e] = static_cast<int32_t>(before[e]);
    for (uint32_t i = threadIdx.x; i < a.tokens * a.chosen; i += kThreads) {
        const uint32_t t = i / a.chosen, e = static_cast<uint32_t>(a.experts[i]);  // written by this workgroup, in front of the barriers
        uint32_t slot = before[e] + __popcll(mask[t / 64][e] & ((1ull << (t % 64)) - 1ull));
        for (uint32_t k = 0; k < t / 64; k++) slot += __popcll(mask[k][e]);
        a.slots[i] = static_cast<int32_t>(slot);
        a.rows[slot] = static_cast<int32_t>(t);
    }
}

// Many tokens, first launch: the choices of a chunk of 64 tokens, its mask and its count per expert into the workspace, [chunk][expert]
// each.
template <int kLanes, int kR>
__global__ __launch_bounds__(kThreads) void route_choose_kernel(RouteArgs a, unsigned long long* __restrict__ masks, uint8_t* __restrict__ counts) {
    __shared__ unsigned long long mask[kLanes * kR];
    for (uint32_t i = threadIdx.x; i < kLanes * kR; i += kThreads) mask[i] = 0;
    __syncthreads();
    for (uint32_t t = threadIdx.x / kLanes; t < 64; t += kThreads / kLanes) {
        const uint32_t token = blockIdx.x * 64u + t;
        choose<kLanes, kR>(a, min(token, a.tokens - 1u), threadIdx.x % kLanes, token < a.tokens, [&](uint32_t e) { atomicOr(&mask[e], 1ull << t); });
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.num_experts; e += kThreads) masks[static_cast<uint64_t>(blockIdx.x) * a.num_experts + e] = mask[e];
    const uint32_t pitch = counts_pitch(a.num_experts);
    for (uint32_t e = threadIdx.x; e < pitch; e += kThreads)
        counts[static_cast<uint64_t>(blockIdx.x) * pitch + e] = e < a.num_experts ? static_cast<uint8_t>(__popcll(mask[e])) : 0;
}

// Second launch: a workgroup counts, per expert, the pairs of all chunks and of those in front of its own, and places its chunks'.  A thread
// adds up four experts over every so many chunks: sums of whole numbers, in any order the same.  What a thread needs of its first pair is asked
// for first, so that the launch waits for memory twice and not four times (16.6 -> 7 us for 16381 tokens, 8 of 128 experts).
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a, const unsigned long long* __restrict__ masks, const uint8_t* __restrict__ counts,
                                                               uint32_t chunks, uint32_t chunks_each) {
    __shared__ uint32_t total[CQ_MAX_EXPERTS + 4], before[CQ_MAX_EXPERTS + 4];
    const uint32_t first = blockIdx.x * chunks_each, last = min(chunks, first + chunks_each);
    const uint32_t pairs = (min(a.tokens, last * 64u) - first * 64u) * a.chosen, pair0 = first * 64u * a.chosen;
    const auto expert_of = [&](uint32_t i) { return static_cast<uint32_t>(a.experts[pair0 + i]); };
    const auto mask_of = [&](uint32_t t, uint32_t e) { return masks[static_cast<uint64_t>(t / 64u) * a.num_experts + e] & ((1ull << (t % 64u)) - 1ull); };
    uint32_t e0 = 0;
    unsigned long long mask0 = 0;
    if (threadIdx.x < pairs) e0 = expert_of(threadIdx.x);
    for (uint32_t e = threadIdx.x; e < a.num_experts + 4u; e += kThreads) total[min(e, CQ_MAX_EXPERTS + 3u)] = before[min(e, CQ_MAX_EXPERTS + 3u)] = 0;
    __syncthreads();
    const uint32_t pitch = counts_pitch(a.num_experts), fours = pitch / 4u, slices = kThreads / fours, four = threadIdx.x % fours, slice = threadIdx.x / fours;
    if (slice < slices) {
        uint32_t all[4] = {}, front[4] = {};
#pragma unroll 8
        for (uint32_t c = slice; c < chunks; c += slices) {
            const uint32_t n = *reinterpret_cast<const uint32_t*>(counts + static_cast<uint64_t>(c) * pitch + four * 4u);
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                all[k] += n >> (8u * k) & 0xffu;
                front[k] += c < first ? n >> (8u * k) & 0xffu : 0u;
            }
        }
        if (threadIdx.x < pairs) mask0 = mask_of((pair0 + threadIdx.x) / a.chosen, e0);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            atomicAdd(&total[four * 4u + k], all[k]);
            atomicAdd(&before[four * 4u + k], front[k]);
        }
    } else if (threadIdx.x < pairs) {
        mask0 = mask_of((pair0 + threadIdx.x) / a.chosen, e0);
    }
    __syncthreads();
    scan_experts(total, a.num_experts);
    if (blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i <= a.num_experts; i += kThreads) a.offsets[i] = static_cast<int32_t>(total[i]);
    for (uint32_t i = threadIdx.x; i < pairs; i += kThreads) {
        const uint32_t pair = pair0 + i, t = pair / a.chosen, e = i == threadIdx.x ? e0 : expert_of(i);
        uint32_t slot = total[e] + before[e];
        for (uint32_t c = first; c < t / 64u; c++) slot += counts[static_cast<uint64_t>(c) * pitch + e];
        slot += __popcll(i == threadIdx.x ? mask0 : mask_of(t, e));
        a.slots[pair] = static_cast<int32_t>(slot);
        a.rows[slot] = static_cast<int32_t>(t);
    }
}

template <int kLanes, int kR>
hipError_t route(hipStream_t s, const RouteArgs& from) {
    RouteArgs a = from;
    const uint64_t size = a.dtype == CQ_F32 ? 4 : 2, vector = kR * size < 16 ? kR * size : 16;
    a.vector_logits = a.stride_expert == 1 && a.stride_token * size % vector == 0 && reinterpret_cast<uintptr_t>(a.logits) % vector == 0;
    if (a.tokens <= kChunk) {
        hipLaunchKernelGGL((route_small_kernel<kLanes, kR>), dim3(1), dim3(kThreads), 0, s, a);
        return hipGetLastError();
    }
    const uint32_t chunks = (a.tokens + 63) / 64, each = (chunks + 255) / 256;
    auto* const masks = static_cast<unsigned long long*>(a.workspace);
    auto* const counts = reinterpret_cast<uint8_t*>(masks + static_cast<uint64_t>(chunks) * a.num_experts);
    hipLaunchKernelGGL((route_choose_kernel<kLanes, kR>), dim3(chunks), dim3(kThreads), 0, s, a, masks, counts);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(route_place_kernel, dim3((chunks + each - 1) / each), dim3(kThreads), 0, s, a, static_cast<const unsigned long long*>(masks),
                       static_cast<const uint8_t*>(counts), chunks, each);
    return hipGetLastError();
}

__global__ __launch_bounds__(256) void route_nothing_kernel(RouteArgs a) {
    for (uint32_t e = threadIdx.x; e <= a.num_experts; e += 256) a.offsets[e] = 0;
}

// Eight columns of a row of h as they lie in memory, so that all rows of a step are on their way before the first is looked at.
template <int kDtype>
struct EightOf {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 bits[kDtype == CQ_F32 ? 2 : 1];

    __device__ void load(const char* h, uint64_t at) {
        const u32x4* const p = reinterpret_cast<const u32x4*>(h + at * (kDtype == CQ_F32 ? 4 : 2));
#pragma unroll
        for (int k = 0; k < (kDtype == CQ_F32 ? 2 : 1); k++) bits[k] = __builtin_nontemporal_load(p + k);
    }
    __device__ f32x8 floats() const { return load_floats8(kDtype, reinterpret_cast<const char*>(bits), 0); }
};

// A thread makes eight columns of a token, or the last ones: bound by the read of h, eight rows of it in flight.  bf16, 8191 tokens of 8 rows
// with 2048 columns and a residual: 54 us, 6.2 TB/s (9 % more without nontemporal loads: every row is read once; twice as long with a branch on
// the type at each load, which waits for one row before the next).  8 tokens: 4 us, a launch.
template <int kDtype>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a, uint32_t parts, uint32_t tokens_each) {
    // parts of a token, 256 of them or whole tokens to a workgroup
    const uint32_t in = parts < 256u ? threadIdx.x / parts : 0u, part = parts < 256u ? threadIdx.x % parts : blockIdx.x * 256u + threadIdx.x;
    if (part >= parts || in >= tokens_each) return;
    const uint32_t n = part * 8u, rest = a.cols - n;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.y) * tokens_each + in; t < a.tokens; t += static_cast<uint64_t>(gridDim.y) * tokens_each) {
        const int32_t* const slots = a.slots + t * a.chosen;
        const float* const weights = a.weights + t * a.chosen;
        const uint64_t at = t * a.y_stride + n;
        if (rest < 8u) {
            for (uint32_t k = 0; k < rest; k++) {
                float sum = 0.0f;
                for (uint32_t j = 0; j < a.chosen; j++) {
                    const uint32_t slot = static_cast<uint32_t>(slots[j]);
                    if (slot < a.positions) sum = __builtin_fmaf(weights[j], load_float(kDtype, a.h, slot * a.h_stride + n + k), sum);
                }
                if (a.residual) sum += load_float(a.y_dtype, a.residual, t * a.residual_stride + n + k);
                store_float(a.y_dtype, a.y, at + k, sum);
            }
            continue;
        }
        f32x8 sum = {};
        const uint32_t chosen = a.positions ? a.chosen : 0u;
#pragma unroll 1
        for (uint32_t j0 = 0; j0 < chosen; j0 += 8) {
            EightOf<kDtype> v[8];
            uint32_t slot[8];
            float w[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t from = min(j0 + j, chosen - 1u);
                slot[j] = static_cast<uint32_t>(slots[from]);
                w[j] = weights[from];
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                if (j0 + j < chosen) v[j].load(a.h, (slot[j] < a.positions ? slot[j] : 0u) * a.h_stride + n);  // (a row in place of one that is not there)
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const bool there = j0 + j < chosen && slot[j] < a.positions;
                const f32x8 row = v[j].floats();
#pragma unroll
                for (int k = 0; k < 8; k++) sum[k] = there ? __builtin_fmaf(w[j], row[k], sum[k]) : sum[k];
            }
        }
        if (a.residual) sum += load_floats8(a.y_dtype, a.residual, t * a.residual_stride + n);
        store8(a.y_dtype, a.y, at, sum);
    }
}

}  // namespace

uint64_t route_workspace_bytes(uint64_t tokens, uint64_t experts, uint64_t) {
    return tokens <= kChunk ? 0 : (tokens + 63) / 64 * (experts * 8 + counts_pitch(static_cast<uint32_t>(experts)));  // masks, then counts
}

hipError_t launch_route(hipStream_t s, const RouteArgs& a) {
    if (a.tokens == 0) {
        hipLaunchKernelGGL(route_nothing_kernel, dim3(1), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    if (a.chosen <= 16) {
        if (a.num_experts <= 16) return route<16, 1>(s, a);
        if (a.num_experts <= 32) return route<16, 2>(s, a);
        if (a.num_experts <= 64) return route<16, 4>(s, a);
        if (a.num_experts <= 128) return route<16, 8>(s, a);
    }
    if (a.num_experts <= 128) return route<64, 2>(s, a);
    if (a.num_experts <= 256) return route<64, 4>(s, a);
    if (a.num_experts <= 512) return route<64, 8>(s, a);
    return route<64, 16>(s, a);
}

hipError_t launch_combine(hipStream_t s, const CombineArgs& a) {
    const uint32_t parts = (a.cols + 7) / 8, each = parts < 256 ? 256 / parts : 1, ys = (a.tokens + each - 1) / each;
    const dim3 grid(parts < 256 ? 1 : (parts + 255) / 256, ys < 65535 ? ys : 65535);
    const auto kernel = a.h_dtype == CQ_F32 ? combine_kernel<CQ_F32> : a.h_dtype == CQ_F16 ? combine_kernel<CQ_F16> : combine_kernel<CQ_BF16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, parts, each);
    return hipGetLastError();
}

}  // namespace cq
