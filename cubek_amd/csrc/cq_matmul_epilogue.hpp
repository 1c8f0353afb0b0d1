// What stands behind a product, in f32: bias, activation, gate, residual, and the one rounding to the type of y.
#pragma once

#include "cq_matmul_internal.hpp"

namespace cq {
namespace {

__device__ __forceinline__ float load_float(int dtype, const char* p, uint64_t i) {
    if (dtype == CQ_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == CQ_F16) return static_cast<float>(reinterpret_cast<const _Float16*>(p)[i]);
    return static_cast<float>(reinterpret_cast<const __bf16*>(p)[i]);
}

__device__ __forceinline__ void store_float(int dtype, char* p, uint64_t i, float v) {
    if (dtype == CQ_F32)
        reinterpret_cast<float*>(p)[i] = v;
    else if (dtype == CQ_F16)
        reinterpret_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    else
        reinterpret_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
}

// `activation` is uniform over the launch.
__device__ __forceinline__ float activated(uint32_t activation, float v) {
    switch (activation) {
        case CQ_ACT_RELU: return v < 0.0f ? 0.0f : v;
        case CQ_ACT_SILU: return v / (1.0f + expf(-v));
        case CQ_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        case CQ_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

// The workgroup's tile: positions first .. last - 1 of expert e.
struct TileOfPositions {
    uint32_t expert, first, last;
};

// Tile number `tile` when the positions of every expert are cut into tiles of 2^size_log2, expert by expert; false past the last one.  The
// offsets lie in device memory, where the host cannot check them: they are taken into 0 .. positions, and a range that runs
// backwards is empty.  Every wave looks at 64 experts at a time, so that 128 of them take two rounds of loads instead of 128.
__device__ __forceinline__ bool find_tile(const MatmulArgs& a, uint32_t tile, uint32_t size_log2, TileOfPositions* out) {
    const uint32_t round_up = (1u << size_log2) - 1u;
    if (a.offsets == nullptr) {
        out->expert = 0;
        out->first = tile << size_log2;
        out->last = min(a.positions, out->first + round_up + 1u);
        return out->first < a.positions;
    }
    const uint32_t lane = threadIdx.x & 63u;
    const int32_t most = static_cast<int32_t>(a.positions);
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 64) {
        const uint32_t e = min(e0 + lane, a.experts - 1u);
        const uint32_t first = static_cast<uint32_t>(min(max(a.offsets[e], 0), most)), last = static_cast<uint32_t>(min(max(a.offsets[e + 1], 0), most));
        const uint32_t tiles = e0 + lane < a.experts && last > first ? (last - first + round_up) >> size_log2 : 0u;
        uint32_t sum = tiles;
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t below = __shfl_up(sum, d);
            sum += lane >= d ? below : 0u;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(tile < sum);
        if (past != 0) {
            const uint32_t l = static_cast<uint32_t>(__builtin_ctzll(past));
            const uint32_t in = tile - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
            out->expert = e0 + l;
            out->first = __builtin_amdgcn_readlane(first, l) + (in << size_log2);
            out->last = min(static_cast<uint32_t>(__builtin_amdgcn_readlane(last, l)), out->first + round_up + 1u);
            return true;
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// Tiles that a launch has to hold for any offsets: every expert may end in a tile that is not full.
inline uint64_t most_tiles(const MatmulArgs& a, uint32_t size_log2) {
    const uint64_t full = (static_cast<uint64_t>(a.positions) + (1u << size_log2) - 1u) >> size_log2;
    return a.offsets ? full + (a.experts < a.positions ? a.experts : a.positions) : full;
}

__device__ __forceinline__ uint32_t row_of_position(const MatmulArgs& a, uint32_t p) {
    if (a.row_of == nullptr) return p;
    return static_cast<uint32_t>(min(max(a.row_of[p], 0), static_cast<int32_t>(a.tokens) - 1));
}

}  // namespace
}  // namespace cq
