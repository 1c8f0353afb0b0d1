// The grid of the products on the matrix cores: which tile a workgroup takes, and which shape of tile a launch.
#pragma once

#include "../../include/cubek_quant_device.hpp"
#include "cq_matmul_internal.hpp"

namespace cq {

enum class TilesShape { k256x256, k256x128, k256x64, k256x32 };  // rows of W x positions

struct TilesGrid {
    uint32_t n_tiles, p_tiles;
    uint32_t scale_size, scale_col_bytes;
    cubek_quant::device::FastDivmod halves_per_block, by_group;  // by 32 columns; by kGroup * n_tiles

    static constexpr uint32_t kUnits = 8, kGroup = 4;  // dies with an L2 each; tiles of positions that share one die's weights

    TilesGrid(const MatmulArgs& a, uint32_t n_tiles, uint64_t p_tiles)
        : n_tiles(n_tiles), p_tiles(static_cast<uint32_t>(p_tiles)), scale_size(a.param_dtype == CQ_F32 ? 4u : 2u),
          scale_col_bytes(static_cast<uint32_t>(a.scale_col * scale_size)), halves_per_block(a.block_cols ? a.block_cols / 32u : 0x7fffffffu),
          by_group(kGroup * n_tiles) {}

    uint32_t workgroups() const { return n_tiles * p_tiles; }

    // Workgroups go round the dies one by one.  Each die gets a run of tiles of its own, in groups of kGroup tiles of positions by all tiles of
    // rows, positions first: what its workgroups read at a time are few rows of x and few of W.
    __device__ void tile(uint32_t block, uint32_t* n, uint32_t* p) const {
        const uint32_t total = n_tiles * p_tiles, each = total / kUnits, rest = total % kUnits;
        const uint32_t die = block % kUnits, in = block / kUnits;
        const uint32_t id = die * each + min(die, rest) + in;
        uint32_t group, within;
        by_group.div_mod(id, &group, &within);
        const uint32_t size = min(kGroup, p_tiles - group * kGroup);
        *n = within / size;
        *p = group * kGroup + within % size;
    }
};

// The kernel of a decode step (cq_kernels_matmul_few.hip): positions of a tile, stages that a wave's loads are ahead.
constexpr uint32_t kFewLog2 = 3, kFewDepth = 2;

struct FewGrid {
    uint32_t shares_log2, scale_size, scale_col_bytes;
    cubek_quant::device::FastDivmod units_per_block;

    FewGrid(const MatmulArgs& a, uint32_t unit, uint32_t shares_log2)
        : shares_log2(shares_log2), scale_size(a.param_dtype == CQ_F32 ? 4u : 2u), scale_col_bytes(static_cast<uint32_t>(a.scale_col * scale_size)),
          units_per_block(a.block_cols ? a.block_cols / unit : 0x7fffffffu) {}
};

struct FewShape {
    uint32_t groups, tokens, shares_log2;  // groups of 16 rows of a wave; most tokens of a tile; shares of a row's columns
};

// Whether it takes a product that tiles_take() lets through: a unit of 16 bytes of codes has one scale.
inline bool few_takes(const MatmulArgs& a, FewShape* shape) {
    const uint32_t unit = 128 / a.bits, stages = (a.cols / unit + 7) / 8;
    const uint64_t each = a.offsets ? (a.positions + a.experts - 1ull) / a.experts : a.positions;
    if (each > (a.offsets ? 4u : 8u) || a.block_cols % unit || most_tiles(a, kFewLog2) > 65535) return false;
    shape->tokens = a.positions < 8 ? a.positions : 8;
    shape->groups = a.gated ? 2 : 1;
    if (a.bits == 2 && shape->tokens > 4) return false;  // a stage of x, 512 columns of each token, is more than a wave's part of LDS
    shape->shares_log2 = stages >= 8 ? 3 : stages >= 4 ? 2 : stages >= 2 ? 1 : 0;
    return true;
}

// Whether the kernels on the matrix cores take a product: 16-bit x, rows of whole 16-byte pieces on boundaries of 16 bytes, scales that serve
// 32 columns at least, and distances within a tile that fit 32 bits.
inline bool tiles_take(const MatmulArgs& a) {
    const auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const uint64_t scale_size = a.param_dtype == CQ_F32 ? 4 : 2, rows = 256 + (a.gated ? a.out_cols : 0);
    const uint64_t x_rows = a.row_of ? a.tokens : 256;
    constexpr uint64_t kFits = 0xf0000000ull;
    if (a.dtype == CQ_F32 || a.cols == 0 || a.cols % 32 || static_cast<uint64_t>(a.cols) * a.bits % 128 || a.block_cols % 32) return false;
    if (!on16(a.words) || !on16(a.x) || a.row_bytes % 16 || a.expert_bytes % 16 || a.x_stride % 8) return false;
    if (a.row_bytes >= kFits / rows || a.x_stride * 2 >= kFits / x_rows) return false;
    if (a.block_rows && (a.scale_row >= kFits / scale_size / 4 / (rows / a.block_rows + 2) ||
                         a.scale_col >= kFits / scale_size / 4 / (a.cols / a.block_cols + 1)))
        return false;
    return (a.out_cols / 16ull + 1) * most_tiles(a, 5) < (1ull << 22);  // workgroups of a launch
}

inline TilesShape tiles_shape(const MatmulArgs& a) {
    const uint64_t each = a.positions / (a.offsets ? a.experts : 1u);
    return each >= 192 ? TilesShape::k256x256 : each >= 96 ? TilesShape::k256x128 : each >= 48 ? TilesShape::k256x64 : TilesShape::k256x32;
}

hipError_t launch_matmul_tiles(hipStream_t s, const MatmulArgs& a);

#define CQ_TILES_CODES(X, f) X(f, 2) X(f, 4) X(f, 8) X(f, 100) X(f, 101) X(f, 102)
#define CQ_TILES_DECLARE(f, c)                                                              \
    hipError_t matmul_tiles_##f##_##c(hipStream_t s, const MatmulArgs& a, TilesShape shape); \
    hipError_t matmul_few_##f##_##c(hipStream_t s, const MatmulArgs& a, const FewShape& shape);
CQ_TILES_CODES(CQ_TILES_DECLARE, BF16)
CQ_TILES_CODES(CQ_TILES_DECLARE, F16)

}  // namespace cq
