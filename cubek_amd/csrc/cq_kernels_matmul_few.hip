// Products with quantized weights for up to eight positions of an expert (or of the whole product): a decode step.
//
// A wave takes 16 or 32 rows of W (gated: 16 and their gated ones) and a share of their columns, in stages of a line of 128 bytes of every
// row.  Codes, scales and x of a stage come into the wave's own part of LDS by direct loads, kDepth stages ahead, so that waves wait for
// nobody and for nothing but their own loads; 16 x 16 x 32 matrix instructions take lane (i, g)'s eight columns of row i, and the same of
// token i.  The eight waves of a workgroup are one to eight groups of rows by eight to one shares of the columns; the shares' sums meet
// in LDS at the end.  Bound by the read of W, and in launches of few stages by the time from a workgroup's start to its first
// stage and from its last one to its sums.
#include <hip/hip_runtime.h>

#include "cq_gemv_operand.hpp"
#include "cq_matmul_epilogue.hpp"
#include "cq_matmul_tiles.hpp"
#include "cq_matmul_weights.hpp"

namespace cq {
namespace {

template <dev::Float kF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (kF == dev::Float::BF16) {
        typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// kNT: groups of 16 rows of a wave; kX: loads of 1 KiB that hold a stage of x.
template <dev::Float kF, int kCode, int kNT, int kX>
__global__ __launch_bounds__(512) void matmul_few_kernel(MatmulArgs a, FewGrid grid) {
    constexpr uint32_t kBits = bits_of(kCode), kUnit = 128 / kBits;  // columns of 16 bytes of codes
    constexpr uint32_t kM = kUnit / 8, kPieces = 8 * kM;             // matrix instructions of a unit; a stage's 16-byte pieces of x of a token
    constexpr uint32_t kCodeBytes = kNT * 2048, kScaleBytes = kNT * 512, kSlot = kCodeBytes + kScaleBytes + kX * 1024;
    constexpr uint32_t kLoads = kNT * 4 + kX, kDepth = kFewDepth;
    extern __shared__ char lds[];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t i = lane & 15u, g = lane >> 4;
    const uint32_t shares = 1u << grid.shares_log2, share = wave & (shares - 1u), group = wave >> grid.shares_log2;
    char* const mine = lds + wave * (kDepth * kSlot);

    TileOfPositions at;
    if (!find_tile(a, blockIdx.y, kFewLog2, &at)) return;
    const uint32_t tokens = at.last - at.first;
    constexpr uint32_t kPlainRows = 16 * kNT;
    const uint32_t wave_rows = a.gated ? kPlainRows / 2 : kPlainRows;  // columns of y of a wave
    const uint32_t row0 = min((blockIdx.x * (8u >> grid.shares_log2) + group) * wave_rows, a.out_cols - 1u);
    // rows past the last are the last again and never stored; gated: the second 16 belong to the first
    const auto weight_row = [&](uint32_t r) {
        return a.gated ? min(row0 + r % 16u, a.out_cols - 1u) + r / 16u * a.out_cols : min(row0 + r, a.out_cols - 1u);
    };
    const uint32_t units = a.cols / kUnit, stages = (units + 7u) / 8u;
    const char* const words = a.words + at.expert * a.expert_bytes + row0 * a.row_bytes;
    const uint32_t scale_row0 = a.block_rows ? row0 / a.block_rows : 0u;
    const uint64_t scale_at = (at.expert * a.scale_expert + scale_row0 * a.scale_row) * grid.scale_size + (reinterpret_cast<uintptr_t>(a.scales) & 3u);
    const char* const scales = a.scales - (reinterpret_cast<uintptr_t>(a.scales) & 3u) + (scale_at & ~3ull);
    const uint32_t scale_base = static_cast<uint32_t>(scale_at & 3u);
    const auto scale_row_of = [&](uint32_t r) {
        return scale_base + (a.block_rows ? (weight_row(r) / a.block_rows - scale_row0) * static_cast<uint32_t>(a.scale_row * grid.scale_size) : 0u);
    };

    // Where a lane's pieces come from.  Codes: place p of row r holds unit p ^ (r / 2 % 8); scales: place u of row r that of unit u; x: place p of
    // token v piece p ^ (v % 16).  Positions past the last are the last again.
    uint32_t code_from[2 * kNT], code_unit[2 * kNT], scale_from[2 * kNT], x_piece[kX];
    const char* x_from[kX];
#pragma unroll
    for (uint32_t q = 0; q < 2 * kNT; q++) {
        const uint32_t r = q * 8u + lane / 8u;
        code_unit[q] = (lane & 7u) ^ ((r >> 1) & 7u);
        code_from[q] = (weight_row(r) - row0) * static_cast<uint32_t>(a.row_bytes);
        scale_from[q] = scale_row_of(r);
    }
#pragma unroll
    for (uint32_t q = 0; q < kX; q++) {
        const uint32_t pl = q * 64u + lane, v = min(pl / kPieces, tokens - 1u);
        x_piece[q] = (pl % kPieces) ^ (v & 15u);
        x_from[q] = a.x + row_of_position(a, at.first + v) * a.x_stride * 2u;
    }
    const auto load = [&](uint32_t stage, uint32_t slot) {
        char* const to = mine + slot * kSlot;
        const uint32_t unit0 = stage * 8u;
#pragma unroll
        for (uint32_t q = 0; q < 2 * kNT; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(words + (code_from[q] + min(unit0 + code_unit[q], units - 1u) * 16u)),
                                             CQ_LDS_PTR(to + q * 1024u), 16, 0, 2 /* nt */);
        const uint32_t block = grid.units_per_block.div(min(unit0 + (lane & 7u), units - 1u)) * grid.scale_col_bytes;
#pragma unroll
        for (uint32_t q = 0; q < 2 * kNT; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(scales + ((scale_from[q] + block) & ~3u)), CQ_LDS_PTR(to + kCodeBytes + q * 256u), 4, 0, 0);
        const uint32_t pieces = (units - unit0) * kM;
#pragma unroll
        for (uint32_t q = 0; q < kX; q++) {
            const char* p = x_from[q] + (static_cast<uint64_t>(unit0) * kM + x_piece[q]) * 16u;
            if (pieces < kPieces && x_piece[q] >= pieces) p = kZeros;  // columns past the row's end
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(p), CQ_LDS_PTR(to + kCodeBytes + kScaleBytes + q * 1024u), 16, 0, 0);
        }
    };

    f32x4 acc[kNT][2] = {};
    const uint32_t column = min(i, tokens - 1u);
    uint32_t scale_of_row[kNT];
#pragma unroll
    for (uint32_t n = 0; n < kNT; n++) scale_of_row[n] = scale_row_of(n * 16u + i);
    const uint32_t count = stages > share ? (stages - share + shares - 1u) >> grid.shares_log2 : 0u;  // this wave's stages
#pragma unroll
    for (uint32_t d = 0; d < kDepth; d++) load(min(share + (d << grid.shares_log2), stages - 1u), d);
    uint32_t slot = 0;
    for (uint32_t n = 0; n < count; n++) {
        const uint32_t stage = share + (n << grid.shares_log2);
        // the oldest stage is there
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kDepth - 1) * kLoads) : "memory");
        const char* const from = mine + slot * kSlot;
        u32x4 w[kNT][2], xv[2][kM];
        uint32_t word[kNT][2];
#pragma unroll
        for (uint32_t q = 0; q < 2; q++) {
            const uint32_t unit = q * 4u + g;
#pragma unroll
            for (uint32_t t = 0; t < kNT; t++) {
                word[t][q] = *reinterpret_cast<const uint32_t*>(from + kCodeBytes + t * 512u + i * 32u + unit * 4u);
                w[t][q] = *reinterpret_cast<const u32x4*>(from + t * 2048u + i * 128u + (unit ^ ((i >> 1) & 7u)) * 16u);
            }
#pragma unroll
            for (uint32_t m = 0; m < kM; m++)
                xv[q][m] = *reinterpret_cast<const u32x4*>(from + kCodeBytes + kScaleBytes + (column * kPieces + ((unit * kM + m) ^ column)) * 16u);
        }
        // it has been read: its place takes the stage kDepth ahead
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        load(min(stage + (kDepth << grid.shares_log2), stages - 1u), slot);
        slot = slot + 1 == kDepth ? 0 : slot + 1;
        float scale[kNT][2];
        bool mine_short = true;
#pragma unroll
        for (uint32_t q = 0; q < 2; q++) {
            const uint32_t block = grid.units_per_block.div(min(stage * 8u + q * 4u + g, units - 1u)) * grid.scale_col_bytes;
#pragma unroll
            for (uint32_t t = 0; t < kNT; t++) {
                scale[t][q] = dev::round_to<kF>(scale_of(a.param_dtype, word[t][q], scale_of_row[t] + block));
                mine_short = mine_short && takes_short<kF, kCode>(scale[t][q]);
            }
        }
        const bool whole = stage * 8u + 8u <= units;
        if (whole && (kCode > 8 || __builtin_amdgcn_ballot_w64(!mine_short) == 0)) {
#pragma unroll
            for (uint32_t q = 0; q < 2; q++)
#pragma unroll
                for (uint32_t m = 0; m < kM; m++)
#pragma unroll
                    for (uint32_t t = 0; t < kNT; t++) acc[t][m & 1] = mfma<kF>(unit_slice<kF, kCode, true>(w[t][q], m, scale[t][q]), xv[q][m], acc[t][m & 1]);
        } else {
#pragma unroll
            for (uint32_t q = 0; q < 2; q++)
#pragma unroll
                for (uint32_t m = 0; m < kM; m++)
#pragma unroll
                    for (uint32_t t = 0; t < kNT; t++) {
                        u32x4 v = unit_slice<kF, kCode, false>(w[t][q], m, scale[t][q]);
                        if (stage * 8u + q * 4u + g >= units) v = u32x4{0, 0, 0, 0};
                        acc[t][m & 1] = mfma<kF>(v, xv[q][m], acc[t][m & 1]);
                    }
        }
    }

    // sums [wave][group of 16 rows][token][row], the shares of a group side by side; loads on their way are waited for, LDS is used again
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
    for (uint32_t t = 0; t < kNT; t++) *reinterpret_cast<f32x4*>(part + ((wave * kNT + t) * 16u + i) * 16u + 4u * g) = acc[t][0] + acc[t][1];
    __syncthreads();
    const uint32_t rows_each = wave_rows, outputs = (8u >> grid.shares_log2) * rows_each * tokens;
    for (uint32_t o = threadIdx.x; o < outputs; o += 512) {
        const uint32_t r = o % rows_each, rest = o / rows_each, t = rest % tokens, in_group = rest / tokens;
        const uint32_t col = (blockIdx.x * (8u >> grid.shares_log2) + in_group) * rows_each + r;
        if (col >= a.out_cols) continue;
        const auto sum = [&](uint32_t row) {
            float v = 0.0f;
            for (uint32_t s = 0; s < shares; s++) v += part[((((in_group << grid.shares_log2) + s) * kNT + row / 16u) * 16u + t) * 16u + row % 16u];
            return v;
        };
        finish1(a, at.expert, at.first + t, col, sum(r), a.gated ? sum(16u + r) : 0.0f);
    }
}

template <dev::Float kF, int kCode, int kNT, int kX>
hipError_t launch_few(hipStream_t s, const MatmulArgs& a, uint32_t shares_log2) {
    constexpr uint32_t kSlot = kNT * 2560 + kX * 1024, kParts = 8 * kNT * 256 * 4, kLds = 8 * kFewDepth * kSlot;
    static_assert(kParts <= kLds && kLds <= 160 * 1024, "the sums fit where the stages were");
    const uint32_t columns = (8u >> shares_log2) * (a.gated ? 8u : 16u) * kNT;
    const FewGrid grid(a, 128 / bits_of(kCode), shares_log2);
    hipLaunchKernelGGL((matmul_few_kernel<kF, kCode, kNT, kX>), dim3((a.out_cols + columns - 1) / columns, static_cast<uint32_t>(most_tiles(a, kFewLog2))), dim3(512),
                       kLds, s, a, grid);
    return hipGetLastError();
}

template <dev::Float kF, int kCode, int kNT>
hipError_t launch_loads(hipStream_t s, const MatmulArgs& a, uint32_t tokens, uint32_t shares_log2) {
    constexpr uint32_t kLine = 1024 / bits_of(kCode) * 2;  // bytes of x of a token in a stage
    const uint32_t loads = (tokens * kLine + 1023) / 1024;
    if (loads <= 1) return launch_few<kF, kCode, kNT, 1>(s, a, shares_log2);
    if (loads <= 2) return launch_few<kF, kCode, kNT, 2>(s, a, shares_log2);
    if constexpr (kLine >= 512)
        if (loads <= 4) return launch_few<kF, kCode, kNT, 4>(s, a, shares_log2);
    return hipErrorInvalidValue;
}

}  // namespace

#define CQ_FEW_NAME2(f, c) matmul_few_##f##_##c
#define CQ_FEW_NAME(f, c) CQ_FEW_NAME2(f, c)
hipError_t CQ_FEW_NAME(CQ_TU_FLOAT, CQ_TU_CODE)(hipStream_t s, const MatmulArgs& a, const FewShape& shape) {
    return shape.groups == 1 ? launch_loads<dev::Float::CQ_TU_FLOAT, CQ_TU_CODE, 1>(s, a, shape.tokens, shape.shares_log2)
                             : launch_loads<dev::Float::CQ_TU_FLOAT, CQ_TU_CODE, 2>(s, a, shape.tokens, shape.shares_log2);
}

}  // namespace cq
