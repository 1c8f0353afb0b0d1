// Products with quantized weights on the matrix cores, for more tokens than one 16-row tile: y[p] = epilogue(x[row(p)] * W[e]^T), every
// weight dequantized and rounded as cq_dequantize would store it.
//
// A 32 x 32 x 16 matrix instruction wants in lane (i, h) = (lane % 32, lane / 32) eight values of row i of W and the same eight columns of
// token i, and the columns of the two h may be any that both operands agree on.  A step is 64 columns: h takes 32 of them each, so
// that a lane's codes of a step lie together under one scale, and four instructions take eight each.  W is the first operand: a lane
// ends up with four consecutive columns of y of one token at a time.
//
// A workgroup makes kRows rows of W x kTokens positions.  Each wave dequantizes its own kNT * 32 rows into registers once per step, in between
// the matrix instructions of the step before, and reads all of its tokens from LDS; x and the codes come there by direct
// loads of whole lines, x a step ahead, the codes in chunks of 128 bytes of a row.  The 16-byte places of a line are permuted by row
// so that the sixteen lanes of a read fall on different banks.
#include <hip/hip_runtime.h>

#include "cq_gemv_operand.hpp"
#include "cq_matmul_epilogue.hpp"
#include "cq_matmul_tiles.hpp"
#include "cq_matmul_weights.hpp"

namespace cq {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <dev::Float kF>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (kF == dev::Float::BF16) {
        typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWT>
__global__ __launch_bounds__(64 * kWN * kWT, kWN * kWT >= 8 ? 2 : 1) void matmul_tiles_kernel(MatmulArgs a, TilesGrid grid) {
    constexpr uint32_t kWaves = kWN * kWT, kRows = 32 * kNT * kWN, kTokens = 32 * kTT * kWT, kTokensLog2 = __builtin_ctz(kTokens);
    constexpr uint32_t kBits = bits_of(kCode), kSteps = 16 / kBits;  // steps of a chunk: 128 bytes of codes are 1024 / kBits columns
    constexpr uint32_t kXBytes = kTokens * 128, kCodeBytes = kRows * 128;
    constexpr uint32_t kXLoads = kTokens / 8 / kWaves, kCodeLoads = kRows / 8 / kWaves;
    static_assert(kXLoads * 8 * kWaves == kTokens && kCodeLoads * 8 * kWaves == kRows, "whole loads of eight rows");
    extern __shared__ char lds[];
    char* const x_img = lds;
    char* const code_img = lds + 2 * kXBytes;

    uint32_t n_tile, p_tile;
    grid.tile(blockIdx.x, &n_tile, &p_tile);
    TileOfPositions at;
    if (!find_tile(a, p_tile, kTokensLog2, &at)) return;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wave_n = wave % kWN, wave_t = wave / kWN, i = lane & 31u, h = lane >> 5;
    const uint32_t out0 = n_tile * (a.gated ? kRows / 2 : kRows);  // the workgroup's first column of y
    const uint32_t steps = (a.cols + 63u) / 64u, last_unit = a.cols / (128u / kBits) - 1u;

    // Row of W behind row r of the workgroup's: of a pair of 32 rows the second are the gated ones of the first.  Rows past the last
    // are the last again and never stored.
    const auto weight_row = [&](uint32_t r) {
        const uint32_t pair = r / 64u, second = r / 32u % 2u;
        return a.gated ? second * a.out_cols + min(out0 + pair * 32u + r % 32u, a.out_cols - 1u) : min(out0 + r, a.out_cols - 1u);
    };
    // Distances in 32 bits from addresses that are the same for the workgroup (the dispatch sees to it that they fit)
    const uint32_t row0 = min(out0, a.out_cols - 1u);
    const char* const words = a.words + at.expert * a.expert_bytes + row0 * a.row_bytes;
    uint32_t code_from[kCodeLoads], code_unit[kCodeLoads];
#pragma unroll
    for (uint32_t q = 0; q < kCodeLoads; q++) {
        const uint32_t r = (q * kWaves + wave) * 8u + lane / 8u;
        code_from[q] = (weight_row(r) - row0) * static_cast<uint32_t>(a.row_bytes);
        code_unit[q] = (lane & 7u) ^ ((r >> 1) & 7u);
    }
    const uint32_t x_row0 = a.row_of ? 0u : at.first;
    const char* const x = a.x + x_row0 * a.x_stride * 2u;
    uint32_t x_from[kXLoads], x_piece[kXLoads];
#pragma unroll
    for (uint32_t q = 0; q < kXLoads; q++) {
        const uint32_t t = (q * kWaves + wave) * 8u + lane / 8u;
        x_from[q] = (row_of_position(a, min(at.first + t, at.last - 1u)) - x_row0) * static_cast<uint32_t>(a.x_stride * 2u);
        x_piece[q] = (lane & 7u) ^ ((t >> 1) & 7u);
    }
    // (scales start on multiples of 4 bytes from an address that is one)
    const uint32_t scale_row0 = a.block_rows ? row0 / a.block_rows : 0u;
    const uint64_t scale_at = (at.expert * a.scale_expert + scale_row0 * a.scale_row) * grid.scale_size + (reinterpret_cast<uintptr_t>(a.scales) & 3u);
    const char* const scales = a.scales - (reinterpret_cast<uintptr_t>(a.scales) & 3u) + (scale_at & ~3ull);
    uint32_t scale_from[kNT];
#pragma unroll
    for (uint32_t n = 0; n < kNT; n++)
        scale_from[n] = static_cast<uint32_t>(scale_at & 3u) +
                        (a.block_rows ? (weight_row((wave_n * kNT + n) * 32u + i) / a.block_rows - scale_row0) * static_cast<uint32_t>(a.scale_row * grid.scale_size) : 0u);

    const auto load_x = [&](uint32_t step, uint32_t into) {
        const char* const from = x + step * 128ull;
        const uint32_t pieces = a.cols / 8u - step * 8u;
#pragma unroll
        for (uint32_t q = 0; q < kXLoads; q++) {
            const char* p = from + (x_from[q] + x_piece[q] * 16u);
            if (pieces < 8u && x_piece[q] >= pieces) p = kZeros;  // columns past the row's end
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(p), CQ_LDS_PTR(x_img + into * kXBytes + (q * kWaves + wave) * 1024u), 16, 0, 0);
        }
    };
    const auto load_codes = [&](uint32_t chunk) {
#pragma unroll
        for (uint32_t q = 0; q < kCodeLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(words + (code_from[q] + min(chunk * 8u + code_unit[q], last_unit) * 16u)),
                                             CQ_LDS_PTR(code_img + (chunk & 1u) * kCodeBytes + (q * kWaves + wave) * 1024u), 16, 0, 0);
    };
    uint32_t scale_words[kNT], scale_offsets[kNT];
    const auto load_scales = [&](uint32_t step) {
        const uint32_t block = grid.halves_per_block.div(min(step * 2u + h, a.cols / 32u - 1u));
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++) {
            scale_offsets[n] = scale_from[n] + block * grid.scale_col_bytes;
            scale_words[n] = scale_word(scales, scale_offsets[n]);
        }
    };
    const auto read_codes = [&](uint32_t step, uint32_t n) {
        const uint32_t r = (wave_n * kNT + n) * 32u + i, chunk = step / kSteps, s = step % kSteps;
        const char* const line = code_img + (chunk & 1u) * kCodeBytes + r * 128u;
        const uint32_t turn = (r >> 1) & 7u;
        Codes<kCode> c;
        if constexpr (kBits == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(line + (s ^ turn) * 16u + h * 8u);
            c.word[0] = w.x, c.word[1] = w.y;
        } else {
            constexpr uint32_t kUnits = kBits / 4;
#pragma unroll
            for (uint32_t u = 0; u < kUnits; u++) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(line + (((s * 2u + h) * kUnits + u) ^ turn) * 16u);
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) c.word[u * 4 + k] = w[k];
            }
        }
        return c;
    };

    f32x16 acc[kNT][kTT] = {};
    u32x4 w[kNT][4];  // the step's weights, by instruction
    Codes<kCode> codes[kNT];
    float rounded_scale[kNT];
    bool all_short = true;
    // codes and scales of a step, on their way to be dequantized; columns past the row's end (the second half of a last step) count nothing
    const auto fetch = [&](uint32_t step) {
        bool mine = true;
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++) {
            codes[n] = read_codes(step, n);
            rounded_scale[n] = dev::round_to<kF>(scale_of(a.param_dtype, scale_words[n], scale_offsets[n]));
            mine = mine && takes_short<kF, kCode>(rounded_scale[n]);
        }
        all_short = kCode > 8 || __builtin_amdgcn_ballot_w64(!mine) == 0;
    };
    const auto dequantize = [&](uint32_t m) {
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++) w[n][m] = slice<kF, kCode, true>(codes[n], m, rounded_scale[n]);
    };
    const auto dequantize_any = [&](uint32_t step) {  // scales that are not ordinary, and the last step where it is a half
        const bool past = step * 2u + h >= a.cols / 32u;
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
            for (uint32_t m = 0; m < 4; m++) {
                w[n][m] = slice<kF, kCode, false>(codes[n], m, rounded_scale[n]);
                if (past) w[n][m] = u32x4{0, 0, 0, 0};
            }
    };

    const auto read_x = [&](uint32_t from, uint32_t m, u32x4* xv) {
#pragma unroll
        for (uint32_t t = 0; t < kTT; t++) {
            const uint32_t row = (wave_t * kTT + t) * 32u + i;
            xv[t] = *reinterpret_cast<const u32x4*>(x_img + from * kXBytes + row * 128u + ((h * 4u + m) ^ ((row >> 1) & 7u)) * 16u);
        }
    };
    // x of a step, codes and scales of the next one are there, and everybody has left the step before, whose places the next loads take
    const auto arrive = [] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    u32x4 xv[2][kTT];
    load_codes(0);
    load_x(0, 0);
    load_scales(0);
    if (kSteps < steps) load_codes(1);
    arrive();
    fetch(0);
    dequantize_any(0);
    load_scales(min(1u, steps - 1u));
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step++) {
        const uint32_t from = step & 1u, next = min(step + 1u, steps - 1u);
        arrive();
        read_x(from, 0, xv[0]);
        fetch(next);
        if (step + 1 < steps) load_x(step + 1, from ^ 1u);
        if ((step + 1) % kSteps == 0 && step + 1 + kSteps < steps) load_codes((step + 1) / kSteps + 1);
        load_scales(min(step + 2u, steps - 1u));
        // the next step's weights take the places of this one's as they are used up
#pragma unroll
        for (uint32_t m = 0; m < 4; m++) {
            if (m < 3) read_x(from, m + 1, xv[(m + 1) & 1]);
#pragma unroll
            for (uint32_t t = 0; t < kTT; t++)
#pragma unroll
                for (uint32_t n = 0; n < kNT; n++) acc[n][t] = mfma<kF>(w[n][m], xv[m & 1][t], acc[n][t]);
            dequantize(m);
        }
        if (!all_short || (next + 1) * 64u > a.cols) dequantize_any(next);
    }

    // Lane (i, h) holds position i of each 32, columns 8 q + 4 h + 0 .. 3 of each 32.  They go through the wave's own part of LDS, 32 positions at a
    // time, so that a lane ends up with eight columns side by side and the activation stands in the code once for every eight values.
    constexpr uint32_t kPitch = 32 * kNT + 4;
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds) + wave * (32 * kPitch);
    const uint32_t columns = a.gated ? 16u * kNT : 32u * kNT, lanes = columns / 8u;  // of a wave; lanes of a position
#pragma unroll
    for (uint32_t t = 0; t < kTT; t++) {
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                *reinterpret_cast<f32x4*>(part + i * kPitch + n * 32 + q * 8 + h * 4) =
                    f32x4{acc[n][t][q * 4], acc[n][t][q * 4 + 1], acc[n][t][q * 4 + 2], acc[n][t][q * 4 + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint32_t p0 = at.first + (wave_t * kTT + t) * 32u;
#pragma unroll 1
        for (uint32_t r = lane / lanes; r < 32; r += 64 / lanes) {
            const uint32_t in = lane % lanes * 8u, col = out0 + wave_n * columns + in;
            if (p0 + r < at.last && col < a.out_cols) finish8(a, at.expert, p0 + r, col, part + r * kPitch + in, part + r * kPitch + 32 + in);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWT>
hipError_t launch_tile(hipStream_t s, const MatmulArgs& a) {
    constexpr uint32_t kRows = 32 * kNT * kWN, kTokens = 32 * kTT * kWT, kLds = 2 * (kRows + kTokens) * 128;
    const auto kernel = matmul_tiles_kernel<kF, kCode, kNT, kTT, kWN, kWT>;
    const uint32_t columns = a.gated ? kRows / 2 : kRows;
    const TilesGrid grid(a, (a.out_cols + columns - 1) / columns, most_tiles(a, __builtin_ctz(kTokens)));
    hipLaunchKernelGGL(kernel, dim3(grid.workgroups()), dim3(64 * kWN * kWT), kLds, s, a, grid);
    return hipGetLastError();
}

template <dev::Float kF, int kCode>
hipError_t launch_shape(hipStream_t s, const MatmulArgs& a, TilesShape shape) {
    switch (shape) {
        case TilesShape::k256x256: return launch_tile<kF, kCode, 2, 4, 4, 2>(s, a);
        case TilesShape::k256x128: return launch_tile<kF, kCode, 2, 4, 4, 1>(s, a);
        case TilesShape::k256x64: return launch_tile<kF, kCode, 2, 2, 4, 1>(s, a);
        case TilesShape::k256x32: return launch_tile<kF, kCode, 2, 1, 4, 1>(s, a);
    }
    return hipErrorInvalidValue;
}

}  // namespace

// One object per type of x and kind of codes, so that a process loads the kernels of its weights.
#define CQ_TILES_NAME2(f, c) matmul_tiles_##f##_##c
#define CQ_TILES_NAME(f, c) CQ_TILES_NAME2(f, c)
hipError_t CQ_TILES_NAME(CQ_TU_FLOAT, CQ_TU_CODE)(hipStream_t s, const MatmulArgs& a, TilesShape shape) {
    return launch_shape<dev::Float::CQ_TU_FLOAT, CQ_TU_CODE>(s, a, shape);
}

}  // namespace cq
