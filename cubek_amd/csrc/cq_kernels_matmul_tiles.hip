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

// kNT, kTT: tiles of 32 rows and 32 positions of a wave; kWN, kWT, kWK: waves along rows, positions and columns.  Waves along the columns
// take a run of chunks each, with images of their own; their sums meet in LDS at the end.  Several workgroups may share the columns too: then they
// leave their sums in the workspace, and matmul_finish_kernel adds them up.
template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWT, int kWK, int kLine>
__global__ __launch_bounds__(64 * kWN * kWT * kWK, (TilesTraits<kNT, kTT, kWN, kWT, kWK, kLine>::kWavesPerSimd)) void matmul_tiles_kernel(MatmulArgs a, TilesGrid grid) {
    using Traits = TilesTraits<kNT, kTT, kWN, kWT, kWK, kLine>;
    constexpr uint32_t kWaves = kWN * kWT, kRows = Traits::kRows, kTokens = Traits::kTokens, kTokensLog2 = __builtin_ctz(kTokens);
    constexpr uint32_t kBits = bits_of(kCode), kSteps = kLine / 8 / kBits;  // steps of a chunk: 128 bytes of codes are 1024 / kBits columns
    constexpr uint32_t kUnits = kLine / 16, kTurn = 256 / kLine;            // 16-byte pieces of a line; rows side by side in the 256 bytes of all banks
    static_assert(kSteps >= 1, "whole steps");
    constexpr uint32_t kXBytes = Traits::kXBytes, kCodeBytes = Traits::kCodeBytes;
    constexpr uint32_t kXLoads = kTokens / 8 / kWaves, kCodeLoads = kCodeBytes / 1024 / kWaves;
    static_assert(kXLoads * 8 * kWaves == kTokens && kCodeLoads * 1024 * kWaves == kCodeBytes, "whole loads of 1 KiB");
    extern __shared__ char lds[];

    uint32_t n_tile, p_tile;
    grid.tile(blockIdx.x, &n_tile, &p_tile);
    TileOfPositions at;
    if (!find_tile(a, p_tile, kTokensLog2, &at)) return;
    const uint32_t lane = threadIdx.x & 63u, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wave = any_wave % kWaves, wave_k = any_wave / kWaves;
    const uint32_t wave_n = wave % kWN, wave_t = wave / kWN, i = lane & 31u, h = lane >> 5;
    const uint32_t positions = at.last - at.first;
    const uint32_t out0 = n_tile * (a.gated ? kRows / 2 : kRows);  // the workgroup's first column of y
    const uint32_t last_unit = a.cols / (128u / kBits) - 1u;
    char* const x_img = lds + wave_k * (2 * kXBytes + 2 * kCodeBytes);
    char* const code_img = x_img + 2 * kXBytes;

    // this wave's run of chunks, and the steps that the workgroup's longest one has
    const uint32_t all_steps = (a.cols + 63u) / 64u, chunks = (all_steps + kSteps - 1u) / kSteps;
    const uint32_t parts = grid.splits * kWK, my_part = blockIdx.y * kWK + wave_k;
    const uint32_t first_chunk = chunks * my_part / parts, first_step = first_chunk * kSteps;
    const uint32_t last_step = min(all_steps, chunks * (my_part + 1u) / parts * kSteps), steps = last_step > first_step ? last_step - first_step : 0u;
    const uint32_t rounds = kWK == 1 ? steps : (chunks + parts - 1u) / parts * kSteps;

    // Row of W behind row r of the workgroup's: gated, the second 16 of each 32 belong to the first.  Rows past the last are the last again
    // and never stored.
    const auto weight_row = [&](uint32_t r) {
        return a.gated ? (r / 16u % 2u) * a.out_cols + min(out0 + r / 32u * 16u + r % 16u, a.out_cols - 1u) : min(out0 + r, a.out_cols - 1u);
    };
    // Distances in 32 bits from addresses that are the same for the workgroup (the dispatch sees to it that they fit)
    const uint32_t row0 = min(out0, a.out_cols - 1u);
    const char* const words = a.words + at.expert * a.expert_bytes + row0 * a.row_bytes;
    uint32_t code_from[kCodeLoads], code_unit[kCodeLoads];
#pragma unroll
    for (uint32_t q = 0; q < kCodeLoads; q++) {
        const uint32_t r = ((q * kWaves + wave) * 64u + lane) / kUnits;
        code_from[q] = (weight_row(r) - row0) * static_cast<uint32_t>(a.row_bytes);
        code_unit[q] = (lane % kUnits) ^ (r / kTurn % kUnits);
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
            // positions that the tile does not have leave what was there: they have columns of their own in every product
            if (kTokens <= 64 && (q * kWaves + wave) * 8u >= positions) continue;
            const char* p = from + (x_from[q] + x_piece[q] * 16u);
            if (pieces < 8u && x_piece[q] >= pieces) p = kZeros;  // columns past the row's end
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(p), CQ_LDS_PTR(x_img + into * kXBytes + (q * kWaves + wave) * 1024u), 16, 0, 0);
        }
    };
    const auto load_codes = [&](uint32_t chunk) {
#pragma unroll
        for (uint32_t q = 0; q < kCodeLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(words + (code_from[q] + min(chunk * kUnits + code_unit[q], last_unit) * 16u)),
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
        const char* const line = code_img + (chunk & 1u) * kCodeBytes + r * kLine;
        const uint32_t turn = r / kTurn % kUnits;
        Codes<kCode> c;
        if constexpr (kBits == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(line + (s ^ turn) * 16u + h * 8u);
            c.word[0] = w.x, c.word[1] = w.y;
        } else {
            constexpr uint32_t kOwn = kBits / 4;  // 32 columns
#pragma unroll
            for (uint32_t u = 0; u < kOwn; u++) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(line + (((s * 2u + h) * kOwn + u) ^ turn) * 16u);
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
    const auto fetch = [&](uint32_t step) {  // codes and scales of a step, to be dequantized
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
    if (kWK == 1 || steps != 0) {
        load_codes(first_chunk);
        load_x(first_step, 0);
        load_scales(first_step);
        if (kSteps < steps) load_codes(first_chunk + 1u);
    }
    arrive();
    if (kWK == 1 || steps != 0) {
        fetch(first_step);
        dequantize_any(first_step);
        load_scales(first_step + min(1u, steps - 1u));
    }
#pragma unroll 1
    for (uint32_t n_step = 0; n_step < rounds; n_step++) {
        arrive();
        if (kWK > 1 && n_step >= steps) continue;  // waves along the columns may have a chunk less than others
        const uint32_t from = n_step & 1u, next = first_step + min(n_step + 1u, steps - 1u);
        read_x(from, 0, xv[0]);
        fetch(next);
        if (n_step + 1 < steps) load_x(next, from ^ 1u);
        if ((n_step + 1) % kSteps == 0 && n_step + 1 + kSteps < steps) load_codes(first_chunk + (n_step + 1) / kSteps + 1);
        load_scales(first_step + min(n_step + 2u, steps - 1u));
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

    // Lane (i, h) holds position i of each 32, rows 8 q + 4 h + 0 .. 3 of each 32.  They go through the wave's own part of LDS, 32 positions at a
    // time, so that a lane ends up with eight columns side by side, the waves along the columns meet, and the activation stands in the
    // code once for every eight values.
    constexpr uint32_t kPitch = Traits::kPitch, kPart = 32 * kPitch;
    float* const part = reinterpret_cast<float*>(lds) + any_wave * kPart;
    float* const parts_of = reinterpret_cast<float*>(lds) + wave * kPart;  // those of the other waves along the columns behind it
    const bool pairs = a.gated && grid.splits == 1;                        // (with shared columns the rows are stored as they are)
    const uint32_t columns = pairs ? 16u * kNT : 32u * kNT, lanes = columns / 8u;
    __syncthreads();
#pragma unroll
    for (uint32_t t = 0; t < kTT; t++) {
        if (t != 0 && kWK > 1) __syncthreads();
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                *reinterpret_cast<f32x4*>(part + i * kPitch + n * 32 + q * 8 + h * 4) =
                    f32x4{acc[n][t][q * 4], acc[n][t][q * 4 + 1], acc[n][t][q * 4 + 2], acc[n][t][q * 4 + 3]};
        if (kWK > 1)
            __syncthreads();
        else
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint32_t p0 = at.first + (wave_t * kTT + t) * 32u;
#pragma unroll 1
        for (uint32_t r = (wave_k * 64u + lane) / lanes; r < 32; r += 64u * kWK / lanes) {
            const uint32_t in = lane % lanes * 8u, p = p0 + r;
            if (p >= at.last) continue;
            const float* const from = parts_of + r * kPitch + (pairs ? in / 16u * 32u + in % 16u : in);
            const auto sum_at = [&](const float* at_part) {
                f32x8 v = load8(at_part);
#pragma unroll
                for (uint32_t k = 1; k < kWK; k++) v += load8(at_part + k * (kWaves * kPart));
                return v;
            };
            if (grid.splits > 1) {
                // [part][position][row of W]: gated, 16 columns and then their 16 gated ones
                const uint32_t row = wave_n * 32u * kNT + in, col = a.gated ? out0 + row / 32u * 16u + row % 16u : out0 + row;
                if (col >= a.out_cols) continue;
                const f32x8 v = sum_at(from);
                float* const to = static_cast<float*>(a.workspace) +
                                  (static_cast<uint64_t>(blockIdx.y) * a.positions + p) * grid.pitch + col + (a.gated && row % 32u >= 16u ? grid.pitch / 2 : 0u);
                *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};  // (the pitch has room for whole eights)
                *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                const uint32_t col = out0 + wave_n * columns + in;
                if (col < a.out_cols) finish8(a, at.expert, p, col, sum_at(from), a.gated ? sum_at(from + 16) : f32x8{});
            }
        }
        if (kWK == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWT, int kWK, int kLine>
hipError_t launch_tile(hipStream_t s, const MatmulArgs& a, uint32_t splits) {
    using Traits = TilesTraits<kNT, kTT, kWN, kWT, kWK, kLine>;
    const TilesGrid grid(a, Traits::kRows, Traits::kTokens, splits);
    hipLaunchKernelGGL((matmul_tiles_kernel<kF, kCode, kNT, kTT, kWN, kWT, kWK, kLine>), dim3(grid.workgroups(), splits), dim3(64 * kWN * kWT * kWK), Traits::kLds, s, a, grid);
    return hipGetLastError();
}

template <dev::Float kF, int kCode>
hipError_t launch_shape(hipStream_t s, const MatmulArgs& a, const TilesChoice& c) {
    switch (c.shape) {
        case TilesShape::k256x128: return launch_tile<kF, kCode, 2, 4, 4, 1, 1, 64>(s, a, c.splits);
        case TilesShape::k128x64: return launch_tile<kF, kCode, 1, 2, 4, 1, 2, 64>(s, a, c.splits);
        case TilesShape::k128x32: return launch_tile<kF, kCode, 1, 1, 4, 1, 2, 64>(s, a, c.splits);
        case TilesShape::k32x32: return launch_tile<kF, kCode, 1, 1, 1, 1, 8, 128>(s, a, c.splits);
    }
    return hipErrorInvalidValue;
}

}  // namespace

// One object per type of x and kind of codes, so that a process loads the kernels of its weights.
#define CQ_TILES_NAME2(f, c) matmul_tiles_##f##_##c
#define CQ_TILES_NAME(f, c) CQ_TILES_NAME2(f, c)
hipError_t CQ_TILES_NAME(CQ_TU_FLOAT, CQ_TU_CODE)(hipStream_t s, const MatmulArgs& a, const TilesChoice& choice) {
    return launch_shape<dev::Float::CQ_TU_FLOAT, CQ_TU_CODE>(s, a, choice);
}

}  // namespace cq
