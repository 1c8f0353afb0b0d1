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
//
// Bound by power on large products (bf16 e2m1 [28672, 8192], 4096 tokens 1.83 ms, 1.05 PFLOP/s at 1.6 GHz; 1.73 without the dequantization, 1.86 without
// the reads of x).  Smaller ones by their steps' loads, dequantization and barriers side by side, which half the positions hardly shorten, and by what a
// workgroup takes before its first products and after its last ones: 64 experts [2816, 2048] f16 8 bits gated, 6126 positions 173 us, a fifth of it in
// front and behind, the matrix units busy for a quarter.  Codes of 8 bits are waited for in every step, as a line of 64 bytes holds one.  256 x 128 rather than 256 x 256 or 512 x 128: two workgroups on a compute unit, no slower; rather than
// one wave of 64 x 256 per SIMD: 2.09 ms.
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

// kNT, kTT: tiles of 32 rows and 32 positions of a wave; kWN, kWK: waves along rows and columns.  Waves along the columns take a run of chunks
// each, with images of their own; their sums meet in LDS at the end.  Several workgroups may share the columns too: then they leave their sums in the
// workspace, and matmul_finish_kernel adds them up.
template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWK, int kLine>
__global__ __launch_bounds__(64 * kWN * kWK, (TilesTraits<kNT, kTT, kWN, kWK, kLine>::kWavesPerSimd)) void matmul_tiles_kernel(MatmulArgs a, TilesGrid grid) {
    using Traits = TilesTraits<kNT, kTT, kWN, kWK, kLine>;
    constexpr uint32_t kWaves = kWN, kRows = Traits::kRows, kTokens = Traits::kTokens, kTokensLog2 = __builtin_ctz(kTokens);
    constexpr uint32_t kBits = bits_of(kCode), kSteps = kLine / 8 / kBits;  // steps of a chunk: 128 bytes of codes are 1024 / kBits columns
    constexpr uint32_t kUnits = kLine / 16, kTurn = 256 / kLine;            // 16-byte pieces of a line; rows side by side in the 256 bytes of all banks
    static_assert(kSteps >= 1, "whole steps");
    constexpr uint32_t kXRing = Traits::kXRing, kCodeRing = Traits::kCodeRing;
    constexpr uint32_t kXBytes = Traits::kXBytes, kCodeBytes = Traits::kCodeBytes;
    constexpr uint32_t kXLoads = kTokens / 8 / kWaves, kCodeLoads = kCodeBytes / 1024 / kWaves, kScaleLoads = kRows * 2 / 64 / kWaves;
    static_assert(kXLoads * 8 * kWaves == kTokens && kCodeLoads * 1024 * kWaves == kCodeBytes && kScaleLoads * 32 * kWaves == kRows, "whole loads of 1 KiB");
    extern __shared__ char lds[];

    uint32_t n_tile, p_tile;
    TileOfPositions at;
    if (!grid.tile(blockIdx.x, &n_tile, &p_tile) || !find_tile(a, p_tile, kTokensLog2, &at)) return;
    const uint32_t lane = threadIdx.x & 63u, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wave = any_wave % kWaves, wave_k = any_wave / kWaves;
    const uint32_t i = lane & 31u, h = lane >> 5;
    const uint32_t positions = at.last - at.first;
    const uint32_t out0 = n_tile * (a.gated ? kRows / 2 : kRows);  // the workgroup's first column of y
    const uint32_t last_unit = a.cols / (128u / kBits) - 1u;
    char* const x_img = lds + wave_k * Traits::kImage;
    char* const code_img = x_img + kXRing * kXBytes;
    char* const scale_img = code_img + kCodeRing * kCodeBytes;

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
        x_piece[q] = (lane & 7u) ^ ((t >> 1) & 7u);
        x_from[q] = (row_of_position(a, min(at.first + t, at.last - 1u)) - x_row0) * static_cast<uint32_t>(a.x_stride * 2u) + x_piece[q] * 16u;
    }
    // (scales start on multiples of 4 bytes from an address that is one)
    const uint32_t scale_row0 = a.block_rows ? row0 / a.block_rows : 0u;
    const uint64_t scale_at = (at.expert * a.scale_expert + scale_row0 * a.scale_row) * grid.scale_size + (reinterpret_cast<uintptr_t>(a.scales) & 3u);
    const char* const scales = a.scales - (reinterpret_cast<uintptr_t>(a.scales) & 3u) + (scale_at & ~3ull);
    // a step's scales lie [row][half of its columns], a word around each
    const auto scale_row = [&](uint32_t r) {
        return static_cast<uint32_t>(scale_at & 3u) +
               (a.block_rows ? (weight_row(r) / a.block_rows - scale_row0) * static_cast<uint32_t>(a.scale_row * grid.scale_size) : 0u);
    };
    uint32_t scale_from[kScaleLoads], scale_own[kNT];
#pragma unroll
    for (uint32_t q = 0; q < kScaleLoads; q++) scale_from[q] = scale_row((q * kWaves + wave) * 32u + lane / 2u);
#pragma unroll
    for (uint32_t n = 0; n < kNT; n++) scale_own[n] = scale_row((wave * kNT + n) * 32u + i);
    const auto scale_block = [&](uint32_t step, uint32_t half) { return grid.block_of(min(step * 2u + half, a.cols / 32u - 1u)) * grid.scale_col_bytes; };

    const auto load_x = [&](uint32_t step, uint32_t into) {
        const char* const from = x + step * 128ull;
        const uint32_t pieces = a.cols / 8u - step * 8u;
        const auto load = [&](auto all) {
#pragma unroll
            for (uint32_t q = 0; q < kXLoads; q++) {
                // positions that the tile does not have leave what was there: they have columns of their own in every product
                if (kTokens <= 64 && (q * kWaves + wave) * 8u >= positions) continue;
                const char* p = from + x_from[q];
                if (!decltype(all)::value && x_piece[q] >= pieces) p = kZeros;  // columns past the row's end
                __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(p), CQ_LDS_PTR(x_img + into * kXBytes + (q * kWaves + wave) * 1024u), 16, 0, 0);
            }
        };
        if (pieces >= 8u)
            load(std::true_type{});
        else
            load(std::false_type{});
    };
    const auto load_codes = [&](uint32_t chunk, uint32_t into) {
#pragma unroll
        for (uint32_t q = 0; q < kCodeLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(words + (code_from[q] + min(chunk * kUnits + code_unit[q], last_unit) * 16u)),
                                             CQ_LDS_PTR(code_img + into * kCodeBytes + (q * kWaves + wave) * 1024u), 16, 0, 0);
    };
    const auto load_scales = [&](uint32_t step, uint32_t into) {
        const uint32_t block = scale_block(step, lane & 1u);
#pragma unroll
        for (uint32_t q = 0; q < kScaleLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(scales + ((scale_from[q] + block) & ~3u)),
                                             CQ_LDS_PTR(scale_img + into * Traits::kScaleBytes + (q * kWaves + wave) * 256u), 4, 0, 0);
    };
    // `in`: a step of the wave's run, from 0 on
    const auto read_codes = [&](uint32_t in, uint32_t n) {
        const uint32_t r = (wave * kNT + n) * 32u + i, s = in % kSteps;
        const char* const line = code_img + in / kSteps % kCodeRing * kCodeBytes + r * kLine;
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

    const ScaleMasks masks(a.param_dtype);
    f32x16 acc[kNT][kTT] = {};
    u32x4 w[kNT][4];  // the step's weights, by instruction
    Codes<kCode> codes[kNT];
    float rounded_scale[kNT];
    bool all_short = true;
    const auto fetch = [&](uint32_t in) __attribute__((always_inline)) {  // codes and scales of a step, to be dequantized
        bool mine = true;
        const uint32_t block = scale_block(first_step + in, h);
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++) {
            codes[n] = read_codes(in, n);
            const uint32_t word = *reinterpret_cast<const uint32_t*>(scale_img + in % Traits::kScaleRing * Traits::kScaleBytes + ((wave * kNT + n) * 32u + i) * 8u + h * 4u);
            rounded_scale[n] = dev::round_to<kF>(scale_of(masks, word, scale_own[n] + block));
            mine = mine && takes_short<kF, kCode>(rounded_scale[n]);
        }
        all_short = kCode > 8 || __builtin_amdgcn_ballot_w64(!mine) == 0;
    };
    const auto dequantize = [&](uint32_t m) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t n = 0; n < kNT; n++) w[n][m] = slice<kF, kCode, true>(codes[n], m, rounded_scale[n]);
    };
    // What the short way does not do: scales that are not ordinary; and where the row ends in the middle of a step, whose second half counts
    // nothing.
    const auto amend = [&](uint32_t step) __attribute__((always_inline)) {
        if (kCode <= 8 && !all_short) {
#pragma unroll
            for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
                for (uint32_t m = 0; m < 4; m++) w[n][m] = slice<kF, kCode, false>(codes[n], m, rounded_scale[n]);
        }
        if ((step + 1) * 64u > a.cols) {
#pragma unroll
            for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
                for (uint32_t m = 0; m < 4; m++) w[n][m] = h == 1 ? u32x4{0, 0, 0, 0} : w[n][m];
        }
    };
    const auto read_x = [&](auto tiles, uint32_t from, uint32_t m, u32x4* xv) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t t = 0; t < decltype(tiles)::value; t++) {
            const uint32_t row = t * 32u + i;
            xv[t] = *reinterpret_cast<const u32x4*>(x_img + from * kXBytes + row * 128u + ((h * 4u + m) ^ ((row >> 1) & 7u)) * 16u);
        }
    };
    // What is asked for in an iteration: scales three steps ahead, x kXAhead steps ahead, and in the last step of a chunk the chunk that comes
    // kCodeRing - 1 behind the next one's; all into places whose last reader was done an iteration before.
    constexpr uint32_t kXAhead = kXRing - 1, kCodeLead = (kCodeRing - 1) * kSteps;  // iterations until a chunk is read
    const auto begin = [](auto outstanding) {
        // everybody's loads up to those that may still be on their way are there, and everybody has left the iteration before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(outstanding)::value) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    bool codes_after_x = false;  // a chunk's loads were issued behind the x that an iteration waits for, and are not wanted yet
    const auto issue = [&](uint32_t in) __attribute__((always_inline)) {
        if (in + 3 < steps) load_scales(first_step + in + 3, (in + 3) % Traits::kScaleRing);
        if (in + kXAhead < steps) load_x(first_step + in + kXAhead, (in + kXAhead) % kXRing);
        const uint32_t chunk = (in + 1) / kSteps - 1 + kCodeRing;
        codes_after_x = (in + 1) % kSteps == 0 && chunk * kSteps < steps;
        if (codes_after_x) load_codes(first_chunk + chunk, chunk % kCodeRing);
    };
    u32x4 xv[2][kTT];
#pragma unroll
    for (uint32_t k = 0; k < kCodeRing; k++)
        if (k * kSteps < steps) load_codes(first_chunk + k, k);
#pragma unroll
    for (uint32_t k = 0; k < 3; k++)
        if (k < steps) load_scales(first_step + k, k);
#pragma unroll
    for (uint32_t k = 0; k < kXAhead; k++)
        if (k < steps) load_x(first_step + k, k);
    begin(std::integral_constant<int, 0>{});
    if (kWK == 1 || steps != 0) {
        fetch(0);
#pragma unroll
        for (uint32_t m = 0; m < 4; m++) dequantize(m);
        amend(first_step);
    }
    // The steps, for all tiles of 32 positions or for the first half of them, where an expert's last positions need no more (64 experts with 25
    // positions each, [10707, 608] 4 bits, 149 -> 133 us; a version for three of four would leave the sums no registers).
    const auto run = [&](auto tiles) __attribute__((always_inline)) {
        constexpr uint32_t kHave = decltype(tiles)::value;
#pragma unroll 1
        for (uint32_t in = 0; in < rounds; in++) {
            static_assert(kXAhead == 1, "the x of an iteration is what the one before asked for");
            if (kCodeLead >= 2 && codes_after_x)
                begin(std::integral_constant<int, kCodeLoads>{});
            else
                begin(std::integral_constant<int, 0>{});
            codes_after_x = false;
            if (kWK > 1 && in >= steps) continue;  // waves along the columns may have a chunk less than others
            const uint32_t next = min(in + 1u, steps - 1u);
            read_x(tiles, in % kXRing, 0, xv[0]);
            fetch(next);
            issue(in);
            // the next step's weights take the places of this one's as they are used up
#pragma unroll
            for (uint32_t m = 0; m < 4; m++) {
                if (m < 3) read_x(tiles, in % kXRing, m + 1, xv[(m + 1) & 1]);
#pragma unroll
                for (uint32_t t = 0; t < kHave; t++)
#pragma unroll
                    for (uint32_t n = 0; n < kNT; n++) acc[n][t] = mfma<kF>(w[n][m], xv[m & 1][t], acc[n][t]);
                dequantize(m);
            }
            if constexpr (kHave >= 4 && kCode != 8) {
                // A matrix instruction keeps its unit busy for 32 cycles, in which the wave may issue seven others; x of the next products comes in front of
                // the next weights ([28672, 8192] 4 bits, 4096 positions 1.96 -> 1.88 ms; the 8-bit fields have no registers left for it).
#pragma unroll
                for (uint32_t k = 0; k < 4 * kNT * kHave; k++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
                    if (k % (kNT * kHave) < kHave) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
            }
            amend(first_step + next);
        }
    };
    const uint32_t have = min((positions + 31u) / 32u, static_cast<uint32_t>(kTT));
    if (kTT == 1 || have > kTT / 2u)
        run(std::integral_constant<int, kTT>{});
    else if constexpr (kTT > 1)
        run(std::integral_constant<int, kTT / 2>{});

    // Lane (i, h) holds position i of each 32, rows 8 q + 4 h + 0 .. 3 of each 32.  They go through the wave's own part of LDS, 32 positions at a
    // time, so that a lane ends up with eight columns side by side, the waves along the columns meet, and the activation stands in the
    // code once for every eight values.
    constexpr uint32_t kPitch = Traits::kPitch, kPart = 32 * kPitch;
    float* const part = reinterpret_cast<float*>(lds) + any_wave * kPart;
    float* const parts_of = reinterpret_cast<float*>(lds) + wave * kPart;  // those of the other waves along the columns behind it
    const bool pairs = a.gated && grid.splits == 1;                        // (with shared columns the rows are stored as they are)
    const uint32_t columns = pairs ? 16u * kNT : 32u * kNT, lanes = columns / 8u;
    const uint32_t in = lane % lanes * 8u, own_col = out0 + wave * columns + in;
    f32x8 bias = {}, bias_up = {};
    if (grid.splits == 1 && own_col < a.out_cols) {
        bias = load_bias8(a, at.expert, own_col);
        if (a.gated) bias_up = load_bias8(a, at.expert, a.out_cols + own_col);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t t = 0; t < kTT; t++) {
        if (kTT > 1 && t >= have) break;
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
        const uint32_t p0 = at.first + t * 32u;
#pragma unroll 1
        for (uint32_t r = (wave_k * 64u + lane) / lanes; r < 32; r += 64u * kWK / lanes) {
            const uint32_t p = p0 + r;
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
                const uint32_t row = wave * 32u * kNT + in, col = a.gated ? out0 + row / 32u * 16u + row % 16u : out0 + row;
                if (col >= a.out_cols) continue;
                const f32x8 v = sum_at(from);
                float* const to = static_cast<float*>(a.workspace) +
                                  (static_cast<uint64_t>(blockIdx.y) * a.positions + p) * grid.pitch + col + (a.gated && row % 32u >= 16u ? grid.pitch / 2 : 0u);
                *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};  // (the pitch has room for whole eights)
                *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                if (own_col < a.out_cols) finish8(a, p, own_col, sum_at(from) + bias, a.gated ? sum_at(from + 16) + bias_up : f32x8{});
            }
        }
        if (kWK == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kWN, int kWK, int kLine>
hipError_t launch_tile(hipStream_t s, const MatmulArgs& a, uint32_t splits) {
    using Traits = TilesTraits<kNT, kTT, kWN, kWK, kLine>;
    const TilesGrid grid(a, Traits::kRows, Traits::kTokens, splits);
    hipLaunchKernelGGL((matmul_tiles_kernel<kF, kCode, kNT, kTT, kWN, kWK, kLine>), dim3(grid.workgroups(), splits), dim3(64 * kWN * kWK), Traits::kLds, s, a, grid);
    return hipGetLastError();
}

template <dev::Float kF, int kCode>
hipError_t launch_shape(hipStream_t s, const MatmulArgs& a, const TilesChoice& c) {
    switch (c.shape) {
        case TilesShape::k256x128: return launch_tile<kF, kCode, 2, 4, 4, 1, 64>(s, a, c.splits);
        case TilesShape::k256x128x2: return launch_tile<kF, kCode, 2, 4, 4, 2, 64>(s, a, c.splits);
        case TilesShape::k128x64: return launch_tile<kF, kCode, 1, 2, 4, 2, 64>(s, a, c.splits);
        case TilesShape::k128x32: return launch_tile<kF, kCode, 1, 1, 4, 2, 64>(s, a, c.splits);
        case TilesShape::k32x32: return launch_tile<kF, kCode, 1, 1, 1, 8, 128>(s, a, c.splits);
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
