// Products with quantized weights for up to 32 positions of an expert (or of the whole product): a decode step.
//
// A wave takes 16 or 32 rows of W (gated: 16 and their gated ones) and a share of their columns, in stages of a line of 128 bytes of every
// row or of half a line (FewShape).  Codes, scales and x of a stage come into LDS by direct loads, kAhead stages ahead: codes and scales into
// the wave's own part, x into one that the waves of a share have together.  16 x 16 x 32 matrix instructions take lane (i, g)'s eight columns
// of row i, and the same of token i.  The eight waves of a workgroup are one to eight groups of rows by eight to one shares of the columns; the shares' sums meet
// in LDS at the end.  Bound by the read of W and the instructions of its dequantization side by side, and in launches of few stages by the
// time from a workgroup's start to its first stage and from its last one to its sums.
//
// bf16, 4 bits: one token on [4096, 4096] 5.6 us (a launch 3.5), on [28672, 8192] 35, 16 tokens 37; 32 positions of eight experts [28672, 4096]
// gated 127 us, 4.6 TB/s, with 2.4 vector instructions per weight; 24 tokens on [28672, 4096] f16 gated 25 us, twice its read: 224 workgroups, each
// with one stage of 20 KiB of codes and scales on its way, wait for memory.
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

// kNT: groups of 16 rows of a wave; kTT: groups of 16 positions; kUnits: units of a row in a stage; kX: loads of 1 KiB by which a wave takes part in a stage of its share's x.
template <dev::Float kF, int kCode, int kNT, int kTT, int kUnits, int kX>
__global__ __launch_bounds__(512) void matmul_few_kernel(MatmulArgs a, FewGrid grid) {
    constexpr uint32_t kBits = bits_of(kCode), kUnit = 128 / kBits;  // columns of 16 bytes of codes
    constexpr uint32_t kQ = kUnits / 4, kM = kUnit / 8, kPieces = kUnits * kM;  // a lane's units; matrix instructions of one; 16-byte pieces of x of a token
    constexpr uint32_t kCodeBytes = kNT * 16 * kUnits * 16, kSlot = kCodeBytes + kNT * 16 * kUnits * 4, kAhead = kFewAhead, kRing = kAhead + 1;
    constexpr uint32_t kCodeLoads = kCodeBytes / 1024, kScaleLoads = kNT * kUnits / 4, kLoads = kCodeLoads + kScaleLoads + kX;
    extern __shared__ char lds[];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t i = lane & 15u, g = lane >> 4;
    const uint32_t shares_log2 = grid.shares_log2, shares = 1u << shares_log2, share = wave & (shares - 1u), group = wave >> shares_log2, groups = 8u >> shares_log2;
    char* const x_img = lds + share * (kRing * grid.x_bytes);
    char* const mine = lds + shares * (kRing * grid.x_bytes) + wave * (kRing * kSlot);

    TileOfPositions at;
    if (!find_tile(a, blockIdx.y, grid.tokens_log2, &at)) return;
    const uint32_t tokens = at.last - at.first;
    constexpr uint32_t kPlainRows = 16 * kNT;
    const uint32_t wave_rows = a.gated ? kPlainRows / 2 : kPlainRows;  // columns of y of a wave
    const uint32_t row0 = min((blockIdx.x * groups + group) * wave_rows, a.out_cols - 1u);
    // rows past the last are the last again and never stored; gated: the second 16 belong to the first
    const auto weight_row = [&](uint32_t r) {
        return a.gated ? min(row0 + r % 16u, a.out_cols - 1u) + r / 16u * a.out_cols : min(row0 + r, a.out_cols - 1u);
    };
    const uint32_t units = a.cols / kUnit, stages = (units + kUnits - 1u) / kUnits;
    const char* const words = a.words + at.expert * a.expert_bytes + row0 * a.row_bytes;
    const uint32_t scale_row0 = a.block_rows ? row0 / a.block_rows : 0u;
    const uint64_t scale_at = (at.expert * a.scale_expert + scale_row0 * a.scale_row) * grid.scale_size + (reinterpret_cast<uintptr_t>(a.scales) & 3u);
    const char* const scales = a.scales - (reinterpret_cast<uintptr_t>(a.scales) & 3u) + (scale_at & ~3ull);
    const uint32_t scale_base = static_cast<uint32_t>(scale_at & 3u);
    const auto scale_row_of = [&](uint32_t r) {
        return scale_base + (a.block_rows ? (weight_row(r) / a.block_rows - scale_row0) * static_cast<uint32_t>(a.scale_row * grid.scale_size) : 0u);
    };

    // Where a lane's pieces come from.  Codes: place p of row r holds unit p ^ (r / 2 % 8), of half lines p ^ (r / 4 % 4); scales: place u of row
    // r that of unit u; x: place p of token v piece p ^ (v % 16), of fewer than 16 pieces p ^ (v / 2 % 8): sixteen lanes' reads fall on
    // different banks.  Positions past the last are the last again.
    const auto code_turn = [](uint32_t r) { return kUnits == 8 ? (r >> 1) & 7u : (r >> 2) & 3u; };
    const auto x_turn = [](uint32_t v) { return kPieces >= 16 ? v & 15u : (v >> 1) & 7u; };
    uint32_t code_from[kCodeLoads], code_unit[kCodeLoads], scale_from[kScaleLoads], x_to[kX], x_from[kX];
    const uint32_t x_row0 = a.row_of ? 0u : at.first;
    const char* const x = a.x + x_row0 * a.x_stride * 2u;
#pragma unroll
    for (uint32_t q = 0; q < kCodeLoads; q++) {
        const uint32_t r = (q * 64u + lane) / kUnits;
        code_unit[q] = (lane % kUnits) ^ code_turn(r);
        code_from[q] = (weight_row(r) - row0) * static_cast<uint32_t>(a.row_bytes);
    }
#pragma unroll
    for (uint32_t q = 0; q < kScaleLoads; q++) scale_from[q] = scale_row_of((q * 64u + lane) / kUnits);
    const auto x_token = [&](uint32_t q, uint32_t lane) { return min((x_to[q] / 16u + lane) / kPieces, tokens - 1u); };
    const auto x_piece = [&](uint32_t q, uint32_t lane) { return lane % kPieces ^ x_turn(x_token(q, lane)); };
#pragma unroll
    for (uint32_t q = 0; q < kX; q++) {
        x_to[q] = min(q * groups + group, grid.x_bytes / 1024u - 1u) * 1024u;  // (some waves may bring the last one together)
        x_from[q] = (row_of_position(a, at.first + x_token(q, lane)) - x_row0) * static_cast<uint32_t>(a.x_stride * 2u) + x_piece(q, lane) * 16u;
    }
    const auto load = [&](uint32_t stage, uint32_t slot) {
        char* const to = mine + slot * kSlot;
        const uint32_t unit0 = stage * kUnits;
#pragma unroll
        for (uint32_t q = 0; q < kCodeLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(words + (code_from[q] + min(unit0 + code_unit[q], units - 1u) * 16u)),
                                             CQ_LDS_PTR(to + q * 1024u), 16, 0, kUnits == 8 ? 2 : 0 /* whole lines past the caches */);
        const uint32_t block = grid.block_of(min(unit0 + lane % kUnits, units - 1u)) * grid.scale_col_bytes;
#pragma unroll
        for (uint32_t q = 0; q < kScaleLoads; q++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(scales + ((scale_from[q] + block) & ~3u)), CQ_LDS_PTR(to + kCodeBytes + q * 256u), 4, 0, 0);
        const char* const from = x + static_cast<uint64_t>(unit0) * (kM * 16u);
        const uint32_t pieces = (units - unit0) * kM;
#pragma unroll
        for (uint32_t q = 0; q < kX; q++) {
            const char* p = from + x_from[q];
            if (pieces < kPieces) {  // columns past the row's end; the piece is worked out again here, so that no register holds it in the loop
                uint32_t again = lane;
                asm volatile("" : "+v"(again));
                if (x_piece(q, again) >= pieces) p = kZeros;
            }
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const u32x4*>(p), CQ_LDS_PTR(x_img + slot * grid.x_bytes + x_to[q]), 16, 0, 0);
        }
    };

    const ScaleMasks masks(a.param_dtype);
    f32x4 acc[kNT][kTT][2] = {};
    uint32_t scale_of_row[kNT], column[kTT];
#pragma unroll
    for (uint32_t n = 0; n < kNT; n++) scale_of_row[n] = scale_row_of(n * 16u + i);
#pragma unroll
    for (uint32_t t = 0; t < kTT; t++) column[t] = min(t * 16u + i, tokens - 1u);
    const uint32_t rounds = (stages + shares - 1u) >> shares_log2;
    const auto stage_of = [&](uint32_t n) { return min(share + (n << shares_log2), stages - 1u); };
#pragma unroll
    for (uint32_t d = 0; d < kAhead; d++) load(stage_of(d), d);
    uint32_t slot = 0, free_slot = kAhead;
    for (uint32_t n = 0; n < rounds; n++) {
        const uint32_t stage = share + (n << shares_log2);
        // the oldest stage is there, and nobody reads the one before it any more, whose place the next loads take
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kAhead - 1) * kLoads) : "memory");
        if (groups > 1) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load(stage_of(n + kAhead), free_slot);
        const char* const from = mine + slot * kSlot;
        const char* const x_now = x_img + slot * grid.x_bytes;
        slot = slot == kAhead ? 0 : slot + 1;
        free_slot = free_slot == kAhead ? 0 : free_slot + 1;
        if (stage >= stages) continue;  // a share may have a stage less than others
        u32x4 w[kNT][kQ];
        uint32_t word[kNT][kQ];
#pragma unroll
        for (uint32_t q = 0; q < kQ; q++)
#pragma unroll
            for (uint32_t k = 0; k < kNT; k++) {
                const uint32_t unit = q * 4u + g;
                word[k][q] = *reinterpret_cast<const uint32_t*>(from + kCodeBytes + ((k * 16u + i) * kUnits + unit) * 4u);
                w[k][q] = *reinterpret_cast<const u32x4*>(from + ((k * 16u + i) * kUnits + (unit ^ code_turn(i))) * 16u);
            }
        // x of eight columns' products, asked of LDS kEarly products before they come: for few tokens everything at once
        constexpr uint32_t kProducts = kQ * kM, kEarly = kTT == 1 ? kProducts : 2;
        u32x4 xv[kProducts][kTT];
        const auto read_x = [&](uint32_t k) {
#pragma unroll
            for (uint32_t t = 0; t < kTT; t++)
                xv[k][t] = *reinterpret_cast<const u32x4*>(x_now + (column[t] * kPieces + ((((k / kM) * 4u + g) * kM + k % kM) ^ x_turn(column[t]))) * 16u);
        };
#pragma unroll
        for (uint32_t k = 0; k < kEarly; k++) read_x(k);
        __builtin_amdgcn_sched_barrier(0);
        float scale[kNT][kQ];
        bool mine_short = true;
#pragma unroll
        for (uint32_t q = 0; q < kQ; q++) {
            const uint32_t block = grid.block_of(min(stage * kUnits + q * 4u + g, units - 1u)) * grid.scale_col_bytes;
#pragma unroll
            for (uint32_t k = 0; k < kNT; k++) {
                scale[k][q] = dev::round_to<kF>(scale_of(masks, word[k][q], scale_of_row[k] + block));
                mine_short = mine_short && takes_short<kF, kCode>(scale[k][q]);
            }
        }
        const bool plain = (stage + 1u) * kUnits <= units && (kCode > 8 || __builtin_amdgcn_ballot_w64(!mine_short) == 0);
        const auto multiply = [&](auto ordinary) {
#pragma unroll
            for (uint32_t k = 0; k < kProducts; k++) {
                if (k + kEarly < kProducts) read_x(k + kEarly);
                const uint32_t q = k / kM, m = k % kM;
#pragma unroll
                for (uint32_t n_ = 0; n_ < kNT; n_++) {
                    u32x4 v = unit_slice<kF, kCode, decltype(ordinary)::value>(w[n_][q], m, scale[n_][q]);
                    if (!decltype(ordinary)::value && stage * kUnits + q * 4u + g >= units) v = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (uint32_t t = 0; t < kTT; t++) acc[n_][t][k & 1] = mfma<kF>(v, xv[k][t], acc[n_][t][k & 1]);
                }
            }
        };
        if (plain)
            multiply(std::true_type{});
        else
            multiply(std::false_type{});
    }

    // sums [wave][group of 16 rows][token][row], the shares of a group side by side; loads on their way are waited for, LDS is used again
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds);
    constexpr uint32_t kTokens = 16 * kTT;
#pragma unroll
    for (uint32_t n = 0; n < kNT; n++)
#pragma unroll
        for (uint32_t t = 0; t < kTT; t++)
            *reinterpret_cast<f32x4*>(part + ((wave * kNT + n) * kTokens + t * 16u + i) * 16u + 4u * g) = acc[n][t][0] + acc[n][t][1];
    __syncthreads();
    const uint32_t outputs = groups * wave_rows * tokens;
    for (uint32_t o = threadIdx.x; o < outputs; o += 512) {
        const uint32_t r = o % wave_rows, rest = o / wave_rows, in_group = rest % groups, t = rest / groups;
        const uint32_t col = (blockIdx.x * groups + in_group) * wave_rows + r;
        if (col >= a.out_cols) continue;
        const auto sum = [&](uint32_t row) {
            float v = 0.0f;
            for (uint32_t s = 0; s < shares; s++) v += part[((((in_group << shares_log2) + s) * kNT + row / 16u) * kTokens + t) * 16u + row % 16u];
            return v;
        };
        finish1(a, at.expert, at.first + t, col, sum(r), a.gated ? sum(16u + r) : 0.0f);
    }
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kUnits, int kX>
hipError_t launch_few(hipStream_t s, const MatmulArgs& a, const FewShape& c) {
    const FewGrid grid(a, c);
    hipLaunchKernelGGL((matmul_few_kernel<kF, kCode, kNT, kTT, kUnits, kX>), dim3(c.workgroups(a), static_cast<uint32_t>(most_tiles(a, c.tokens_log2))),
                       dim3(512), c.lds(), s, a, grid);
    return hipGetLastError();
}

template <dev::Float kF, int kCode, int kNT, int kTT, int kUnits>
hipError_t launch_loads(hipStream_t s, const MatmulArgs& a, const FewShape& c) {
    switch (c.x_loads()) {
        case 1: return launch_few<kF, kCode, kNT, kTT, kUnits, 1>(s, a, c);
        case 2: return launch_few<kF, kCode, kNT, kTT, kUnits, 2>(s, a, c);
        case 3: case 4: return launch_few<kF, kCode, kNT, kTT, kUnits, 4>(s, a, c);
        default: return launch_few<kF, kCode, kNT, kTT, kUnits, 8>(s, a, c);
    }
}

template <dev::Float kF, int kCode, int kNT>
hipError_t launch_units(hipStream_t s, const MatmulArgs& a, const FewShape& c) {
    if (c.tokens_log2 == 5) return launch_loads<kF, kCode, kNT, 2, 4>(s, a, c);
    if constexpr (kCode != 2) {
        if (c.units == 8) return launch_loads<kF, kCode, kNT, 1, 8>(s, a, c);
    }
    return launch_loads<kF, kCode, kNT, 1, 4>(s, a, c);
}

template <dev::Float kF, int kCode>
hipError_t launch_shape(hipStream_t s, const MatmulArgs& a, const FewShape& c) {
    return c.groups == 1 ? launch_units<kF, kCode, 1>(s, a, c) : launch_units<kF, kCode, 2>(s, a, c);
}

}  // namespace

#define CQ_FEW_NAME2(f, c) matmul_few_##f##_##c
#define CQ_FEW_NAME(f, c) CQ_FEW_NAME2(f, c)
hipError_t CQ_FEW_NAME(CQ_TU_FLOAT, CQ_TU_CODE)(hipStream_t s, const MatmulArgs& a, const FewShape& shape) {
    return launch_shape<dev::Float::CQ_TU_FLOAT, CQ_TU_CODE>(s, a, shape);
}

}  // namespace cq
