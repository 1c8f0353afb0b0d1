// What the attention kernels on the matrix cores share: codes to operands, tiles of rows, the partial results of a split.
#pragma once

#include <hip/hip_runtime.h>

#include "cq_attention_rows.hpp"

namespace cq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2E = 1.44269504088896340736f;
// Weights are exp2(t - top) * 2^5, with a `top` that the largest score so far exceeds by at most kLazy: f16 holds them up to 2^13 and down to 2^-29 of that of
// `top`.  A new largest score costs all results a product, so most of them are let pass.
constexpr float kLazy = 8.0f, kWeightLog2 = 5.0f, kWeightOne = 32.0f;

template <int kCode>
constexpr uint32_t kCodeBits = kCode == kCacheFloat ? 16u : (kCode == kCacheInt4 || kCode == kCacheE2M1 ? 4u : 8u);

// What may be infinite or not a number in a code; else only its scale can.
template <int kCode>
constexpr bool kCodeHasNaN = kCode == kCacheFloat || kCode == kCacheE4M3 || kCode == kCacheE5M2;

// The entry that stands at place i of eight decoded ones: 4-bit integers come in pairs (k, k + 4).
template <int kCode>
__device__ __forceinline__ constexpr uint32_t place_of(uint32_t i) {
    return kCode == kCacheInt4 ? i / 2u + i % 2u * 4u : i;
}

// Eight codes (8 bits: `low` then `high`; 4 bits: `low`) as numbers of f16, exactly.
//   i8 : the byte, its sign bit turned, under the exponent of 1024, less 1024 + 128
//   4-bit integers : nibbles 0 and 4 under the exponent of 1024, less 1024 + 8; nibbles 1 and 5 as 16 times themselves there, times 1/16, less 64 + 8
//   fp8, fp4 : one conversion for two
template <int kCode>
__device__ __forceinline__ u32x4 numbers(uint32_t low, uint32_t high) {
    const auto bits = [](f16x2 v) { return __builtin_bit_cast(uint32_t, v); };
    const auto half2 = [](uint32_t v) { return __builtin_bit_cast(f16x2, v); };
    if constexpr (kCode == kCacheInt8) {
        const f16x2 less = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        low ^= 0x80808080u, high ^= 0x80808080u;
        return u32x4{bits(half2(__builtin_amdgcn_perm(0x64646464u, low, 0x04010400u)) + less), bits(half2(__builtin_amdgcn_perm(0x64646464u, low, 0x04030402u)) + less),
                     bits(half2(__builtin_amdgcn_perm(0x64646464u, high, 0x04010400u)) + less), bits(half2(__builtin_amdgcn_perm(0x64646464u, high, 0x04030402u)) + less)};
    } else if constexpr (kCode == kCacheInt4) {
        const f16x2 less = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)}, less16 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)},
                    by = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
        low ^= 0x88888888u;
        const uint32_t next = low >> 8;
        return u32x4{bits(half2((low & 0x000f000fu) | 0x64006400u) + less), bits(__builtin_elementwise_fma(half2((low & 0x00f000f0u) | 0x64006400u), by, less16)),
                     bits(half2((next & 0x000f000fu) | 0x64006400u) + less), bits(__builtin_elementwise_fma(half2((next & 0x00f000f0u) | 0x64006400u), by, less16))};
    } else if constexpr (kCode == kCacheE2M1) {
        return u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(low, 1.0f, 0)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(low, 1.0f, 1)),
                     bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(low, 1.0f, 2)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(low, 1.0f, 3))};
    } else if constexpr (kCode == kCacheE4M3) {
        return u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, true)),
                     bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, true))};
    } else {
        return u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(low, 1.0f, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(low, 1.0f, true)),
                     bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(high, 1.0f, false)), bits(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8(high, 1.0f, true))};
    }
}

// Two f32 to a pair of 16 bits, each to the nearest.
template <bool kBF16>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
    if constexpr (kBF16) return BF16::pack2(a, b);
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

template <bool kBF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (kBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool kBF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (kBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

#define CQ_LDS_AT(T, p) ((__attribute__((address_space(3))) T*)(p))
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));

// The exponent field of the power of two that a row of queries is divided by, so that its largest entry lies between 1 and 2; f16 stays as it is, and
// so does a row of zeros or with an infinity.
__device__ __forceinline__ uint32_t power_of_row(float most, bool bf16) {
    const uint32_t field = f32_bits(most) >> 23;
    return bf16 && field > 0u && field < 255u ? min(field, 253u) : 127u;
}

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
    v = max(v, dpp<kDppXor1>(v));
    v = max(v, dpp<kDppXor2>(v));
    v = max(v, dpp<kDppHalfMirror>(v));
    v = max(v, dpp<kDppMirror>(v));
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(halves[0], halves[1]);
    const auto quarters = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(quarters[0], quarters[1]);
}

// The larger of a value's copies in the four groups of 16 lanes.
__device__ __forceinline__ float max_of_groups(float v) {
    const auto halves = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    v = fmaxf(bits_f32(halves[0]), bits_f32(halves[1]));
    const auto quarters = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return fmaxf(bits_f32(quarters[0]), bits_f32(quarters[1]));
}
__device__ __forceinline__ float sum_of_groups(float v) {
    const auto halves = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    v = bits_f32(halves[0]) + bits_f32(halves[1]);
    const auto quarters = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return bits_f32(quarters[0]) + bits_f32(quarters[1]);
}

// Whether eight entries of 16 bits have one that is infinite or not a number.
template <bool kBF16>
__device__ __forceinline__ bool has_odd(u32x4 v) {
    constexpr uint32_t kExponent = kBF16 ? 0x7f80u : 0x7c00u;
    bool found = false;
#pragma unroll
    for (uint32_t p = 0; p < 4; p++) {
        const uint32_t w = v[p];
        found = found || (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
    }
    return found;
}

// A stored scale is loaded as the word around it, from `offset & ~3` on, and made a number later: a load is not waited for where it is issued.
struct ScaleWords {
    uint32_t log2, up;
    bool f16;
    __device__ explicit ScaleWords(uint32_t dtype) : log2(dtype == CQ_F32 ? 2u : 1u), up(dtype == CQ_BF16 ? 16u : 0u), f16(dtype == CQ_F16) {}
    __device__ __forceinline__ float number(uint32_t word, uint32_t offset) const {
        const uint32_t bits = __builtin_amdgcn_alignbyte(0u, word, offset & 3u) << up;
        return f16 ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits))) : bits_f32(bits);
    }
};
// The exponent field of a scale, zero of one that is no number.
__device__ __forceinline__ uint32_t exponent_of(float v) {
    const uint32_t field = f32_bits(v) >> 23 & 255u;
    return field == 255u ? 0u : field;
}

// Weights times the scales of values (few rows, and kExact of many), or entries (many rows), are held in f16 over the largest scale so far, 2^power, to half of its
// smallest step, 2^-25.  Scales down to 2^-kSpread of the largest leave a weight 2^-18 of the largest one and an entry 2^-12 of its code's step.  A smaller one, unless it is zero,
// loses bits to keys that a row may not even see, or give no weight; rows whose results are small enough to show that are taken once more (rows_again).  A model's scales lie within
// 2^10 or so of one another.  A thread keeps the smallest of its scales, by twice their bits less one, so that zero is the largest of all and its sign does not count: two
// instructions a scale, and one question at the end (asked in every step, prompt_longest took 650 us instead of 624).
constexpr int32_t kSpread = 12;
__device__ __forceinline__ uint32_t smaller_of(uint32_t least, float scale) { return min(least, 2u * f32_bits(scale) - 1u); }
__device__ __forceinline__ bool lost_below(uint32_t least, int32_t power) { return least < max(static_cast<uint32_t>(max(127 + power - kSpread, 0)) << 24, 1u) - 1u; }
// A row shows it if its scores may be off by more than kScoreOff, or if 32 neighbouring entries of its result are all below kShows times what they may be off by: else that is less
// than 2^-11 of the largest of them, as it is of keys that have weight.
constexpr float kScoreOff = 0x1p-12f, kShows = 0x1p11f;
struct Losses {
    float key, value;  // in a score (times log2 e) by the sum of |query|; in a result
};
template <int kCode>
constexpr float kMostCode = kCode == kCacheInt8 ? 128.0f : kCode == kCacheInt4 ? 8.0f : kCode == kCacheE4M3 ? 448.0f : kCode == kCacheE5M2 ? 57344.0f : 6.0f;
// Of `keys` weights each is off by 2^-25 times its code; their sum is 2^5 at least.
template <int kCode>
__device__ __forceinline__ float lost_by_weights(uint32_t keys, int32_t power) { return ldexpf(kMostCode<kCode> * static_cast<float>(keys), power - 30); }

// What a row's products become before their weights: capped, with the bias of their distance, keys that the row does not see at -infinity.  `of` are a lane's
// products with the keys key0 + place(i); what is returned is left to be multiplied by, `times` where nothing of this is wanted.  `behind`: no key is past
// the position, so that the distance is linear and costs two instructions a score instead of five.  The conditions are uniform over the wave and each has a loop
// of its own: as choices within one loop they are all computed for all scores (509 tokens with a bias behind 7681 keys: 214 us instead of 154).
// The exponential's difference is off by 2^-22 of the cap, whatever the score: up to a cap of 64 (times log2 e) that is 2^-16 of a score's unit, less than weights of 16 bits
// show.  Of larger ones, |t / cap| < 1/4 takes tanh's series (what follows its last term is below 2^-21 of it); above, the difference is off by 2^-20 of itself.  kApart: small caps
// in a loop of their own, which is faster (a draft of 20 rows 36.8 us instead of 40.3, prompt_longest in f16 885 instead of 920), but where it moves what stands around it: calls without any
// cap took 650 us instead of 630 (prompt_longest), 121 instead of 116 (decode_batch).
constexpr float kExponentialCap = 64.0f * kLog2E;
// A cap as log2(e) times itself, and what `times` holds of it: no infinities of the highest and lowest numbers of f32 (a cap past 10^38 is 10^38).
__device__ __forceinline__ float cap_log2(float cap) { return fminf(cap, 1e38f) * kLog2E; }
__device__ __forceinline__ float times_of_cap(float times, float cap) { return fminf(times * fminf(2.0f * kLog2E / fminf(cap, 1e38f), 3e38f), 3e38f); }
template <bool kApart, uint32_t kCount, class Place>
__device__ __forceinline__ float shape_scores(float (&of)[kCount], float times, float cap, bool biased, float slope, int32_t position, int32_t key0, Place place, bool behind,
                                              bool partial, int32_t row_low, int32_t row_high) {
    if (cap > 0.0f) {  // cap tanh(t / cap) = cap - 2 cap / (1 + exp(2 t / cap)); `times` holds the 2 / cap
        const auto of_exponential = [&](float v) { return __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * times)), cap); };
        const bool small = cap <= kExponentialCap;
        const float edge = small ? 0.0f : 0.25f;
        if (kApart && small) {
#pragma unroll
            for (uint32_t i = 0; i < kCount; i++) of[i] = of_exponential(of[i]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kCount; i++) {
                const float x = of[i] * times * 0.34657359028f, x2 = x * x;  // t / cap: times ln(2) / 2
                const float series = __builtin_fmaf(x2, __builtin_fmaf(x2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f);
                of[i] = fabsf(x) < edge ? cap * __builtin_fmaf(x * x2, series, x) : of_exponential(of[i]);
            }
        }
        times = 1.0f;
    }
    if (biased) {
        if (behind) {
            const float first = slope * static_cast<float>(key0 - position);
#pragma unroll
            for (uint32_t i = 0; i < kCount; i++) of[i] = __builtin_fmaf(of[i], times, __builtin_fmaf(slope, static_cast<float>(place(i)), first));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kCount; i++) of[i] = __builtin_fmaf(of[i], times, -slope * static_cast<float>(abs(position - key0 - static_cast<int32_t>(place(i)))));
        }
        times = 1.0f;
    }
    if (partial) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; i++) {
            const int32_t key = key0 + static_cast<int32_t>(place(i));
            of[i] = key >= row_low && key <= row_high ? of[i] * times : -INFINITY;
        }
        times = 1.0f;
    }
    return times;
}

// The tile of rows (token, head of a group) that a workgroup has: tile t of a sequence's own begins at its row t * rows.  Sequence s owns the tiles from
// offsets[s] * group / rows + s on, which is room enough: floor(a + b) - floor(a) + 1 >= ceil(b).
struct RowTile {
    Sequence s;
    uint32_t row0, rows;  // first row within the sequence and how many there are
};
__device__ __forceinline__ uint64_t first_tile(const AttentionArgs& a, uint32_t seq, int32_t offset, uint32_t rows_log2) {
    return (static_cast<uint64_t>(min(static_cast<uint32_t>(max(offset, 0)), a.tokens)) * a.group >> rows_log2) + seq;
}
__device__ __forceinline__ bool rows_of(const AttentionArgs& a, const Sequence& s, uint64_t first, uint32_t tile, uint32_t rows_log2, RowTile* out) {
    const uint64_t rows = static_cast<uint64_t>(s.last - s.first) * a.group;
    if (tile < first) return false;
    const uint64_t row0 = (tile - first) << rows_log2;
    if (row0 >= rows) return false;
    out->s = s;
    out->row0 = static_cast<uint32_t>(row0);
    out->rows = static_cast<uint32_t>(min(rows - row0, static_cast<uint64_t>(1u << rows_log2)));
    return true;
}
__device__ __forceinline__ bool find_rows(const AttentionArgs& a, uint32_t tile, uint32_t rows_log2, RowTile* out) {
    const uint32_t s = __builtin_amdgcn_readfirstlane(last_at_or_below(a.seqs, tile, [&](uint32_t i) { return first_tile(a, i, a.offsets[i], rows_log2); }));
    return rows_of(a, sequence_of(a, s), first_tile(a, s, a.offsets[s], rows_log2), tile, rows_log2, out);
}

// Sums of the lanes up to each one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    const auto add = [&](uint32_t from) { v += from; };
    add(__builtin_amdgcn_update_dpp(0u, v, 0x111, 0xf, 0xf, true));  // one to the right within rows of 16 lanes, two, four, eight
    add(__builtin_amdgcn_update_dpp(0u, v, 0x112, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0u, v, 0x114, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0u, v, 0x118, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0u, v, 0x142, 0xa, 0xf, false));  // the last of rows 0 and 2 to rows 1 and 3, that of row 1 to rows 2 and 3
    add(__builtin_amdgcn_update_dpp(0u, v, 0x143, 0xc, 0xf, false));
    return v;
}

// The rows and the part of the keys that workgroup `index` of a head has, and how many steps of 2^keys_log2 keys a part is to have: as many as make a part for
// most of 256 compute units, not below split.fewest; split.enough where that is fewer, for then some units would
// have two parts and others one; more where all tiles of all sequences would come to more than about split.wanted parts.  Every workgroup works it out from the offsets and lengths.  Parts lie far
// apart in the grid, so that those which some tiles do not have come last.  Up to 64 sequences take one round of loads, and their tiles lie side by side.
// More sequences' tiles have gaps between them (find_rows), which would leave every other die idle where a sequence has exactly a tile's rows (64 sequences of 16 rows:
// 228 us with gaps, 127 without): every other one first, then the ones between.
template <bool kReversed>
__device__ __forceinline__ bool find_rows_and_steps(const AttentionArgs& a, const Split& split, uint32_t index, uint32_t rows_log2, uint32_t keys_log2, RowTile* out,
                                                    uint32_t* steps, uint32_t* part) {
    const uint32_t lane = threadIdx.x & 63u;
    const bool few = a.seqs <= 64;
    Sequence s{};
    uint32_t total = 0, own = 0;  // steps of the lane's sequences, at most 2^20 of each and of all; tiles of its last one
    *steps = ~0u;
    if (few || split.splits > 1) {
        for (uint32_t i = lane; i < a.seqs; i += 64) {
            s = sequence_of(a, i);
            own = static_cast<uint32_t>((static_cast<uint64_t>(s.last - s.first) * a.group + ((1u << rows_log2) - 1u)) >> rows_log2);
            const uint32_t length = static_cast<uint32_t>(s.length), seen = a.window && a.window < length ? min(length, a.window + (s.last - s.first)) : length;
            total = static_cast<uint32_t>(min(total + static_cast<uint64_t>(own) * ((seen >> keys_log2) + 1u), static_cast<uint64_t>(1u << 20)));
        }
    }
    const uint32_t upto = few ? wave_scan(own) : 0u, tiles = few ? static_cast<uint32_t>(__builtin_amdgcn_readlane(upto, 63)) : split.tiles;
    if (split.splits > 1) {
        const uint64_t all = static_cast<uint64_t>(__builtin_amdgcn_readlane(wave_scan(total), 63)) * a.cache.kv_heads;
        const auto of = [&](uint32_t parts) { return static_cast<uint32_t>((all + parts - 1u) / parts); };
        uint32_t each = of(250u);
        if (each > split.enough + split.enough / 4u) each = split.enough;
        *steps = max(max(each, split.fewest), of(split.wanted));
    }
    if (tiles == 0) return false;
    *part = index / tiles;
    uint32_t tile = index % tiles;
    if (*part >= split.splits) return false;
    if (kReversed) tile = tiles - 1u - tile;
    if (!few) {
        const uint32_t half = (tiles + 1u) / 2u;
        return find_rows(a, tile < half ? 2u * tile : 2u * (tile - half) + 1u, rows_log2, out);
    }
    const uint32_t at = static_cast<uint32_t>(__builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > tile)));
    const auto from_lane = [&](auto v) { return static_cast<decltype(v)>(__builtin_amdgcn_readlane(static_cast<int>(v), at)); };
    out->s.index = at;
    out->s.first = from_lane(s.first), out->s.last = from_lane(s.last), out->s.length = from_lane(s.length), out->s.position = from_lane(s.position), out->s.prefix = from_lane(s.prefix);
    out->row0 = (tile - (from_lane(upto) - from_lane(own))) << rows_log2;
    out->rows = min((out->s.last - out->s.first) * a.group - out->row0, 1u << rows_log2);
    return true;
}

// Parts of a tile's keys: [token][head][split] results over their own sums and {largest score, sum} (split.parts, split.stats).  A tile with one part writes y.
// What the parts it does not have would have left is written by its first part: sums of zero, or kWhole where there is nothing to join.
constexpr float kWhole = -1.0f;
__device__ __forceinline__ void note_parts(const AttentionArgs& a, const Split& split, const RowTile& at, uint32_t kv_head, uint32_t parts) {
    for (uint32_t r = threadIdx.x; r < at.rows; r += blockDim.x) {
        const uint32_t row = at.row0 + r, token = at.s.first + row / a.group, head = kv_head * a.group + row % a.group;
        float* const of = split.stats + 2ull * (static_cast<uint64_t>(token) * a.heads + head) * split.splits;
        if (parts == 1) of[0] = -INFINITY, of[1] = kWhole;
        for (uint32_t p = max(parts, 1u); p < split.splits; p++) of[2 * p] = -INFINITY, of[2 * p + 1] = 0.0f;
    }
}

// A kernel's first two arguments, read again: what is only needed behind its steps takes no registers from them.
struct Arguments {
    AttentionArgs a;
    Split split;
};
__device__ __forceinline__ const Arguments& arguments_again() {
    uint64_t again = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(again));
    return *reinterpret_cast<const Arguments*>(again);
}

// Rows of a tile once more, one by one, over the keys from first to last, in f32: all of them (`whole`) where an entry of a value that is infinite or not a number lies among
// keys that not every row of the tile sees, for a weight of zero does not keep such an entry out of a product of tiles; else those that show that scales are far apart (kSpread),
// whose results are written already.  All threads of the workgroup
// come here, with its LDS free for (kDim + 64) floats a wave.
template <uint32_t kDim>
__device__ __forceinline__ void rows_again(uint32_t seq, uint32_t row0, uint32_t rows, uint32_t part, uint32_t parts, uint32_t kv_head, int64_t first, int64_t last, bool whole,
                                           Losses losses, float* lds) {
    const Arguments& arguments = arguments_again();
    const AttentionArgs& a = arguments.a;
    const Split& split = arguments.split;
    const Sequence s = sequence_of(a, seq);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    float* const query = lds + wave * (kDim + 64u);
    for (uint32_t row = wave; row < rows; row += blockDim.x / 64u) {
        const uint32_t in_sequence = row0 + row, token = s.first + in_sequence / a.group, head = kv_head * a.group + in_sequence % a.group;
        const uint64_t of = (static_cast<uint64_t>(token) * a.heads + head) * split.splits + part;
        float of_query = 0.0f;
        for (uint32_t d = lane; d < a.cache.dim; d += 64) {
            const float q = load_dtype(a.dtype, a.q, token * a.q_token + head * a.q_head + d);
            query[d] = q;
            of_query += fabsf(q);
        }
        __builtin_amdgcn_wave_barrier();
        if (!whole) {
            bool shows = losses.key * wave_sum(of_query) > kScoreOff;
            for (uint32_t d = lane; d < a.cache.dim; d += 64) {
                float most = fabsf(parts > 1 ? split.parts[of * a.cache.dim + d] : load_dtype(a.dtype, a.y, token * a.y_token + head * a.y_head + d));
#pragma unroll
                for (int other = 16; other; other >>= 1) most = fmaxf(most, __shfl_xor(most, other, 64));  // of 32 entries, whose lanes are all here or none
                shows |= most < kShows * losses.value;
            }
            if (__builtin_amdgcn_ballot_w64(shows) == 0) continue;
        }
        const int32_t position = s.position + static_cast<int32_t>(in_sequence / a.group);
        const Seen seen = seen_from(a, s, position);
        float top, sum, v[kDim / 64];
        attend_row<kDim / 64>(a, s, kv_head, position, a.slopes ? a.slopes[head] : 0.0f, query, query + kDim, max(first, static_cast<int64_t>(seen.low)), 64,
                              min(last, static_cast<int64_t>(seen.high)), &top, &sum, v);
#pragma unroll
        for (uint32_t i = 0; i < kDim / 64; i++) {
            const uint32_t d = i * 64u + lane;
            if (d >= a.cache.dim) continue;
            const float y = sum != 0.0f ? v[i] / sum : 0.0f;
            if (parts > 1)
                split.parts[of * a.cache.dim + d] = y;
            else
                store_dtype(a.dtype, a.y, token * a.y_token + head * a.y_head + d, y);
        }
        if (parts > 1 && lane == 0) split.stats[2 * of] = top * kLog2E, split.stats[2 * of + 1] = sum * kWeightOne;
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace
}  // namespace cq
