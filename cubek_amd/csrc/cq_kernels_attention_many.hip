// Attention of many rows (token, head of a group): prompts and their chunks.  An object per kind of code (CQ_TU_CODE).
//
// A workgroup takes 256 rows (128 of heads longer than 128) that share a head of the cache, a wave 32 of them.  Keys come 64 at a time: the
// workgroup loads their codes one step ahead, makes numbers of f16 of them (a cache of floats: as they are) and lays keys and values into LDS, two
// steps in turn, one barrier a step.  Each wave then computes S^T = K Q^T and O^T = V^T P^T by 32 x 32 x 16 matrix instructions with queries,
// weights and results in registers: the scores that lane (n, h) gets are those of row n, and stand in the order of keys in which the second product takes
// its weights; values are read transposed.
// Entries are scaled by powers of two (of the largest scale so far, one for keys, one for values; queries by one per row), so that f16 holds them whatever
// the range of bf16 (kSpread says how far apart scales may be).  What is rounded to 16 bits, and why:
//   keys : scale * code in f32, once to the 11 bits of f16, where dequantize for bf16 would round to 8.  With its scale rounded to f16 first, as a value's is, all of a key's score is
//     off by that: 8191 tokens of fp8 0.0021 of the result's norm instead of 0.0018 (0.0017 of it is the result's own rounding to bf16), for 2 % less time (641 us, and 653)
//   values : the scale to 11 bits and the product to 11 bits, one instruction for two entries; once would take another 1.5 % and change 0.00175 to 0.00174
//   weights : 11 bits, and over a bf16 cache of floats, which enters the matrix instructions as it is, the 8 of bf16: off by 0.0023 of the norm (7 prompts of 33 to 2047 tokens).  In two
//     numbers of bf16, as attention_few_kernel has them, it is 0.0017, for half as many matrix instructions again: 562 us and 731 of 8191 tokens, 82 and 104 of these.  Their sum is f32.
// For results of f16 rounded entries show (0.0012, where the result's own rounding is 0.0002): kExact keeps codes, exact in f16, and puts their scales in f32 behind the first product
// and on the weights (0.0003).
//
// A step of a head of 128 is 32 matrix instructions of a wave (1024 cycles) beside about 250 vector instructions, 150 of them the softmax's; with two waves on a
// SIMD they overlap in part, and no unit is full: a prompt of 8191 tokens, 32 heads over 8 of fp8, 630-645 us, 850-870 TFLOP/s at 1.8 GHz, vector units busy 47 %, matrix units
// 36 %, LDS 46 %, waves waiting for a barrier or for LDS in 39 % of their cycles.
#include <hip/hip_runtime.h>

#include "cq_attention_tiles.hpp"
#include "cq_magic_div.hpp"

namespace cq {
namespace {

template <int kCode, int kDim>
struct Many {
    static constexpr uint32_t kBits = kCodeBits<kCode>, kKeys = 64;
    // Waves that share rows: of heads past 128 two compute all scores of the same 32 rows and half of the result each, whose registers leave room for two waves a SIMD
    // (4096 tokens of heads of 256: 513 us, and 616 with a wave's rows its own and one a SIMD).
    static constexpr uint32_t kWaves = 8, kThreads = 64 * kWaves, kShare = kDim > 128 ? 2 : 1, kRowWaves = kWaves / kShare;
    static constexpr uint32_t kRows = kRowWaves * 32, kRowsLog2 = kRows == 256 ? 8 : 7;
    static constexpr uint32_t kRow = kDim * kBits / 8;                                                  // bytes of a key as it is stored
    static constexpr uint32_t kChunk = kRow * kKeys / kThreads < 16 ? kRow * kKeys / kThreads : 16, kLanes = kRow / kChunk;  // of a thread; threads of a row
    static constexpr uint32_t kEntries = kChunk * 8 / kBits, kChunks = kKeys * kLanes / kThreads;             // entries of a chunk; chunks of a thread
    static constexpr uint32_t kPitch = kDim * 2 + 32, kSide = kKeys * kPitch, kBuffer = 2 * kSide;       // bytes in LDS: of a row, of keys or values, of both
};

// Forms that would keep reading spilled registers from scratch memory work out their lanes' addresses in LDS again in every step (7 prompts of 33 to 2047 tokens over i8 of heads of
// 256, f16: 735 us, and 769).  Heads of 64 put up to four registers away in front of their steps and take them back behind, which costs less than this would (99 us, and 102).
template <int kDim, bool kExact>
constexpr bool kAgain = kExact && kDim == 256;

// Eight numbers in the order of their entries.
template <int kCode>
__device__ __forceinline__ u32x4 in_order(u32x4 v) {
    if constexpr (kCode != kCacheInt4) return v;
    return u32x4{__builtin_amdgcn_perm(v[1], v[0], 0x05040100u), __builtin_amdgcn_perm(v[3], v[2], 0x05040100u), __builtin_amdgcn_perm(v[1], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[2], 0x07060302u)};
}

// kExact: entries enter as their codes, scales in f32 behind the first product and on the weights; else as numbers of f16.
template <int kCode, int kDim, bool kBF16, bool kExact>
__global__ __launch_bounds__((Many<kCode, kDim>::kThreads), (kDim == 64 && !kExact ? 4 : 1)) void attention_many_kernel(AttentionArgs a, Split split) {
    using S = Many<kCode, kDim>;
    constexpr bool kFloat = kCode == kCacheFloat;
    constexpr uint32_t kSlices = kDim / 16, kOut = kDim / 32 / S::kShare;  // tiles of 32 entries of the wave's part
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t* const powers = reinterpret_cast<uint32_t*>(lds + 2 * S::kBuffer);  // [step % 2][keys, values]: exponents, the largest of every other step so far
    uint32_t* const found = powers + 4;                                          // whether values that are no numbers, or scales far apart, need rows one by one
    uint32_t* const lost = powers + 5;                                           // whether scales are far apart, of keys, of values
    float* const scales_at = reinterpret_cast<float*>(powers + 8);               // kExact: [step % 2][keys, values][block][64]
    constexpr uint32_t kScales = kDim / 32 * S::kKeys;                           // of a side of a step
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31u, h = lane >> 5;
    // Neighbours in the grid are heads of the cache: with eight of them each die keeps one in its L2.  The tiles with most keys come first, the parts that some
    // tiles do not have last (next to those that they have, they leave parts of the dies idle: 1000 tokens behind 7190 keys, whose
    // tiles have two of four parts, 190 us, and 322).
    const uint32_t kv_head = blockIdx.x % a.cache.kv_heads, dim = a.cache.dim;

    RowTile at;
    uint32_t steps_wanted, part;
    if (!find_rows_and_steps<true>(a, split, blockIdx.x / a.cache.kv_heads, S::kRowsLog2, 6, &at, &steps_wanted, &part)) return;
    const auto position_of = [&](uint32_t row) { return at.s.position + static_cast<int32_t>((at.row0 + row) / a.group); };
    const Seen top_row = seen_from(a, at.s, position_of(0)), bottom_row = seen_from(a, at.s, position_of(at.rows - 1u));
    const int32_t low = top_row.low, high = bottom_row.high, tile_low = bottom_row.low, tile_high = top_row.high;  // seen by some, and by all
    const uint32_t step0 = static_cast<uint32_t>(low) / S::kKeys, steps_all = high < low ? 0u : static_cast<uint32_t>(high) / S::kKeys + 1u - step0;
    const uint32_t parts = min(max(steps_all / steps_wanted + (steps_all % steps_wanted != 0), 1u), split.splits), each = (steps_all + parts - 1u) / parts;
    if (part >= parts) return;
    if (split.splits > 1 && part == 0) note_parts(a, split, at, kv_head, parts);
    const uint32_t from = min(part * each, steps_all), to = min(from + each, steps_all);
    const uint32_t last_tile = static_cast<uint32_t>(max(high, 0)) / 16u;

    // the wave's rows, and the keys that some of them see and that all of them do
    const uint32_t wave_row = (S::kShare == 1 ? wave : wave % S::kRowWaves) * 32u, first_out = S::kShare == 1 ? 0u : wave / S::kRowWaves * kOut, wave_last = min(wave_row + 32u, at.rows) - 1u;
    const bool rows_here = wave_row < at.rows;
    const int32_t first_position = position_of(min(wave_row, at.rows - 1u));
    const Seen first = seen_from(a, at.s, first_position), last = seen_from(a, at.s, position_of(rows_here ? wave_last : at.rows - 1u));
    const int32_t wave_low = first.low, wave_high = rows_here ? last.high : -1, all_low = last.low, all_high = first.high;

    // the lane's row (past the tile's last one: that one, but nothing seen)
    const uint32_t own = wave_row + n;
    const auto row_of = [&] { return min(own, at.rows - 1u) + at.row0; };
    const auto token_of = [&] { return static_cast<uint64_t>(at.s.first + row_of() / a.group); };
    const auto head_of = [&] { return kv_head * a.group + row_of() % a.group; };
    const int32_t position = position_of(min(own, at.rows - 1u));
    const Seen seen = seen_from(a, at.s, position);
    const int32_t row_low = seen.low, row_high = own < at.rows ? seen.high : -1;
    const float slope = a.slopes ? a.slopes[head_of()] * kLog2E : 0.0f;
    u32x4 q[kSlices];
    const char* const from_q = a.q + (token_of() * a.q_token + head_of() * a.q_head) * 2u;
#pragma unroll
    for (uint32_t t = 0; t < kSlices; t++) {
        const uint32_t d = 16u * t + 8u * h;
        q[t] = d < dim ? *reinterpret_cast<const u32x4*>(from_q + d * 2u) : u32x4{0, 0, 0, 0};
    }
    if (a.scale < 0.0f) {  // into the queries: the largest score is that of the largest product
#pragma unroll
        for (uint32_t t = 0; t < kSlices; t++) q[t] ^= 0x80008000u;
    }
    float times = fabsf(a.scale);
    if constexpr (!kFloat) {
        float most = 0.0f, v[8];
        const bool bf16 = a.dtype == CQ_BF16;
        const auto unpack = [&](u32x4 w) { bf16 ? BF16::unpack(w, v) : F16::unpack(w, v); };
#pragma unroll
        for (uint32_t t = 0; t < kSlices; t++) {
            unpack(q[t]);
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) most = fmaxf(most, fabsf(v[e]));
        }
        const auto halves = __builtin_amdgcn_permlane32_swap(f32_bits(most), f32_bits(most), false, false);
        most = fmaxf(bits_f32(halves[0]), bits_f32(halves[1]));
        const uint32_t down = power_of_row(most, bf16);
        if constexpr (kSlices > 8) {  // unpacked again, not kept: they would take twice the queries' registers
#pragma unroll
            for (uint32_t t = 0; t < kSlices; t++) asm volatile("" : "+v"(q[t]));
        }
#pragma unroll
        for (uint32_t t = 0; t < kSlices; t++) {
            unpack(q[t]);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) q[t][e] = pair_of<false>(v[2 * e] * bits_f32((254u - down) << 23), v[2 * e + 1] * bits_f32((254u - down) << 23));
        }
        times *= bits_f32(down << 23);
    }
    times = a.cap > 0.0f ? times_of_cap(times, a.cap) : times * kLog2E;
    const float cap = cap_log2(a.cap);

    // Pages of the next 16 steps, a lane a tile of 16 keys.
    const uint32_t tiles_of_page = a.cache.page_size / 16u;
    const auto tile_of = [&](uint32_t step, uint32_t k) { return min((step0 + step) * 4u + k, last_tile); };
    uint32_t pages = 0;
    const auto look_up = [&](uint32_t step) { pages = page_of(a, at.s, magic_div(tile_of(step + lane / 4u, lane % 4u), split.page_magic, split.page_shift)); };
    const auto place_of_tile = [&](uint32_t t) { return (t - magic_div(t, split.page_magic, split.page_shift) * tiles_of_page) * 16u; };

    // What a thread brings of a step: chunks of keys and of values, and their scales.
    struct Raw {
        uint32_t k[S::kChunks][S::kChunk / 4], v[S::kChunks][S::kChunk / 4];
    };
    struct Scales {
        uint32_t k[S::kChunks], v[S::kChunks], odd;  // words; bits 2 c ... of keys and 16 + 2 c ... of values: half a word that their tile begins with
    };
    constexpr uint32_t kPass = S::kThreads / S::kLanes;  // keys of the workgroup's chunks at once
    static_assert(kPass % 16 == 0);
    const ScaleWords words(a.cache.param_dtype);
    const uint32_t row_bytes = dim * S::kBits / 8u, byte = threadIdx.x % S::kLanes * S::kChunk, entry = byte * 8u / S::kBits;
    const uint32_t block = min(entry, dim - 1u) >> split.block_log2, block_mask = (1u << split.block_log2) - 1u;
    const auto key_of = [&](uint32_t c) { return c * kPass + threadIdx.x / S::kLanes; };
    // a thread's offsets from the tile of 16 keys that holds its key; what is left is the same for the wave
    const uint32_t in_tile = threadIdx.x / S::kLanes % 16u, at_byte = min(byte, row_bytes - S::kChunk);
    const uint32_t key_at = in_tile * static_cast<uint32_t>(a.cache.keys.slot) + at_byte, value_at = in_tile * static_cast<uint32_t>(a.cache.values.slot) + at_byte;
    const auto scale_at = [&](const CacheSide& side) { return (in_tile * static_cast<uint32_t>(side.scale_slot) + block * static_cast<uint32_t>(side.scale_block)) << words.log2; };
    const uint32_t key_scale_at = scale_at(a.cache.keys), value_scale_at = scale_at(a.cache.values);
    // the page of a chunk's tile and the row in it
    const auto place = [&](uint32_t step, uint32_t c, uint32_t* page, uint32_t* slot) {
        const uint32_t k = (c * kPass + wave * (64u / S::kLanes)) / 16u;
        *page = __builtin_amdgcn_readlane(pages, (step - from) % 16u * 4u + k);
        *slot = place_of_tile(tile_of(step, k));
    };
    const auto rows_at = [&](const CacheSide& side, uint32_t page, uint32_t slot) {
        return side.base + kv_head * side.head + static_cast<uint64_t>(page) * static_cast<uint32_t>(side.page) + slot * static_cast<uint32_t>(side.slot);
    };
    const auto load = [&](uint32_t step, Raw& raw) {
#pragma unroll
        for (uint32_t c = 0; c < S::kChunks; c++) {
            uint32_t page, slot;
            place(step, c, &page, &slot);
            const char* const k = rows_at(a.cache.keys, page, slot) + key_at;
            const char* const v = rows_at(a.cache.values, page, slot) + value_at;
            if constexpr (S::kChunk == 4) {
                raw.k[c][0] = *reinterpret_cast<const uint32_t*>(k), raw.v[c][0] = *reinterpret_cast<const uint32_t*>(v);
            } else if constexpr (S::kChunk == 16) {
                const u32x4 kw = *reinterpret_cast<const u32x4*>(k), vw = *reinterpret_cast<const u32x4*>(v);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) raw.k[c][e] = kw[e], raw.v[c][e] = vw[e];
            } else {
                const u32x2 kw = *reinterpret_cast<const u32x2*>(k), vw = *reinterpret_cast<const u32x2*>(v);
                raw.k[c][0] = kw[0], raw.k[c][1] = kw[1], raw.v[c][0] = vw[0], raw.v[c][1] = vw[1];
            }
        }
    };
    const auto load_scales = [&](uint32_t step, Scales& s) {
        s.odd = 0;
#pragma unroll
        for (uint32_t c = 0; c < S::kChunks; c++) {
            uint32_t page, slot;
            place(step, c, &page, &slot);
            const auto from_word = [&](const CacheSide& side, uint32_t at, uint32_t shift) {
                const char* const of = side.scales + ((kv_head * side.scale_head + static_cast<uint64_t>(page) * static_cast<uint32_t>(side.scale_page) + slot * static_cast<uint32_t>(side.scale_slot)) << words.log2);
                const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(of)) & 2u;
                s.odd |= odd << shift;
                return *reinterpret_cast<const uint32_t*>(of - odd + ((at + odd) & ~3u));
            };
            s.k[c] = from_word(a.cache.keys, key_scale_at, 2 * c), s.v[c] = from_word(a.cache.values, value_scale_at, 16 + 2 * c);
        }
    };
    int32_t key_power = -126, value_power = -126;  // of the largest scales of what was laid so far: entries are taken times 2^-power / 2
    uint32_t least_key = ~0u, least_value = ~0u;   // of the smallest (smaller_of)
    // A step's scales as numbers, and for the workgroup the exponents of its largest ones that any row sees, where they pass what was there before.
    float key_scale[S::kChunks], value_scale[S::kChunks];
    const auto publish = [&](uint32_t step, const Scales& s) {
        const int32_t step_key = static_cast<int32_t>((step0 + step) * S::kKeys);
        float of_keys = 0.0f, of_values = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < S::kChunks; c++) {
            key_scale[c] = words.number(s.k[c], key_scale_at + (s.odd >> (2 * c) & 2u));
            value_scale[c] = words.number(s.v[c], value_scale_at + (s.odd >> (16 + 2 * c) & 2u));
        }
        if (step_key < low || step_key + static_cast<int32_t>(S::kKeys) - 1 > high) {
#pragma unroll
            for (uint32_t c = 0; c < S::kChunks; c++) {
                const int32_t key = step_key + static_cast<int32_t>(key_of(c));
                if (key < low || key > high) key_scale[c] = value_scale[c] = 0.0f;
            }
        }
#pragma unroll
        for (uint32_t c = 0; c < S::kChunks; c++) of_keys = fmaxf(of_keys, fabsf(key_scale[c])), of_values = fmaxf(of_values, fabsf(value_scale[c]));
        const auto limit = [](int32_t power) { return bits_f32(static_cast<uint32_t>(128 + power) << 23); };  // 2^(power + 1)
        if (__builtin_amdgcn_ballot_w64(!(of_keys < limit(key_power)) || !(of_values < limit(value_power)))) {
            uint32_t keys = 0, values = 0;
#pragma unroll
            for (uint32_t c = 0; c < S::kChunks; c++) keys = max(keys, exponent_of(key_scale[c])), values = max(values, exponent_of(value_scale[c]));
            keys = wave_max_bits(keys), values = wave_max_bits(values);
            if (lane == 0) atomicMax(powers + (step & 1u) * 2u, keys), atomicMax(powers + (step & 1u) * 2u + 1u, values);
        }
    };

    f32x16 out[kOut] = {};
    float top = -INFINITY, sum = 0.0f;
    int32_t score_power = -126, out_power = -126;  // of the keys that scores are made of, and of the values in `out`

    // A step's codes as numbers into LDS.  In a step that some row sees only a part of, values that no row sees become zeros, and others that are no
    // numbers are reported.
    const auto lay = [&](uint32_t step, Raw& raw) {
        char* const to_keys = lds + (step & 1u) * S::kBuffer;
        const int32_t step_key = static_cast<int32_t>((step0 + step) * S::kKeys);
        const bool partial = step_key < tile_low || step_key + static_cast<int32_t>(S::kKeys) - 1 > tile_high;
        float down_keys = 0.0f, down_values = 0.0f;
        if constexpr (!kFloat) {
            const uint32_t* const of = powers + (step & 1u) * 2u;
            const int32_t now_keys = min(static_cast<int32_t>(__builtin_amdgcn_readfirstlane(of[0])) - 127, 126);
            const int32_t now_values = min(static_cast<int32_t>(__builtin_amdgcn_readfirstlane(of[1])) - 127, 126);
            key_power = max(key_power, now_keys);
            value_power = max(value_power, now_values);
            down_keys = 0.5f * bits_f32(static_cast<uint32_t>(127 - key_power) << 23), down_values = 0.5f * bits_f32(static_cast<uint32_t>(127 - value_power) << 23);
        }
#pragma unroll
        for (uint32_t c = 0; c < S::kChunks; c++) {
            char* const row = to_keys + key_of(c) * S::kPitch + entry * 2u;
            if constexpr (!kFloat) least_value = smaller_of(least_value, value_scale[c]);
            if constexpr (!kFloat && !kExact) least_key = smaller_of(least_key, key_scale[c]);
            if constexpr (kExact) {
                if ((entry & block_mask) == 0) {
                    float* const to = scales_at + (step & 1u) * 2u * kScales + (entry >> split.block_log2) * S::kKeys + key_of(c);
                    to[0] = key_scale[c], to[kScales] = value_scale[c] * 2.0f * down_values;
                }
                if (partial && !(fabsf(value_scale[c]) < INFINITY)) *found = 1u;
            }
            if (row_bytes < S::kRow) {  // a shorter head: nothing past its end
#pragma unroll
                for (uint32_t e = 0; e < S::kChunk / 4; e++) raw.k[c][e] = byte < row_bytes ? raw.k[c][e] : 0u, raw.v[c][e] = byte < row_bytes ? raw.v[c][e] : 0u;
            }
            if (partial) {
                const int32_t key = step_key + static_cast<int32_t>(key_of(c));
                if (key < low || key > high) {
#pragma unroll
                    for (uint32_t e = 0; e < S::kChunk / 4; e++) raw.v[c][e] = 0;
                }
            }
            const auto look = [&](u32x4 v) {
                if (partial && has_odd<kBF16>(v)) *found = 1u;
            };
            if constexpr (kFloat) {
                const u32x4 v = {raw.v[c][0], raw.v[c][1], raw.v[c][2], raw.v[c][3]};
                look(v);
                *reinterpret_cast<u32x4*>(row) = u32x4{raw.k[c][0], raw.k[c][1], raw.k[c][2], raw.k[c][3]};
                *reinterpret_cast<u32x4*>(row + S::kSide) = v;
            } else {
                constexpr uint32_t kEach = S::kBits == 8 ? 2 : 1;  // words of eight entries
                const auto put = [&](char* to, const uint32_t* w, float scale, bool of_values) {
                    const uint32_t both = pair_of<false>(scale, scale);
                    const f16x2 by = __builtin_bit_cast(f16x2, both);
#pragma unroll
                    for (uint32_t e = 0; e < S::kChunk / 4; e += kEach) {
                        u32x4 v = in_order<kCode>(numbers<kCode>(w[e], kEach == 2 ? w[e + kEach - 1] : 0u));
                        if constexpr (!kExact) {
#pragma unroll
                            for (uint32_t p = 0; p < 4; p++) {
                                const uint32_t word = v[p];
                                f16x2 two = __builtin_bit_cast(f16x2, word);
                                if (of_values) {
                                    two = two * by;
                                } else {
#pragma unroll
                                    for (uint32_t i = 0; i < 2; i++) two[i] = static_cast<_Float16>(__builtin_fmaf(static_cast<float>(two[i]), scale, 0.0f));
                                }
                                v[p] = __builtin_bit_cast(uint32_t, two);
                            }
                        }
                        if (of_values) look(v);
                        *reinterpret_cast<u32x4*>(to + e / kEach * 16u) = v;
                    }
                };
                put(row, raw.k[c], key_scale[c] * down_keys, false);
                put(row + S::kSide, raw.v[c], value_scale[c] * down_values, true);
            }
        }
    };

    // Scores, weights and results of kSpan keys: of all 64 of a step where registers allow it, which halves the waits for LDS and for the largest score
    // (heads of 128: 633 us instead of 665 of a prompt of 8191 tokens); two waves of a head of 64 share a SIMD with two others, which hides them.
    constexpr uint32_t kHalves = kDim == 128 && !kExact ? 2 : 1, kSpan = 32 * kHalves;
    const auto compute = [&](uint32_t step, uint32_t half) {
        const int32_t key0 = static_cast<int32_t>((step0 + step) * S::kKeys + 32u * half);
        if (key0 > wave_high || key0 + static_cast<int32_t>(kSpan) - 1 < wave_low) return;
        const bool partial = key0 < all_low || key0 + static_cast<int32_t>(kSpan) - 1 > all_high;
        uint32_t own_lane = lane;
        if constexpr (kAgain<kDim, kExact>) asm volatile("" : "+v"(own_lane));
        const uint32_t n = own_lane & 31u, h = own_lane >> 5;
        const char* const keys = lds + (step & 1u) * S::kBuffer + 32u * half * S::kPitch;
        const char* const values = keys + S::kSide;
        // the scales of lane (n, h)'s keys, of one block of entries: four behind one another of every eight
        const auto scales_of = [&](uint32_t side, uint32_t block, uint32_t four) {
            return *reinterpret_cast<const f32x4*>(scales_at + ((step & 1u) * 2u + side) * kScales + block * S::kKeys + 32u * half + four * 8u + 4u * h);
        };
        float t[kSpan / 2];
        f32x16 s[kHalves] = {};
        if constexpr (kExact) {
#pragma unroll
            for (uint32_t v = 0; v < 16; v++) t[v] = 0.0f;
        }
        const auto operand_of = [&](uint32_t slice, uint32_t k) { return *reinterpret_cast<const u32x4*>(keys + (k * 32u + n) * S::kPitch + slice * 32u + h * 16u); };
        u32x4 ahead[kHalves];  // of the next slice, asked for in front of this one's products: so written, it stays so where registers are short
#pragma unroll
        for (uint32_t k = 0; k < kHalves; k++) ahead[k] = operand_of(0, k);
#pragma unroll
        for (uint32_t slice = 0; slice < kSlices; slice++) {
            u32x4 operand[kHalves];
#pragma unroll
            for (uint32_t k = 0; k < kHalves; k++) {
                operand[k] = ahead[k];
                if (slice + 1 < kSlices) ahead[k] = operand_of(slice + 1, k);
            }
#pragma unroll
            for (uint32_t k = 0; k < kHalves; k++) s[k] = mfma32<kBF16>(operand[k], q[slice], s[k]);
            if constexpr (kSlices > 8)
                if (slice % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more operands at once than there are registers for
            if constexpr (kExact) {
                if (slice + 1 == kSlices || ((slice + 1) * 16u & block_mask) == 0) {  // the block's last
#pragma unroll
                    for (uint32_t four = 0; four < 4; four++) {
                        const f32x4 scale = scales_of(0, slice * 16u >> split.block_log2, four);
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) t[four * 4 + e] = __builtin_fmaf(s[0][four * 4 + e], scale[e], t[four * 4 + e]);
                    }
                    s[0] = f32x16{};
                }
            }
        }
        const float by = kFloat || kExact ? times : times * 2.0f * bits_f32(static_cast<uint32_t>(127 + score_power) << 23);
        if constexpr (!kExact) {
#pragma unroll
            for (uint32_t v = 0; v < kSpan / 2; v++) t[v] = s[v / 16u][v % 16u];
        }
        const float times_now = shape_scores<kExact>(t, by, cap, a.slopes, slope, position, key0 + static_cast<int32_t>(4u * h), [](uint32_t v) { return v / 4u * 8u + v % 4u; },
                                             key0 + static_cast<int32_t>(kSpan) - 1 <= first_position, partial, row_low, row_high);
        // largest scores are `top` + kLazy at most: results are taken down to a larger one only where it is needed
        float most = -INFINITY;
#pragma unroll
        for (uint32_t v = 0; v < kSpan / 2; v++) most = fmaxf(most, t[v]);
        most *= times_now;
        const auto halves = __builtin_amdgcn_permlane32_swap(f32_bits(most), f32_bits(most), false, false);
        most = fmaxf(bits_f32(halves[0]), bits_f32(halves[1]));
        if (__builtin_amdgcn_ballot_w64(most > top + kLazy)) {
            const float before = top;
            top = fmaxf(top, most);
            const float shrink = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(before - top);
            sum *= shrink;
#pragma unroll
            for (uint32_t e = 0; e < kOut; e++) out[e] *= shrink;
        }
        const float less = kWeightLog2 - (top == -INFINITY ? 0.0f : top);
        // the weights of a quarter, sixteen keys
        const auto weigh = [&](uint32_t quarter) {
            u32x4 w = {};
#pragma unroll
            for (uint32_t v = quarter * 8u; v < quarter * 8u + 8u; v += 2) {
                t[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[v], times_now, less)), t[v + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[v + 1], times_now, less));
                sum += t[v], sum += t[v + 1];
                if constexpr (!kExact) w[v % 8 / 2] = pair_of<kBF16>(t[v], t[v + 1]);
            }
            return w;
        };
        // lane (n, h): entry n of 32, keys 4 h ... 4 h + 3 and 8 more
        const auto values_of = [&](uint32_t e, uint32_t quarter) {
            u32x4 v;
#pragma unroll
            for (uint32_t eight = 0; eight < 2; eight++) {
                const auto four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    CQ_LDS_AT(i16x4, values + first_out * 64u + (quarter * 16u + eight * 8u + 4u * h + own_lane % 16u / 4u) * S::kPitch + e * 64u + n / 16u * 32u + own_lane % 4u * 8u));
                const u32x2 two = __builtin_bit_cast(u32x2, four);
                v[2 * eight] = two[0], v[2 * eight + 1] = two[1];
            }
            return v;
        };
        if constexpr (kExact) {
            u32x4 w[2] = {weigh(0), weigh(1)};
#pragma unroll
            for (uint32_t e = 0; e < kOut; e++) {
                if (e == 0 || ((first_out + e) * 32u & block_mask) == 0) {  // a block's first, or the wave's: its weights
#pragma unroll
                    for (uint32_t four = 0; four < 4; four++) {
                        const f32x4 scale = scales_of(1, (first_out + e) * 32u >> split.block_log2, four);
#pragma unroll
                        for (uint32_t i = 0; i < 4; i += 2) w[four / 2][four % 2 * 2 + i / 2] = pair_of<false>(t[four * 4 + i] * scale[i], t[four * 4 + i + 1] * scale[i + 1]);
                    }
                }
#pragma unroll
                for (uint32_t quarter = 0; quarter < 2; quarter++) out[e] = mfma32<kBF16>(values_of(e, quarter), w[quarter], out[e]);
            }
        } else {
#pragma unroll
            for (uint32_t quarter = 0; quarter < 2 * kHalves; quarter++) {
                u32x4 v[kOut];  // asked for in front of the weights
#pragma unroll
                for (uint32_t e = 0; e < kOut; e++) v[e] = values_of(e, quarter);
                const u32x4 w = weigh(quarter);
#pragma unroll
                for (uint32_t e = 0; e < kOut; e++) out[e] = mfma32<kBF16>(v[e], w, out[e]);
            }
        }
    };

    if (threadIdx.x < 7) powers[threadIdx.x] = 0u;  // and *found, lost
    __syncthreads();
    if (from < to) {
        Raw raw;
        Scales scales{};
        look_up(from);
        load(from, raw);
        if constexpr (!kFloat) {
            load_scales(from, scales);
            publish(from, scales);
            load_scales(from + 1u, scales);
            __syncthreads();
        }
        lay(from, raw);
        if constexpr (!kFloat) publish(from + 1u, scales);
        if (from + 1u < to) load(from + 1u, raw);
        if constexpr (!kFloat) load_scales(from + 2u, scales);
        // The next step goes to LDS before this one is computed in one half of the waves and behind it in the other, so that the two waves of a SIMD do not
        // want its matrix unit at the same time.
        const bool early = wave >= 4;
        for (uint32_t step = from; step < to; step++) {
            __syncthreads();
            if constexpr (!kFloat) {
                score_power = key_power;
                if (value_power > out_power) {
                    const float shrink = ldexpf(1.0f, out_power - value_power);
                    out_power = value_power;
#pragma unroll
                    for (uint32_t e = 0; e < kOut; e++) out[e] *= shrink;
                }
            }
            // pages are looked up for sixteen steps from `from` on; codes are asked for a step before they are laid, scales two
            const uint32_t done = step - from;
            const auto next = [&]() __attribute__((always_inline)) {
                if (step + 1u < to) {
                    lay(step + 1u, raw);
                    if constexpr (!kFloat) publish(step + 2u, scales);
                }
                if (kFloat && (done + 2u) % 16u == 0) look_up(step + 2u);
                if (step + 2u < to) load(step + 2u, raw);
                if constexpr (!kFloat) {
                    if ((done + 3u) % 16u == 0) look_up(step + 3u);
                    load_scales(step + 3u, scales);
                }
            };
            if (early) next();
#pragma unroll
            for (uint32_t half = 0; half < 2; half += kHalves) compute(step, half);
            if (!early) next();
        }
    }

    const auto halves = __builtin_amdgcn_permlane32_swap(f32_bits(sum), f32_bits(sum), false, false);
    const float all = bits_f32(halves[0]) + bits_f32(halves[1]);
    if constexpr (!kFloat) {
        if (lost_below(least_key, key_power)) lost[0] = 1u;
        if (lost_below(least_value, value_power)) lost[1] = 1u;
    }
    __syncthreads();
    const auto again = [&](bool whole, Losses losses) {
        __syncthreads();
        rows_again<kDim>(at.s.index, at.row0, at.rows, part, parts, kv_head, static_cast<int64_t>(step0 + from) * S::kKeys, static_cast<int64_t>(step0 + to) * S::kKeys - 1, whole, losses,
                         reinterpret_cast<float*>(lds));
    };
    if (*found) {
        again(true, Losses{});
        return;
    }

    const auto store = [&](const AttentionArgs& a, const Split& split) {
        if (own >= at.rows) return;
        const float up = kFloat ? 1.0f : (kExact ? 1.0f : 2.0f) * ldexpf(1.0f, out_power), by = all == 0.0f ? 0.0f : 1.0f / all;
        const uint32_t row = row_of(), head = kv_head * a.group + row % a.group;
        const uint64_t token = at.s.first + row / a.group, of = (token * a.heads + head) * split.splits + part;
        if (parts > 1 && h == 0 && first_out == 0) split.stats[2 * of] = top, split.stats[2 * of + 1] = all;
#pragma unroll
        for (uint32_t e = 0; e < kOut; e++)
#pragma unroll
            for (uint32_t v = 0; v < 16; v += 4) {
                const uint32_t d = (first_out + e) * 32u + v * 2u + 4u * h;
                if (d >= dim) continue;
                f32x4 four;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) four[i] = all == 0.0f ? 0.0f : out[e][v + i] * by * up;
                if (parts > 1)
                    *reinterpret_cast<f32x4*>(split.parts + of * dim + d) = four;
                else
                    *reinterpret_cast<u32x2*>(a.y + (token * a.y_token + head * a.y_head + d) * 2u) =
                        a.dtype == CQ_BF16 ? u32x2{pair_of<true>(four[0], four[1]), pair_of<true>(four[2], four[3])} : u32x2{pair_of<false>(four[0], four[1]), pair_of<false>(four[2], four[3])};
            }
    };
    if constexpr (kExact) {  // whose scalar registers are short (8191 tokens 912 us, and 926 with the arguments kept)
        const Arguments& late = arguments_again();
        store(late.a, late.split);
    } else {
        store(a, split);
    }
    if constexpr (!kFloat) {
        if ((lost[0] | lost[1]) == 0u) return;
        // a score is off by 2^-25 of numbers whose unit is 2^(key_power + 1), times the queries; a result by as much of values' scales, times a code, where those are numbers
        Losses losses{};
        if (lost[0]) losses.key = ldexpf(fabsf(a.scale) * kLog2E, key_power - 24);
        if (lost[1]) losses.value = kExact ? lost_by_weights<kCode>((to - from) * S::kKeys, value_power) : ldexpf(kMostCode<kCode>, value_power - 24);
        again(false, losses);
    }
}

template <int kCode, int kDim, bool kBF16, bool kExact>
hipError_t launch_many(hipStream_t s, const AttentionArgs& a, const Split& split) {
    using S = Many<kCode, kDim>;
    constexpr uint32_t kLds = 2 * S::kBuffer + 32 + (kExact ? 4 * (kDim / 32) * S::kKeys * 4 : 0);
    hipLaunchKernelGGL((attention_many_kernel<kCode, kDim, kBF16, kExact>), dim3(split.tiles * split.splits * a.cache.kv_heads), dim3(S::kThreads), kLds, s, a, split);
    return hipGetLastError();
}

// A number of f16 is rounded to 11 bits: hardly more than a result of bf16 shows (8191 tokens of fp8: off by 0.0018 of its norm, 0.0017 of it the result's own rounding; of codes 0.0017,
// for 40 % more time), more than one of f16 does (0.0012 and 0.0002), so those are made of the codes.
template <int kCode, int kDim>
hipError_t launch_type(hipStream_t s, const AttentionArgs& a, const Split& split) {
    if constexpr (kCode == kCacheFloat) {
        if (a.dtype == CQ_BF16) return launch_many<kCode, kDim, true, false>(s, a, split);
        return launch_many<kCode, kDim, false, false>(s, a, split);
    } else {
        if (a.dtype == CQ_BF16) return launch_many<kCode, kDim, false, false>(s, a, split);
        return launch_many<kCode, kDim, false, true>(s, a, split);
    }
}

}  // namespace

#define CQ_MANY_NAME2(c) launch_attention_many_##c
#define CQ_MANY_NAME(c) CQ_MANY_NAME2(c)
hipError_t CQ_MANY_NAME(CQ_TU_CODE)(hipStream_t s, const AttentionArgs& a, const Split& split) {
    if (a.cache.dim <= 64) return launch_type<CQ_TU_CODE, 64>(s, a, split);
    if (a.cache.dim <= 128) return launch_type<CQ_TU_CODE, 128>(s, a, split);
    return launch_type<CQ_TU_CODE, 256>(s, a, split);
}

}  // namespace cq
