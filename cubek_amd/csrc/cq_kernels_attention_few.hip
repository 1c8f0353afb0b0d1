// Attention of few rows (token, head of a group) over long caches: decode steps, drafts of some tokens.  An object per kind of code (CQ_TU_CODE).
//
// A workgroup takes a tile of 16 or 32 rows that share a head of the cache, and a split of the keys they see; its four or eight waves take steps
// of 32 keys (64 of 4 bits) in turn, each with a running maximum, sum and result of its own, which meet in LDS at the end; the results of several
// splits meet in attention_join_kernel.  Everything else stays in registers:
//   S^T = K Q^T by 16 x 16 x 32 matrix instructions: lane (i, g) has 16 bytes of key i, and gets the scores of row i with the keys 4 g ... 4 g + 3 of a
//   tile of 16, which are the operand that the second product takes: O^T = V^T P^T with the keys in that order.
//   V goes through LDS, each wave's own part (no barrier), and comes back by transposing reads, a lane eight keys of one entry.
// Codes enter as themselves, exact in f16, keys' scales in f32 behind the first product, values' scales in front of the second, on the weights: no
// entry is rounded, and a value of the cache costs 1.25 vector instructions at 8 bits (0.5 of fp8) instead of the 2.5 to 4 of its dequantization.
// Where a scale covers 32 entries of a longer head, lanes swap parts so that one instruction has one block (`kPer` > 1).
// Queries are scaled by a power of two per row, weights by one of the largest scale so far, so that f16 holds them whatever the range of bf16 (kSpread says how far apart scales may
// be).  Weights with their value's scale are rounded to the 11 bits of f16, and over bf16 floats to two numbers of bf16; of bf16 queries what is below 2^-14 of the largest loses bits.
//
// Bound by the read of the cache where sequences are many and long (64 of 4096 keys, 8 heads of 128 of i8: 100 us, 5.5 TB/s; lengths from 257 to 8191: 117,
// 4.9 TB/s); by vector instructions at 4 bits with a scale for 32 entries (one sequence of 131071 keys: 46 us of which 5 join 64 parts,
// 3.3 TB/s, vector units busy 53 %); where there is little to read, by a launch and four rounds of loads that need each other, lengths, pages, codes, and
// then a wave's steps one after another (24 tiles of up to 701 keys: 14 us).
#include <hip/hip_runtime.h>

#include "cq_attention_tiles.hpp"
#include "cq_magic_div.hpp"

namespace cq {
namespace {

// Between a wave's writes to its part of LDS and its reads from it: LDS serves a wave in order, so only the compiler has to keep it.
__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }

template <int kCode, int kDim, int kPer>
struct Shape {
    static constexpr uint32_t kBits = kCodeBits<kCode>;
    static constexpr uint32_t kKeyTiles = kBits == 4 ? 4 : 2, kKeys = 16 * kKeyTiles;  // of a step
    static constexpr uint32_t kRow = kDim * kBits / 8;                                 // bytes of a key
    static constexpr uint32_t kUnits = kRow >= 64 ? kRow / 64 : 1, kWords = kRow >= 64 ? 4 : 2;  // loads of a lane for a key; words of one
    static constexpr uint32_t kEntries = kWords * 32 / kBits, kCover = 4 * kEntries, kUnit = kDim / kPer;               // of a lane's load; of its four groups; of a scale
    static constexpr uint32_t kSlices = kDim / 32;                                     // matrix instructions of a tile of keys
    static constexpr uint32_t kLane = 16, kLanes = kRow / kLane, kLoads = kKeys * kRow / 1024;  // of values: bytes of a lane, lanes of a row, loads of a step
    static constexpr uint32_t kPitch = kRow + 16;                                      // bytes of a row in LDS: 16 keys' reads fall on different banks
    static constexpr uint32_t kScaleLoads = kCode == kCacheFloat ? 0 : (kPer * 16 + 63) / 64;           // of 16 keys' scales, of keys or of values
    static constexpr uint32_t kValueBytes = kKeys * kPitch, kScaleBytes = kCode == kCacheFloat ? 0 : 2 * kPer * kKeys * 4, kWaveBytes = kValueBytes + kScaleBytes;
};

// The first product takes entries in slices of 32, eight of a lane.  A lane's load of a key has kEntries of them in a row, and the four groups of lanes have
// kCover together.  Where a scale covers as many or more, a slice is what the lanes' words at one place are.  Where it covers half of them, lanes 0 - 31
// and 32 - 63 exchange words (swap_halves), where a quarter also neighbouring groups (swap_quarters), so that every slice has one scale.
template <int kCode, int kDim, int kPer>
__device__ __forceinline__ uint32_t slice_entry(uint32_t t, uint32_t g) {
    using S = Shape<kCode, kDim, kPer>;
    if constexpr (S::kBits == 16 || S::kUnit * 4 == S::kCover) return 32u * t + 8u * g;
    constexpr uint32_t kOf = S::kEntries / 8;  // slices of a load
    const uint32_t from = t / kOf * S::kCover, in = t % kOf;
    if constexpr (S::kUnit * 2 == S::kCover) return from + in / (kOf / 2) * (S::kCover / 2) + g % 2u * S::kEntries + g / 2u * (S::kEntries / 2) + in % (kOf / 2) * 8u;
    return from + g * S::kEntries + in * 8u;
}

__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ void swap_quarters(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}

// Whether 16 bytes of codes have one that is infinite or not a number.
template <int kCode, bool kBF16>
__device__ __forceinline__ bool code_is_odd(u32x4 v) {
    if constexpr (kCode == kCacheFloat) return has_odd<kBF16>(v);
    constexpr uint32_t kMask = kCode == kCacheE4M3 ? 0x7fu : 0x7cu;  // e4m3 has one NaN; e5m2's largest exponent is infinity and NaN
    bool found = false;
#pragma unroll
    for (uint32_t p = 0; p < 4; p++) {
        const uint32_t w = v[p];
#pragma unroll
        for (uint32_t b = 0; b < 32; b += 8) found = found || (w >> b & kMask) == kMask;
    }
    return found;
}

// Waves per SIMD that registers are kept for: the most that builds show to need no scratch memory.  (Compiled for one more, loads of spilled registers stood in the loop: 64 tokens
// over 4 bits in blocks of 32, heads of 256, 604 us, 188 without them; five drafted tokens of 20 rows 178 and 76, over 8 bits 178 and 57.)
template <int kCode, int kDim, int kPer, int kTiles>
constexpr int waves_of() {
    constexpr bool kNibbles = kCodeBits<kCode> == 4;
    if (kDim == 64) return kTiles == 1 ? 4 : kNibbles ? 2 : 3;
    if (kDim == 128 && kTiles == 1) return kCode == kCacheFloat || (kNibbles && kPer > 1) ? 2 : 3;
    if (kDim == 128) return kNibbles && kPer > 1 ? 1 : 2;
    return kCode == kCacheFloat ? 1 : 2;
}
// Where that takes it, queries stay in LDS, the same for all waves, and the compiler may not move operands of one tile in front of another's.
template <int kCode, int kDim, int kPer, int kTiles>
constexpr bool kTight = kDim == 256 || kTiles == 2 || (kCodeBits<kCode> == 4 && kDim == 128 && kPer == 1);

// of a workgroup, at most
template <int kCode, int kDim, int kPer, int kTiles>
constexpr uint32_t kMostWaves = waves_of<kCode, kDim, kPer, kTiles>() == 1 ? 4 : 8;

template <int kCode, int kDim, int kPer, int kTiles, bool kBF16>
__global__ __launch_bounds__((64 * kMostWaves<kCode, kDim, kPer, kTiles>), (waves_of<kCode, kDim, kPer, kTiles>())) void attention_few_kernel(AttentionArgs a, Split split) {
    using S = Shape<kCode, kDim, kPer>;
    constexpr bool kFloat = kCode == kCacheFloat;
    constexpr uint32_t kRowsLog2 = kTiles == 1 ? 4 : 5, kRows = 16 * kTiles;
    constexpr uint32_t kOut = kDim / 16;  // tiles of 16 entries of the result
    constexpr bool kShort = kTight<kCode, kDim, kPer, kTiles>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15u, g = lane >> 4;
    // neighbours in the grid are heads of the cache, whose entries lie side by side
    const uint32_t kv_head = blockIdx.x % a.cache.kv_heads, dim = a.cache.dim;
    const uint32_t waves = split.waves;  // 4 or 8
    char* const mine = lds + wave * S::kWaveBytes;
    float* const scales_at = reinterpret_cast<float*>(mine + S::kValueBytes);

    RowTile at;
    uint32_t steps_wanted, part;
    if (!find_rows_and_steps<false>(a, split, blockIdx.x / a.cache.kv_heads, kRowsLog2, S::kKeyTiles == 4 ? 6 : 5, &at, &steps_wanted, &part)) return;
    // the keys that some row of the tile sees, and those that all of them do
    const int32_t first_position = at.s.position + static_cast<int32_t>(at.row0 / a.group), last_position = at.s.position + static_cast<int32_t>((at.row0 + at.rows - 1u) / a.group);
    const Seen first = seen_from(a, at.s, first_position), last = seen_from(a, at.s, last_position);
    const int32_t low = first.low, high = last.high, all_low = last.low, all_high = first.high;
    const uint32_t step0 = static_cast<uint32_t>(low) / S::kKeys, steps_all = high < low ? 0u : static_cast<uint32_t>(high) / S::kKeys + 1u - step0;
    // the nearest number of parts, so that a few steps too many do not make another one (five tokens of eight sequences within a window of 4096: 36 us, and 46)
    const uint32_t parts = min(max((steps_all + steps_wanted / 2u) / steps_wanted, 1u), split.splits);
    if (part >= parts) return;
    if (split.splits > 1 && part == 0) note_parts(a, split, at, kv_head, parts);
    // Where all tiles together would have more parts than split.wanted, which is about as many as the GPU holds at once, the later ones, which start last, are smaller, from 3/2 of
    // the mean down to 1/2, so that all end together (64 sequences of 257 to 8191 keys: 120 us of equal parts, 117; 200 of 257 to 4000: 187 and 181).  Else all are equal (one of
    // 131071: 46, and 52), and so they are of few tiles (up to 32 with keys to split), whose kMostSplits parts each are no more than the GPU holds whatever their length.
    uint32_t from, to;
    if (steps_wanted > split.enough && split.splits < kMostSplits) {
        const float by = static_cast<float>(steps_all) / static_cast<float>(2u * parts * parts);
        const auto begin_of = [&](uint32_t p) { return static_cast<uint32_t>(by * static_cast<float>(p * (3u * parts - p))); };
        from = begin_of(part), to = part + 1u < parts ? begin_of(part + 1u) : steps_all;
    } else {
        const uint32_t each = (steps_all + parts - 1u) / parts;
        from = min(part * each, steps_all), to = min(from + each, steps_all);
    }
    const uint32_t last_tile = static_cast<uint32_t>(max(high, 0)) / 16u;

    // queries: row i of each tile of 16
    u32x4 q[kTiles][S::kSlices];
    float times[kTiles], slope[kTiles];
    int32_t position[kTiles], row_low[kTiles], row_high[kTiles];
#pragma unroll
    for (uint32_t r = 0; r < kTiles; r++) {
        const uint32_t row = min(r * 16u + i, at.rows - 1u) + at.row0, token = at.s.first + row / a.group, head = kv_head * a.group + row % a.group;
        position[r] = at.s.position + static_cast<int32_t>(row / a.group);
        const Seen seen = seen_from(a, at.s, position[r]);
        row_low[r] = seen.low, row_high[r] = r * 16u + i < at.rows ? seen.high : -1;
        slope[r] = a.slopes ? a.slopes[head] * kLog2E : 0.0f;
        const char* const from_q = a.q + (token * a.q_token + head * a.q_head) * 2u;
        float most = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < S::kSlices; t++) {
            const uint32_t d = slice_entry<kCode, kDim, kPer>(t, g);
            q[r][t] = d < dim ? *reinterpret_cast<const u32x4*>(from_q + d * 2u) : u32x4{0, 0, 0, 0};
        }
        if (a.scale < 0.0f) {  // into the queries: the largest score is that of the largest product
#pragma unroll
            for (uint32_t t = 0; t < S::kSlices; t++) q[r][t] ^= 0x80008000u;
        }
        if constexpr (!kFloat) {
            float v[8];
            const bool bf16 = a.dtype == CQ_BF16;
#pragma unroll
            for (uint32_t t = 0; t < S::kSlices; t++) {
                if (bf16)
                    BF16::unpack(q[r][t], v);
                else
                    F16::unpack(q[r][t], v);
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) most = fmaxf(most, fabsf(v[e]));
            }
            most = max_of_groups(most);
            const uint32_t power = power_of_row(most, bf16);
            const float down = bits_f32((254u - power) << 23);
#pragma unroll
            for (uint32_t t = 0; t < S::kSlices; t++) {
                if (bf16)
                    BF16::unpack(q[r][t], v);
                else
                    F16::unpack(q[r][t], v);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) q[r][t][e] = pair_of<false>(v[place_of<kCode>(2 * e)] * down, v[place_of<kCode>(2 * e + 1)] * down);
            }
            times[r] = fabsf(a.scale) * bits_f32(power << 23);
        } else {
            times[r] = fabsf(a.scale);
        }
        // with a cap: 2 log2(e) t / cap, the exponent of its tanh; else log2(e) t
        times[r] = a.cap > 0.0f ? times_of_cap(times[r], a.cap) : times[r] * kLog2E;
    }
    const float cap = cap_log2(a.cap);
    u32x4* const queries = reinterpret_cast<u32x4*>(lds + waves * S::kWaveBytes);  // [tile of rows][slice][lane], the same for all waves
    if constexpr (kShort) {
        if (wave == 0)
#pragma unroll
            for (uint32_t r = 0; r < kTiles; r++)
#pragma unroll
                for (uint32_t t = 0; t < S::kSlices; t++) queries[(r * S::kSlices + t) * 64u + lane] = q[r][t];
        __syncthreads();
    }
    const auto query = [&](uint32_t r, uint32_t t) { return kShort ? queries[(r * S::kSlices + t) * 64u + lane] : q[r][t]; };

    // Pages of the wave's next 64 / kKeyTiles steps, a lane a tile of 16 keys.
    const uint32_t tiles_of_page = a.cache.page_size / 16u;
    const auto tile_of = [&](uint32_t step, uint32_t k) { return min((step0 + step) * S::kKeyTiles + k, last_tile); };
    constexpr uint32_t kAhead = 64 / S::kKeyTiles;
    uint32_t pages = 0;
    const auto look_up = [&](uint32_t step) {
        const uint32_t t = tile_of(step + lane / S::kKeyTiles * waves, lane % S::kKeyTiles);
        pages = page_of(a, at.s, magic_div(t, split.page_magic, split.page_shift));
    };

    // A step's loads.
    struct Raw {
        uint32_t k[S::kKeyTiles][S::kUnits][S::kWords];
        u32x4 v[S::kLoads];
        uint32_t scale[2][S::kKeyTiles][S::kScaleLoads ? S::kScaleLoads : 1], odd;  // of keys, of values; bits 2 (side * kKeyTiles + tile) ...: half a word that a tile's begin with
    };
    const ScaleWords words(a.cache.param_dtype);
    const uint32_t row_bytes = dim * S::kBits / 8u;
    const auto key_byte = [&](uint32_t u) { return u * 64u + g * (4u * S::kWords); };
    constexpr uint32_t kKeysOfLoad = 64 / S::kLanes;  // 32 where rows are 32 bytes
    constexpr bool kOwn = kDim < 256;                 // an offset for each load of values; else one, and what all lanes have in common beside it
    const uint32_t key_row = i * static_cast<uint32_t>(a.cache.keys.slot);
    uint32_t key_offset[S::kUnits];
#pragma unroll
    for (uint32_t u = 0; u < S::kUnits; u++) key_offset[u] = key_row + min(key_byte(u), row_bytes - 4u * S::kWords);
    const auto key_at = [&](uint32_t u) {
        if constexpr (!kFloat || kDim < 256) return key_offset[u];
        uint32_t first = g * 16u;  // worked out at each load: eight of them take registers that there are not
        asm volatile("" : "+v"(first));
        return key_row + min(u * 64u + first, row_bytes - 16u);
    };
    uint32_t value_offset[kOwn ? S::kLoads : 1];
#pragma unroll
    for (uint32_t n = 0; n < (kOwn ? S::kLoads : 1); n++)
        value_offset[n] = (n * 64u + lane) / S::kLanes % 16u * static_cast<uint32_t>(a.cache.values.slot) + min(lane % S::kLanes * S::kLane, row_bytes - S::kLane);
    // The scales of a tile of 16 keys: lane l has unit l % kPer of key l / kPer (of 256 entries in two loads, whose keys are 64 / kPer apart: whole words).
    const uint32_t scale_unit = lane % kPer, scale_lane_key = lane / kPer % 16u;
    const auto scale_key = [&](uint32_t n) { return scale_lane_key + n * (64u / kPer); };
    uint32_t scale_offset[2] = {};
    if constexpr (!kFloat) {
        const uint32_t block = min(scale_unit * S::kUnit, dim - 1u) >> split.block_log2;
        scale_offset[0] = (scale_lane_key * static_cast<uint32_t>(a.cache.keys.scale_slot) + block * static_cast<uint32_t>(a.cache.keys.scale_block)) << words.log2;
        scale_offset[1] = (scale_lane_key * static_cast<uint32_t>(a.cache.values.scale_slot) + block * static_cast<uint32_t>(a.cache.values.scale_block)) << words.log2;
    }
    const char* const keys_base = a.cache.keys.base + kv_head * a.cache.keys.head;
    const char* const values_base = a.cache.values.base + kv_head * a.cache.values.head;
    const char* const key_scales = a.cache.keys.scales + (kv_head * a.cache.keys.scale_head << words.log2);
    const char* const value_scales = a.cache.values.scales + (kv_head * a.cache.values.scale_head << words.log2);
    const auto place_of_tile = [&](uint32_t t) { return (t - magic_div(t, split.page_magic, split.page_shift) * tiles_of_page) * 16u; };
    // where a tile of 16 keys lies: its page (of the wave's next steps, by readlane) and its first slot there
    const auto find_tile = [&](uint32_t step, uint32_t nth, uint32_t k, uint32_t* page, uint32_t* place) {
        *page = __builtin_amdgcn_readlane(pages, (nth % kAhead) * S::kKeyTiles + k);
        *place = place_of_tile(tile_of(step, k));
    };
    const auto offset_of = [](uint32_t page, uint64_t page_stride, uint32_t place, uint64_t slot_stride) {
        return static_cast<uint64_t>(page) * static_cast<uint32_t>(page_stride) + place * static_cast<uint32_t>(slot_stride);
    };
    const auto load_keys = [&](uint32_t step, uint32_t nth, Raw& raw) {
#pragma unroll
        for (uint32_t k = 0; k < S::kKeyTiles; k++) {
            uint32_t page, place;
            find_tile(step, nth, k, &page, &place);
            const char* const rows = keys_base + offset_of(page, a.cache.keys.page, place, a.cache.keys.slot);
#pragma unroll
            for (uint32_t u = 0; u < S::kUnits; u++) {
                if constexpr (S::kWords == 4) {
                    const u32x4 w = stream_load(reinterpret_cast<const u32x4*>(rows + key_at(u)));
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) raw.k[k][u][e] = w[e];
                } else {
                    const u32x2 w = stream_load(reinterpret_cast<const u32x2*>(rows + key_at(u)));
                    raw.k[k][u][0] = w[0], raw.k[k][u][1] = w[1];
                }
            }
        }
    };
    const auto load_values = [&](uint32_t step, uint32_t nth, Raw& raw) {
        uint32_t page[S::kKeyTiles], place[S::kKeyTiles];
#pragma unroll
        for (uint32_t k = 0; k < S::kKeyTiles; k++) find_tile(step, nth, k, &page[k], &place[k]);
#pragma unroll
        for (uint32_t n = 0; n < S::kLoads; n++) {
            const uint32_t k = n * kKeysOfLoad / 16u;
            uint64_t rows = offset_of(page[k], a.cache.values.page, place[k] + (kOwn ? 0u : n * kKeysOfLoad % 16u), a.cache.values.slot);
            if constexpr (kKeysOfLoad > 16) {
                const uint64_t second = offset_of(page[k + 1], a.cache.values.page, place[k + 1], a.cache.values.slot);
                rows = lane / S::kLanes >= 16u ? second : rows;
            }
            raw.v[n] = stream_load(reinterpret_cast<const u32x4*>(values_base + rows + value_offset[kOwn ? n : 0]));
        }
        if constexpr (!kFloat) {
            raw.odd = 0;
#pragma unroll
            for (uint32_t k = 0; k < S::kKeyTiles; k++) {
                const char* const of[2] = {key_scales + (offset_of(page[k], a.cache.keys.scale_page, place[k], a.cache.keys.scale_slot) << words.log2),
                                           value_scales + (offset_of(page[k], a.cache.values.scale_page, place[k], a.cache.values.scale_slot) << words.log2)};
#pragma unroll
                for (uint32_t side = 0; side < 2; side++) {
                    // words: from a word's start on, and half a word further where the tile's first scale is
                    const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(of[side])) & 2u;
                    raw.odd |= odd << (2 * (side * S::kKeyTiles + k));
#pragma unroll
                    for (uint32_t n = 0; n < S::kScaleLoads; n++) {
                        const uint64_t further = n * (64u / kPer) * static_cast<uint64_t>(static_cast<uint32_t>((side == 0 ? a.cache.keys : a.cache.values).scale_slot)) << words.log2;
                        raw.scale[side][k][n] = *reinterpret_cast<const uint32_t*>(of[side] + further - odd + ((scale_offset[side] + odd) & ~3u));
                    }
                }
            }
        }
    };

    f32x4 out[kTiles][kOut] = {};
    float top[kTiles], sum[kTiles];
#pragma unroll
    for (uint32_t r = 0; r < kTiles; r++) top[r] = -INFINITY, sum[r] = 0.0f;
    bool found = false;    // values that are no numbers, among keys that not every row sees
    int32_t power = -126;  // of the largest scale of the values so far: they are taken times 2^-power
    uint32_t least = ~0u;  // of the smallest (smaller_of)

    Raw raw;
    uint32_t nth = 0;
    if (from + wave < to) {
        look_up(from + wave);
        load_values(from + wave, 0, raw);
        load_keys(from + wave, 0, raw);
    }
    for (uint32_t step = from + wave; step < to; step += waves, nth++) {
        if ((nth + 1u) % kAhead == 0) look_up(step + waves);
        const int32_t key0 = static_cast<int32_t>((step0 + step) * S::kKeys);
        const bool partial = key0 < all_low || key0 + static_cast<int32_t>(S::kKeys) - 1 > all_high;

        // this step's values and scales into LDS; of values that can be no numbers those that no row sees become zeros, and others are reported
        if constexpr (kCodeHasNaN<kCode>) {
            if (partial) {
                bool odd = false;
#pragma unroll
                for (uint32_t n = 0; n < S::kLoads; n++) {
                    const int32_t key = key0 + static_cast<int32_t>((n * 64u + lane) / S::kLanes);
                    if (key < low || key > high) raw.v[n] = u32x4{0, 0, 0, 0};
                    odd = odd || code_is_odd<kCode, kBF16>(raw.v[n]);
                }
                found = found || __builtin_amdgcn_ballot_w64(odd) != 0;
            }
        }
#pragma unroll
        for (uint32_t n = 0; n < S::kLoads; n++)
            *reinterpret_cast<u32x4*>(mine + (n * 64u + lane) / S::kLanes * S::kPitch + lane % S::kLanes * S::kLane) = raw.v[n];
        if constexpr (!kFloat) {
            float scale[2][S::kKeyTiles][S::kScaleLoads], most = 0.0f;
#pragma unroll
            for (uint32_t side = 0; side < 2; side++)
#pragma unroll
                for (uint32_t k = 0; k < S::kKeyTiles; k++)
#pragma unroll
                    for (uint32_t n = 0; n < S::kScaleLoads; n++)
                        scale[side][k][n] = words.number(raw.scale[side][k][n], scale_offset[side] + (raw.odd >> (2 * (side * S::kKeyTiles + k)) & 2u));
            if (partial) {
                bool odd = false;
#pragma unroll
                for (uint32_t k = 0; k < S::kKeyTiles; k++)
#pragma unroll
                    for (uint32_t n = 0; n < S::kScaleLoads; n++) {
                        const int32_t key = key0 + static_cast<int32_t>(k * 16u + scale_key(n));
                        if (key < low || key > high) scale[0][k][n] = scale[1][k][n] = 0.0f;  // what no row sees is not looked at
                        odd = odd || !(fabsf(scale[1][k][n]) < INFINITY);
                    }
                found = found || __builtin_amdgcn_ballot_w64(odd) != 0;
            }
#pragma unroll
            for (uint32_t k = 0; k < S::kKeyTiles; k++)
#pragma unroll
                for (uint32_t n = 0; n < S::kScaleLoads; n++) most = fmaxf(most, fabsf(scale[1][k][n])), least = smaller_of(least, scale[1][k][n]);
            if (__builtin_amdgcn_ballot_w64(!(most < bits_f32(static_cast<uint32_t>(128 + power) << 23)))) {  // 2^(power + 1)
                uint32_t field = 0;
#pragma unroll
                for (uint32_t k = 0; k < S::kKeyTiles; k++)
#pragma unroll
                    for (uint32_t n = 0; n < S::kScaleLoads; n++) field = max(field, exponent_of(scale[1][k][n]));
                const int32_t now = max(power, min(static_cast<int32_t>(__builtin_amdgcn_readfirstlane(wave_max_bits(field))) - 127, 126));
                const float shrink = ldexpf(1.0f, power - now);
                power = now;
#pragma unroll
                for (uint32_t r = 0; r < kTiles; r++)
#pragma unroll
                    for (uint32_t e = 0; e < kOut; e++) out[r][e] *= shrink;
            }
            const float down = bits_f32(static_cast<uint32_t>(127 - power) << 23);
#pragma unroll
            for (uint32_t k = 0; k < S::kKeyTiles; k++)
#pragma unroll
                for (uint32_t n = 0; n < S::kScaleLoads; n++) {
                    float* const to = scales_at + scale_unit * S::kKeys + k * 16u + scale_key(n);  // (of 16 or 32 scales some lanes write the same)
                    to[0] = scale[0][k][n];
                    to[kPer * S::kKeys] = scale[1][k][n] * down;
                }
        }
        fence();
        // the next step's, into the registers that have gone to LDS; its keys behind this step's scores
        load_values(step + waves, nth + 1u, raw);

        // scores
        f32x4 s[kTiles][S::kKeyTiles];
#pragma unroll
        for (uint32_t k = 0; k < S::kKeyTiles; k++) {
            if constexpr (kShort) __builtin_amdgcn_sched_barrier(0);
            u32x4 operand[S::kSlices];
#pragma unroll
            for (uint32_t u = 0; u < S::kUnits; u++) {
                uint32_t* const w = raw.k[k][u];
                if constexpr (kCodeHasNaN<kCode>) {  // past a shorter head's end queries are zero, which these codes may not be multiplied by
#pragma unroll
                    for (uint32_t e = 0; e < S::kWords; e++) w[e] = key_byte(u) < row_bytes ? w[e] : 0u;
                }
                if constexpr (!kFloat && S::kUnit < S::kCover) {
                    if constexpr (S::kWords == 4)
                        swap_halves(w[0], w[2]), swap_halves(w[1], w[3]);
                    else
                        swap_halves(w[0], w[1]);
                    if constexpr (S::kUnit * 4 == S::kCover) swap_quarters(w[0], w[1]), swap_quarters(w[2], w[3]);
                }
                if constexpr (kFloat) {
                    operand[u] = u32x4{w[0], w[1], w[2], w[3]};
                } else if constexpr (S::kBits == 8) {
                    operand[2 * u] = numbers<kCode>(w[0], w[1]);
                    operand[2 * u + 1] = numbers<kCode>(w[2], w[3]);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < S::kWords; e++) operand[u * S::kWords + e] = numbers<kCode>(w[e], 0);
                }
            }
            if constexpr (kPer == 1) {
                f32x4 by = {1.0f, 1.0f, 1.0f, 1.0f};
                if constexpr (!kFloat) by = *reinterpret_cast<const f32x4*>(scales_at + k * 16u + 4u * g);
#pragma unroll
                for (uint32_t r = 0; r < kTiles; r++) {
                    f32x4 v = {};
#pragma unroll
                    for (uint32_t t = 0; t < S::kSlices; t++) v = mfma16<kBF16>(operand[t], query(r, t), v);
                    s[r][k] = kFloat ? v : v * by;
                }
            } else {
#pragma unroll
                for (uint32_t unit = 0; unit < kPer; unit++) {
                    const f32x4 by = *reinterpret_cast<const f32x4*>(scales_at + unit * S::kKeys + k * 16u + 4u * g);
#pragma unroll
                    for (uint32_t r = 0; r < kTiles; r++) {
                        f32x4 v = {};
#pragma unroll
                        for (uint32_t t = unit * S::kUnit / 32; t < (unit + 1) * S::kUnit / 32; t++) v = mfma16<kBF16>(operand[t], query(r, t), v);
                        s[r][k] = unit == 0 ? v * by : __builtin_elementwise_fma(v, by, s[r][k]);
                    }
                }
            }
        }

        load_keys(step + waves, nth + 1u, raw);

        // weights
        float p[kTiles][S::kKeyTiles * 4];
#pragma unroll
        for (uint32_t r = 0; r < kTiles; r++) {
            float t[S::kKeyTiles * 4];
#pragma unroll
            for (uint32_t i = 0; i < S::kKeyTiles * 4; i++) t[i] = s[r][i / 4u][i % 4u];
            const float times_now = shape_scores<S::kBits == 8 && (kDim == 256 || kTiles == 2)>(t, times[r], cap, a.slopes, slope[r], position[r], key0 + static_cast<int32_t>(4u * g), [](uint32_t i) { return i / 4u * 16u + i % 4u; },
                                                 key0 + static_cast<int32_t>(S::kKeys) - 1 <= first_position, partial, row_low[r], row_high[r]);
            float most = -INFINITY;
#pragma unroll
            for (uint32_t i = 0; i < S::kKeyTiles * 4; i++) most = fmaxf(most, t[i]);
            most = max_of_groups(most * times_now);
            if (__builtin_amdgcn_ballot_w64(most > top[r] + kLazy)) {
                const float before = top[r];
                top[r] = fmaxf(top[r], most);
                const float shrink = top[r] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(before - top[r]);
                sum[r] *= shrink;
#pragma unroll
                for (uint32_t e = 0; e < kOut; e++) out[r][e] *= shrink;
            }
            const float less = kWeightLog2 - (top[r] == -INFINITY ? 0.0f : top[r]);
#pragma unroll
            for (uint32_t i = 0; i < S::kKeyTiles * 4; i++) {
                p[r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[i], times_now, less));
                sum[r] += p[r][i];
            }
        }

        const auto weights_of = [&](uint32_t r, uint32_t block, uint32_t half) {
            float w[8];
#pragma unroll
            for (uint32_t k = 0; k < 2; k++) {
                f32x4 by = {1.0f, 1.0f, 1.0f, 1.0f};
                if constexpr (!kFloat) by = *reinterpret_cast<const f32x4*>(scales_at + (kPer + block) * S::kKeys + (half * 2u + k) * 16u + 4u * g);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    const float of = p[r][(half * 2u + k) * 4u + e];
                    w[k * 4 + e] = kFloat ? of : of * by[e];
                }
            }
            u32x4 packed;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) packed[e] = pair_of<kBF16>(w[place_of<kCode>(2 * e)], w[place_of<kCode>(2 * e + 1)]);
            return packed;
        };
        constexpr uint32_t kHalves = S::kKeyTiles / 2;  // matrix instructions of a step and a tile of entries
        const auto values_of = [&](uint32_t e, u32x4* v) {
            if constexpr (kFloat) {
#pragma unroll
                for (uint32_t k = 0; k < 2; k++) {
                    const auto four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(CQ_LDS_AT(i16x4, mine + (k * 16u + 4u * g + i / 4u) * S::kPitch + e * 32u + i % 4u * 8u));
                    const u32x2 w = __builtin_bit_cast(u32x2, four);
                    v[0][2 * k] = w[0], v[0][2 * k + 1] = w[1];
                }
            } else if constexpr (S::kBits == 8) {
                const auto w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(CQ_LDS_AT(i32x2, mine + (i / 8u * 16u + 4u * g + i / 2u % 4u) * S::kPitch + e * 16u + i % 2u * 8u));
                v[0] = numbers<kCode>(w[0], w[1]);
            } else {
                const auto w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(CQ_LDS_AT(i32x2, mine + (i / 4u * 16u + 4u * g + i % 4u) * S::kPitch + e * 8u));
                v[0] = numbers<kCode>(w[0], 0), v[1] = numbers<kCode>(w[1], 0);
            }
        };
        u32x4 w[kTiles][kHalves];
        // Weights over a cache of bf16, whose entries enter as they are, would have 8 bits: what these leave of them is multiplied as well, in time that the reads leave
        // (off by 0.0017 of the norm, which is the result's own rounding, instead of 0.0023; 64 tokens of 257 to 8191 keys 198 us with it and without).
        u32x4 rest[kBF16 ? kTiles : 1] = {};
        if constexpr (kBF16) {
#pragma unroll
            for (uint32_t r = 0; r < kTiles; r++) {
                w[r][0] = weights_of(r, 0, 0);
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) rest[r][i] = pair_of<true>(p[r][2 * i] - bits_f32(w[r][0][i] << 16), p[r][2 * i + 1] - bits_f32(w[r][0][i] & 0xffff0000u));
            }
        }
#pragma unroll
        for (uint32_t e = 0; e < kOut; e++) {
            if (!kBF16 && e % (S::kUnit / 16) == 0)
#pragma unroll
                for (uint32_t r = 0; r < kTiles; r++)
#pragma unroll
                    for (uint32_t half = 0; half < kHalves; half++) w[r][half] = weights_of(r, e / (S::kUnit / 16), half);
            if constexpr (kShort)
                if (e % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            u32x4 v[kHalves];
            values_of(e, v);
#pragma unroll
            for (uint32_t half = 0; half < kHalves; half++)
#pragma unroll
                for (uint32_t r = 0; r < kTiles; r++) {
                    out[r][e] = mfma16<kBF16>(v[half], w[r][half], out[r][e]);
                    if constexpr (kBF16) out[r][e] = mfma16<kBF16>(v[half], rest[r], out[r][e]);
                }
        }
        fence();
    }

    const bool whole = __syncthreads_or(found);
    // The waves' results, each by its share of the whole over its sum.  A tile of 16 entries of the result is finished by the wave e % waves, which the others
    // hand theirs.
    float* const tops = reinterpret_cast<float*>(lds);  // [wave][row]
    float* const sums = tops + waves * kRows;
    f32x4* const handed = reinterpret_cast<f32x4*>(sums + waves * kRows);  // [tile of rows][tile of entries][wave that hands][lane]
#pragma unroll
    for (uint32_t r = 0; r < kTiles; r++) {
        sum[r] = sum_of_groups(sum[r]);
        if (g == 0) tops[wave * kRows + r * 16u + i] = top[r], sums[wave * kRows + r * 16u + i] = sum[r];
    }
    const bool far = __syncthreads_or(!kFloat && lost_below(least, power));
    const float up = kFloat ? 1.0f : ldexpf(1.0f, power);
    float most[kTiles], all[kTiles];
#pragma unroll
    for (uint32_t r = 0; r < kTiles; r++) {
        most[r] = -INFINITY, all[r] = 0.0f;
        for (uint32_t w = 0; w < waves; w++) most[r] = fmaxf(most[r], tops[w * kRows + r * 16u + i]);
        const float zero = most[r] == -INFINITY ? 0.0f : most[r];
        for (uint32_t w = 0; w < waves; w++) all[r] += sums[w * kRows + r * 16u + i] * __builtin_amdgcn_exp2f(tops[w * kRows + r * 16u + i] - zero);
        const float share = sum[r] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top[r] - zero) / all[r];
#pragma unroll
        for (uint32_t e = 0; e < kOut; e++) {
            out[r][e] = sum[r] == 0.0f ? f32x4{} : out[r][e] * share * up;
            if ((e & (waves - 1u)) != wave) handed[((r * kOut + e) * (waves - 1u) + (wave - e - 1u & (waves - 1u))) * 64u + lane] = out[r][e];
        }
    }
    __syncthreads();
    const bool bf16 = a.dtype == CQ_BF16;
#pragma unroll
    for (uint32_t r = 0; r < kTiles; r++) {
        if (r * 16u + i >= at.rows) continue;
        const uint32_t in_sequence = at.row0 + r * 16u + i, token = at.s.first + in_sequence / a.group, head = kv_head * a.group + in_sequence % a.group;
        const uint64_t of = (static_cast<uint64_t>(token) * a.heads + head) * split.splits + part;
        if (parts > 1 && wave == 0 && g == 0) split.stats[2 * of] = most[r], split.stats[2 * of + 1] = all[r];
#pragma unroll
        for (uint32_t e = 0; e < kOut; e++) {
            const uint32_t d = e * 16u + 4u * g;
            if ((e & (waves - 1u)) != wave || d >= dim) continue;
            f32x4 v = out[r][e];
            for (uint32_t w = 0; w < waves - 1u; w++) v += handed[((r * kOut + e) * (waves - 1u) + w) * 64u + lane];
            if (parts > 1) {
                *reinterpret_cast<f32x4*>(split.parts + of * dim + d) = v;
            } else {
                const u32x2 w = bf16 ? u32x2{pair_of<true>(v[0], v[1]), pair_of<true>(v[2], v[3])} : u32x2{pair_of<false>(v[0], v[1]), pair_of<false>(v[2], v[3])};
                *reinterpret_cast<u32x2*>(a.y + (token * a.y_token + head * a.y_head + d) * 2u) = w;
            }
        }
    }
    if (!whole && !far) return;
    float* const losses = reinterpret_cast<float*>(lds);  // [wave]
    __syncthreads();
    if (lane == 0) losses[wave] = kFloat ? 0.0f : lost_by_weights<kCode>((to - from) * S::kKeys, power);
    __syncthreads();
    float most_lost = 0.0f;
    for (uint32_t w = 0; w < waves; w++) most_lost = fmaxf(most_lost, losses[w]);
    __syncthreads();
    rows_again<kDim>(at.s.index, at.row0, at.rows, part, parts, kv_head, static_cast<int64_t>(step0 + from) * S::kKeys, static_cast<int64_t>(step0 + to) * S::kKeys - 1, whole,
                     Losses{0.0f, most_lost}, reinterpret_cast<float*>(lds));
}

template <int kCode, int kDim, int kPer, int kTiles, bool kBF16>
hipError_t launch_few(hipStream_t s, const AttentionArgs& a, const Split& split) {
    using S = Shape<kCode, kDim, kPer>;
    const auto lds_of = [](uint32_t waves) {
        const uint32_t steps = waves * S::kWaveBytes + (kTight<kCode, kDim, kPer, kTiles> ? kTiles * S::kSlices * 1024 : 0), join = 2 * waves * 16 * kTiles * 4 + kTiles * (kDim / 16) * (waves - 1) * 1024;
        return steps > join ? steps : join;
    };
    // Where there are not even as many workgroups as compute units, eight waves each, which ask for twice as much at a time (24 workgroups with up to
    // 701 keys: 16.2 us of four waves, 14.2 of eight); their results have to fit in LDS.
    Split by = split;
    const uint32_t workgroups = split.tiles * a.cache.kv_heads * split.splits;
    constexpr uint32_t kMost = kMostWaves<kCode, kDim, kPer, kTiles>;
    by.waves = workgroups <= 256 && lds_of(kMost) <= 160 * 1024 - 512 ? kMost : 4;
    hipLaunchKernelGGL((attention_few_kernel<kCode, kDim, kPer, kTiles, kBF16>), dim3(workgroups), dim3(64 * by.waves), lds_of(by.waves), s, a, by);
    return hipGetLastError();
}

template <int kCode, int kDim, int kPer>
hipError_t launch_tiles(hipStream_t s, const AttentionArgs& a, const Split& split) {
    const auto by_type = [&](auto tiles) {
        if constexpr (kCode == kCacheFloat)
            if (a.dtype == CQ_BF16) return launch_few<kCode, kDim, kPer, tiles.value, true>(s, a, split);
        return launch_few<kCode, kDim, kPer, tiles.value, false>(s, a, split);
    };
    if constexpr (kDim < 256 || kCode == kCacheFloat)  // (split_of)
        if (split.row_tiles == 2) return by_type(std::integral_constant<int, 2>{});
    return by_type(std::integral_constant<int, 1>{});
}

template <int kCode, int kDim>
hipError_t launch_blocks(hipStream_t s, const AttentionArgs& a, const Split& split) {
    if constexpr (kCode != kCacheFloat) {
        const uint32_t block = a.cache.block;
        if (block < a.cache.dim) {
            if constexpr (kDim == 256) {
                if (block == 32) return launch_tiles<kCode, kDim, 8>(s, a, split);
                if (block == 64) return launch_tiles<kCode, kDim, 4>(s, a, split);
            } else if constexpr (kDim == 128) {
                if (block == 32) return launch_tiles<kCode, kDim, 4>(s, a, split);
            }
            return launch_tiles<kCode, kDim, 2>(s, a, split);
        }
    }
    return launch_tiles<kCode, kDim, 1>(s, a, split);
}

}  // namespace

#define CQ_FEW_NAME2(c) launch_attention_few_##c
#define CQ_FEW_NAME(c) CQ_FEW_NAME2(c)
hipError_t CQ_FEW_NAME(CQ_TU_CODE)(hipStream_t s, const AttentionArgs& a, const Split& split) {
    if (a.cache.dim <= 64) return launch_blocks<CQ_TU_CODE, 64>(s, a, split);
    if (a.cache.dim <= 128) return launch_blocks<CQ_TU_CODE, 128>(s, a, split);
    return launch_blocks<CQ_TU_CODE, 256>(s, a, split);
}

}  // namespace cq
