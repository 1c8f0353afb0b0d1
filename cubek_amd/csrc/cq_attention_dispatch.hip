// Which kernel a call of attention takes, and which object holds it.
#include "cq_attention_internal.hpp"
#include "cq_magic_div.hpp"

namespace cq {

hipError_t launch_append_F32(hipStream_t s, const AppendArgs& a);
hipError_t launch_append_F16(hipStream_t s, const AppendArgs& a);
hipError_t launch_append_BF16(hipStream_t s, const AppendArgs& a);

hipError_t launch_append(hipStream_t s, const AppendArgs& a) {
    return a.dtype == CQ_F32 ? launch_append_F32(s, a) : a.dtype == CQ_F16 ? launch_append_F16(s, a) : launch_append_BF16(s, a);
}

namespace {

uint32_t log2_below(uint64_t v) {
    uint32_t l = 0;
    while (v >>= 1) l++;
    return l;
}

// Whether the matrix cores take a call: 16-bit queries, heads of whole 32 entries up to 256, pages of whole 16 slots, a scale for 32, 64, 128 ...
// entries or for a head, rows on 16-byte boundaries, a page within 32 bits.
bool tiles_take(const AttentionArgs& a) {
    const CacheArgs& c = a.cache;
    if (a.dtype == CQ_F32 || c.dim % 32 || c.dim > 256 || c.page_size % 16) return false;
    if (c.block != c.dim && (c.block < 32 || (c.block & (c.block - 1)))) return false;
    const auto on = [](const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    const auto rows = [&](const CacheSide& s) {
        return on(s.base, 16) && s.page % 16 == 0 && s.head % 16 == 0 && s.slot % 16 == 0 && s.page < (1ull << 32) && s.slot < (1u << 26) &&
               s.slot * c.page_size < (1ull << 32) && s.scale_page < (1ull << 32) && s.scale_slot < (1u << 24) && s.scale_slot * c.page_size < (1ull << 32) && s.scale_block < (1u << 24);
    };
    return rows(c.keys) && rows(c.values) && on(a.q, 16) && a.q_token % 8 == 0 && a.q_head % 8 == 0 && on(a.y, 8) && a.y_token % 4 == 0 && a.y_head % 4 == 0;
}

uint64_t part_bytes(const AttentionArgs& a) { return static_cast<uint64_t>(a.tokens) * a.heads * (a.cache.dim + 2) * 4; }

// Tiles of 16 or 32 rows (token, head of a group) by attention_few_kernel, whose sequences have up to 64 on the mean; else tiles of 256 (128 of heads past
// 128) by attention_many_kernel.  The keys are split; how many of the `splits` a sequence has goes by its length, which the device knows.  Measured, in us:
//   16 sequences of 4000 to 8191 keys, 12 rows each: tiles of 16 rows 59, of 32 rows 70; 24 rows: of 16 rows 95, of 32 rows 75; 64 rows: of 32 rows 122, of 256 rows 167;
//     128 rows: of 32 rows 201, of 256 rows 175
//   heads past 128 of a quantized cache, whose tiles of 32 rows want more registers than there are: 8 sequences within a window of 4096 keys, i8 and 4 bits in blocks of 32, 20 rows
//     each: of 16 rows 58 and 80, of 32 rows 112 and 151, of 128 rows 105 and 105; 28 rows twice over (56): of 16 rows 103 and 91, of 128 rows 110 and 108.  Of floats 20 rows: of 16 rows 89, of 32 rows 60
//   parts of few rows, at most 768, 1024, 1536, 2048: 64 sequences of 257 to 8191 keys 120, 117, 119, 123; of 4096 keys 100, 100, 105, 110
//     of 8, 16, 32 steps: one sequence of 3000 keys 14.7, 16.2, 22.5, of 8000 15.4, 16.7, 20.4, of 32000 23.2, 24.2, 23.0; eight of 8000 41, 39, 35;
//     five tokens of eight within a window of 4096 52, 39, 36 (of four parts; 47 of five, which some compute units have two of)
//   of many rows, 128, 256, 512: 509 tokens behind 7681 keys 173, 112, 128; 1000 tokens behind 7190 307, 190, 202.  Tiles that fill the GPU by themselves are
//     not split: 2040 tokens behind 6150 keys 332, and 343
Split split_of(const AttentionArgs& a, uint64_t room) {
    Split f{};
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.group, mean = (rows + a.seqs - 1) / a.seqs;
    f.row_tiles = mean <= 16 ? 1 : mean <= 64 ? (a.cache.dim > 128 && a.cache.code != kCacheFloat ? 1 : 2) : 0;
    const uint64_t of_tile = f.row_tiles ? 16 * f.row_tiles : a.cache.dim > 128 ? 128 : 256;
    const uint64_t step = f.row_tiles && a.cache.code != kCacheInt4 && a.cache.code != kCacheE2M1 ? 32 : 64;
    f.wanted = f.row_tiles ? 1024 : 256;
    f.fewest = f.row_tiles ? 8 : 16;
    f.enough = f.row_tiles ? 32 : 16;
    f.tiles = static_cast<uint32_t>(rows / of_tile + a.seqs);
    const uint64_t busy = a.seqs * ((mean + of_tile - 1) / of_tile) * a.cache.kv_heads;
    uint64_t keys = static_cast<uint64_t>(a.width) * a.cache.page_size;
    const uint64_t behind = a.window + (static_cast<uint64_t>(a.tokens) + a.seqs - 1) / a.seqs;
    if (a.window && behind < keys) keys = behind;
    const uint64_t most = keys / (f.fewest * step);
    // The parts that all tiles want if all sequences are as long as their tables allow, and twice as many of each, for those that are longer than the mean: what is
    // not wanted only looks at the lengths (eight sequences of 8000 keys 34.6 us with twice 1024 parts, 33.5 with these).
    const uint64_t alike = busy * (keys / step) / f.enough, aimed = !f.row_tiles || alike > f.wanted ? f.wanted : alike < 256 ? 256 : alike;
    uint64_t splits = !f.row_tiles && busy >= f.wanted ? 1 : (2 * aimed + busy - 1) / busy;
    if (a.seqs > 1024) splits = 1;  // their lengths are too many for every workgroup to look at
    splits = splits < most ? splits : most;
    splits = splits < kMostSplits ? splits : kMostSplits;
    if (splits > 1 && part_bytes(a) * splits > room) splits = room / part_bytes(a);
    f.splits = splits > 1 ? static_cast<uint32_t>(splits) : 1;
    f.parts = static_cast<float*>(a.workspace);
    f.stats = f.parts + static_cast<uint64_t>(a.tokens) * a.heads * f.splits * a.cache.dim;
    magic_of(a.cache.page_size / 16, &f.page_magic, &f.page_shift);
    f.block_log2 = a.cache.block == a.cache.dim ? 31 : log2_below(a.cache.block);
    return f;
}

bool fits_a_launch(const AttentionArgs& a, const Split& f) {
    return static_cast<uint64_t>(f.tiles) * f.splits * a.cache.kv_heads * (f.row_tiles ? 256 : 512) < kLaunchThreads;
}

}  // namespace

uint64_t attention_workspace_bytes(const AttentionArgs& a) {
    if (a.tokens == 0 || a.heads == 0 || a.seqs == 0 || !tiles_take(a)) return 0;
    const Split f = split_of(a, ~0ull);
    return f.splits == 1 ? 0 : part_bytes(a) * f.splits;
}

hipError_t launch_attention(hipStream_t s, const AttentionArgs& a) {
    if (!tiles_take(a)) return launch_attention_general(s, a);
    const Split f = split_of(a, a.workspace_bytes);
    if (!fits_a_launch(a, f)) return launch_attention_general(s, a);
    const auto tiles = [&]() -> hipError_t {
        switch (a.cache.code) {
#define CQ_CASE_TILES(c) case c: return f.row_tiles ? launch_attention_few_##c(s, a, f) : launch_attention_many_##c(s, a, f);
            CQ_FOR_CODES(CQ_CASE_TILES)
            default: return hipErrorInvalidValue;
        }
    };
    const hipError_t e = tiles();
    return e != hipSuccess || f.splits == 1 ? e : launch_attention_join(s, a, f);
}

}  // namespace cq
