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
// entries or for a head, rows on 16-byte boundaries.
bool tiles_take(const AttentionArgs& a) {
    const CacheArgs& c = a.cache;
    if (a.dtype == CQ_F32 || c.dim % 32 || c.dim > 256 || c.page_size % 16) return false;
    if (c.block != c.dim && (c.block < 32 || (c.block & (c.block - 1)))) return false;
    const auto on = [](const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    const auto rows = [&](const CacheSide& s) { return on(s.base, 16) && s.page % 16 == 0 && s.head % 16 == 0 && s.slot % 16 == 0 && s.slot < (1u << 26); };
    return rows(c.keys) && rows(c.values) && on(a.q, 16) && a.q_token % 8 == 0 && a.q_head % 8 == 0 && on(a.y, 8) && a.y_token % 4 == 0 && a.y_head % 4 == 0;
}

// Sequences of up to 32 rows on the mean go by tiles of 16 or 32.
bool few_rows(const AttentionArgs& a) { return static_cast<uint64_t>(a.tokens) * a.group <= 64ull * a.seqs; }

constexpr uint32_t kMostSplits = 64;  // a lane each in attention_join_kernel

// Enough splits that about four workgroups come to a compute unit, none of less than 512 keys.
FewSplit few_split(const AttentionArgs& a, uint64_t room) {
    FewSplit f{};
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.group, mean = (rows + a.seqs - 1) / a.seqs;
    f.row_tiles = mean <= 16 ? 1 : 2;
    f.tiles = static_cast<uint32_t>(rows / (16 * f.row_tiles) + a.seqs);
    const uint64_t busy = a.seqs * ((mean + 16 * f.row_tiles - 1) / (16 * f.row_tiles)) * a.cache.kv_heads;
    const uint64_t keys = static_cast<uint64_t>(a.width) * a.cache.page_size;
    uint64_t splits = (1024 + busy - 1) / busy, most = keys / 512;
    splits = splits < most ? splits : most;
    splits = splits < kMostSplits ? splits : kMostSplits;
    const uint64_t each = static_cast<uint64_t>(a.tokens) * a.heads * (a.cache.dim + 2) * 4;
    if (splits > 1 && each * splits > room) splits = room / each;
    f.splits = splits > 1 ? static_cast<uint32_t>(splits) : 1;
    f.parts = static_cast<float*>(a.workspace);
    f.stats = f.parts + static_cast<uint64_t>(a.tokens) * a.heads * f.splits * a.cache.dim;
    magic_of(a.cache.page_size / 16, &f.page_magic, &f.page_shift);
    f.block_log2 = log2_below(a.cache.block);
    return f;
}

bool fits_a_launch(const FewSplit& f) { return static_cast<uint64_t>(f.tiles) * f.splits * 256 < kLaunchThreads; }

}  // namespace

uint64_t attention_workspace_bytes(const AttentionArgs& a) {
    if (a.tokens == 0 || a.heads == 0 || a.seqs == 0 || !tiles_take(a) || !few_rows(a)) return 0;
    const FewSplit f = few_split(a, ~0ull);
    return f.splits == 1 ? 0 : static_cast<uint64_t>(a.tokens) * a.heads * f.splits * (a.cache.dim + 2) * 4;
}

hipError_t launch_attention(hipStream_t s, const AttentionArgs& a) {
    if (!tiles_take(a) || !few_rows(a)) return launch_attention_general(s, a);
    const FewSplit f = few_split(a, a.workspace_bytes);
    if (!fits_a_launch(f)) return launch_attention_general(s, a);
    const auto few = [&]() -> hipError_t {
        switch (a.cache.code) {
#define CQ_CASE_FEW(c) case c: return launch_attention_few_##c(s, a, f);
            CQ_FOR_CODES(CQ_CASE_FEW)
            default: return hipErrorInvalidValue;
        }
    };
    const hipError_t e = few();
    return e != hipSuccess || f.splits == 1 ? e : launch_attention_join(s, a, f);
}

}  // namespace cq
