// What the objects of libcubek_attention_hip.so share: the arguments of a launch, sequences and pages on the device.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/cubek_attention.h"

namespace cq {

// Threads of a launch along one dimension.
constexpr uint64_t kLaunchThreads = 1ull << 32;

// How an entry of the cache is stored.
enum CacheCode : uint32_t { kCacheInt8 = 0, kCacheInt4 = 1, kCacheE4M3 = 2, kCacheE5M2 = 3, kCacheE2M1 = 4, kCacheFloat = 5 };

// Keys, or values: row `place` of head h of page p at base + p * page + h * head + place * slot, in bytes; its scales in elements.
struct CacheSide {
    char* base;
    uint64_t page, head, slot;
    char* scales;
    uint64_t scale_page, scale_head, scale_slot, scale_block;
};

struct CacheArgs {
    CacheSide keys, values;
    uint32_t code;         // CacheCode
    uint32_t param_dtype;  // of the scales
    uint32_t dim, block;   // entries of a row; entries of a scale
    uint32_t pages, page_size, kv_heads;
    float lo, hi;           // range of the codes
    uint32_t unrounded;     // CQ_VALUE_E2M1_OCP
};

struct AppendArgs {
    CacheArgs cache;
    const char *k, *v, *q;
    char* q_out;
    const int32_t *slots, *positions;
    const float* frequencies;  // or NULL
    uint64_t k_token, k_head, v_token, v_head, q_token, q_head, out_token, out_head;  // strides in elements
    uint32_t tokens, heads;    // heads 0 without queries
    uint32_t pairs, interleaved;
    float magnitude;
    uint32_t rows;  // heads of q, k and v of one workgroup
    int dtype;
};
hipError_t launch_append(hipStream_t s, const AppendArgs& a);

struct AttentionArgs {
    CacheArgs cache;
    const char* q;
    char* y;
    uint64_t q_token, q_head, y_token, y_head;  // strides in elements
    const int32_t *table, *offsets, *lengths, *prefix;
    const float* slopes;
    uint64_t table_row;
    uint32_t tokens, seqs, heads, group, width;  // width: pages of a row of the table
    float scale, cap;
    uint32_t window;
    int dtype;
    void* workspace;
    uint64_t workspace_bytes;
};
uint64_t attention_workspace_bytes(const AttentionArgs& a);
hipError_t launch_attention(hipStream_t s, const AttentionArgs& a);
hipError_t launch_attention_general(hipStream_t s, const AttentionArgs& a);

constexpr uint32_t kMostSplits = 64;  // a lane each in attention_join_kernel

// How rows and the keys they see are shared out between workgroups.
struct Split {
    uint32_t tiles, row_tiles;  // workgroups for rows, of one head and one split; tiles of 16 rows of one (attention_few_kernel)
    uint32_t splits;            // of the keys, at most
    uint32_t waves;             // of a workgroup of attention_few_kernel
    uint32_t wanted, fewest, enough;  // parts of all tiles together, at most; steps of the smallest part, and of one that is as good as a larger one
    uint32_t page_magic, page_shift, block_log2;  // division by the tiles of 16 keys of a page; log2 of a scale's entries
    float *parts, *stats;  // splits > 1: [token][head][split][dim], each over its own sum; [token][head][split]{largest score, sum}
};
#define CQ_FOR_CODES(x) x(0) x(1) x(2) x(3) x(4) x(5)
#define CQ_DECLARE_TILES(c)                                                                            \
    hipError_t launch_attention_few_##c(hipStream_t s, const AttentionArgs& a, const Split& split); \
    hipError_t launch_attention_many_##c(hipStream_t s, const AttentionArgs& a, const Split& split);
CQ_FOR_CODES(CQ_DECLARE_TILES)
hipError_t launch_attention_join(hipStream_t s, const AttentionArgs& a, const Split& split);

constexpr uint32_t kCopyTensors = 32;
constexpr uint64_t kCopyAccesses = 1024;                          // of a workgroup
constexpr uint64_t kMostCopyGroups = kLaunchThreads / 256 - 1;  // workgroups of a page
struct CopyArgs {
    struct Pool {
        char* base;
        uint64_t stride, bytes;  // of a page
        uint32_t pages, unit;    // unit: bytes of an access
    } pools[kCopyTensors];
    const int32_t* pairs;
    uint32_t count;  // pairs
    uint32_t chunks;  // workgroups of a page
};
inline uint64_t copy_groups(const CopyArgs::Pool& p) { return (p.bytes + kCopyAccesses * p.unit - 1) / (kCopyAccesses * p.unit); }
hipError_t launch_copy(hipStream_t s, const CopyArgs& a, uint32_t tensors);

#if defined(__HIPCC__)

// The last index s < n with begin(s) <= at, 0 where there is none, by 64 questions at once; begin does not fall.  All lanes of the wave take part.
template <class Begin>
__device__ __forceinline__ uint32_t last_at_or_below(uint32_t n, uint64_t at, Begin begin) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t low = 0;
    while (n > 1) {
        const uint32_t step = (n + 63u) / 64u, i = lane * step;
        const uint64_t below = __builtin_amdgcn_ballot_w64(i < n && begin(low + i) <= at);
        const uint32_t last = below ? 63u - static_cast<uint32_t>(__builtin_clzll(below)) : 0u;
        low += last * step;
        n = min(step, n - last * step);
    }
    return low;
}

// A sequence's part of the tokens and the keys of it.
struct Sequence {
    uint32_t index, first, last;  // tokens first <= t < last
    int32_t length;               // keys
    int32_t position;             // of token `first`; negative where there are fewer keys than tokens
    int32_t prefix;               // keys before this one are seen by all
};
__device__ __forceinline__ Sequence sequence_of(const AttentionArgs& a, uint32_t s) {
    Sequence q;
    q.index = s;
    q.first = static_cast<uint32_t>(min(max(a.offsets[s], 0), static_cast<int32_t>(a.tokens)));
    q.last = static_cast<uint32_t>(min(max(a.offsets[s + 1], static_cast<int32_t>(q.first)), static_cast<int32_t>(a.tokens)));
    const int64_t most = static_cast<int64_t>(a.width) * a.cache.page_size;
    const int64_t length = a.lengths[s];
    q.length = a.cache.pages ? static_cast<int32_t>(min(max(length, static_cast<int64_t>(0)), most)) : 0;
    q.position = q.length - static_cast<int32_t>(q.last - q.first);
    q.prefix = a.prefix ? min(max(a.prefix[s], 0), q.length) : 0;  // (the lowest number less one would be the highest)
    return q;
}

// The keys that the query at position p sees, from low to high (high < low: none).
struct Seen {
    int32_t low, high;
};
__device__ __forceinline__ Seen seen_from(const AttentionArgs& a, const Sequence& s, int32_t p) {
    Seen r;
    r.high = max(p, s.prefix - 1);  // p < length
    r.low = a.window && p >= 0 && static_cast<uint32_t>(p) >= a.window ? p - static_cast<int32_t>(a.window) + 1 : 0;
    return r;
}

__device__ __forceinline__ uint32_t page_of(const AttentionArgs& a, const Sequence& s, uint32_t nth) {
    const int32_t page = a.table[s.index * a.table_row + nth];
    return min(static_cast<uint32_t>(max(page, 0)), a.cache.pages - 1u);
}

#endif

}  // namespace cq
