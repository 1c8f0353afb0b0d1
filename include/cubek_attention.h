/* cubek_attention.h — C ABI of libcubek_attention_hip.so: a cache of keys and values in pages, quantized or not, and what a model does
 * around it on MI355X (gfx950): appending new tokens, attention over the pages, copying pages.
 *
 * It stands beside cubek_quant.h, whose tensors, schemes and status codes it uses: what cq_cache_append stores are the codes and scales of
 * cq_quantize_dynamic, and cq_dequantize reads them.  The reference has attention in a crate of its own (crates/cubek-attention), over
 * contiguous floats.
 *
 * As everywhere in this library: device pointers, strides in elements, the caller owns every buffer, calls only enqueue kernels on
 * the caller's stream (no allocation, synchronisation or memset: they can be captured into a HIP graph) and validate before
 * they launch; the current device is the stream's.  Results do not depend on anything but the arguments: no atomics, no order that
 * changes from call to call. */
#ifndef CUBEK_ATTENTION_H
#define CUBEK_ATTENTION_H

#include "cubek_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CQ_MAX_HEAD_DIM 512

/* Keys and values of one layer, [pages, kv_heads, page_size, dim / num_quants]: a slot is page * page_size + place in the page, and any strides
 * but the last dimension's (contiguous) give other orders, [pages, page_size, kv_heads, dim] for one.
 *   scheme : NULL for floats typed like the calls' dtype (no scales); else 8- or 4-bit values in blocks along the last dimension: i8, e4m3,
 *            e5m2 and e2m1 of the native store, the two's-complement fields of the U32 store of Q8*, Q4*, E2M1 and E2M1_OCP (codes and strides
 *            of the U32 store in words).  Else CQ_ERR_UNSUPPORTED_SCHEME.
 *   key_scales, value_scales : [pages, kv_heads, page_size, dim / block] typed scheme->param, any strides.  Scales of 16 bits are read as the aligned
 *            four bytes around them: up to two bytes in front of such a tensor and behind it are read, and not used.
 * The entries of a cache are scale * code; cq_attention says what becomes of them. */
typedef struct cq_cache {
    const cq_tensor* keys;
    const cq_tensor* key_scales;
    const cq_tensor* values;
    const cq_tensor* value_scales;
    const cq_scheme* scheme;
} cq_cache;

/* Rotary positions: of each head the first 2 * (number of frequencies) entries are turned in pairs (a, b) by the angle position * frequency,
 *   a' = a c - b w, b' = b c + a w, with c = magnitude cos(angle) and w = magnitude sin(angle),
 * in 64 bits, rounded to f32 and from there to `dtype`; the other entries stay.  Longer contexts are a matter of the frequencies and of the magnitude.
 *   frequencies : f32 [n], contiguous, 2 n <= dim.  Angles of 2^31 and more have no meaning.
 *   interleaved : 0: entry i pairs with entry i + n; 1: entry 2 i with entry 2 i + 1 */
typedef struct cq_rotary {
    const cq_tensor* frequencies;
    float magnitude;
    uint32_t interleaved;
} cq_rotary;

/* New tokens into their slots: keys turned by their positions (and so rounded to `dtype`) and quantized, values quantized; queries turned.
 *   k, v  : [tokens, kv_heads, dim] typed `dtype`, the last dimension contiguous (views of a common projection for one)
 *   slots : i32 [tokens], contiguous.  A token whose slot lies outside of the cache (-1 for one) is not stored.  Two tokens in one slot: what it
 *           holds afterwards may be parts of both.
 *   q, q_out : NULL, or [tokens, heads, dim], last dimensions contiguous; q_out may be q itself, with the same strides
 *   positions : i32 [tokens], contiguous; NULL where rotary is NULL: nothing is turned */
cq_status cq_cache_append(cq_stream_t stream, const cq_cache* cache, const cq_tensor* k, const cq_tensor* v, const cq_tensor* slots,
                          const cq_tensor* q, const cq_tensor* q_out, const cq_tensor* positions, const cq_rotary* rotary, cq_dtype dtype);

/* What stands between queries and weights, in f32:
 *   t = scale * (q . k);  t = cap * tanh(t / cap) where cap > 0;  t -= slopes[head] * |position - key|
 * The query at position p sees the keys 0 <= j < length with j <= p or j < prefix, and, where window > 0, p - j < window.
 *   slopes : NULL or f32 [heads], contiguous
 *   prefix : NULL or i32 [sequences], contiguous, each taken as the nearest number between 0 and the sequence's length
 * cap is 0 (none) or a positive number, of which those past 10^38 count as that.  Every field not used is 0. */
typedef struct cq_scores {
    float scale;
    float cap;
    uint32_t window;
    uint32_t reserved;
    const cq_tensor* slopes;
    const cq_tensor* prefix;
} cq_scores;

/* y = softmax(scores of q) V for the new tokens of all sequences, whose keys and values are in the cache already.
 *   q, y    : [tokens, heads, dim] typed `dtype`, last dimensions contiguous, not in the same memory; heads is a multiple of kv_heads, and heads
 *             h * group ... h * group + group - 1 share head h of the cache
 *   table   : i32 [sequences, most pages of one], rows contiguous: page j / page_size of a sequence holds its key j.  Entries behind a
 *             sequence's length are not read; one outside of the cache is taken as the nearest inside.
 *   offsets : i32 [sequences + 1], contiguous: tokens offsets[s] <= t < offsets[s + 1] are the newest of sequence s, in order.  Values outside
 *             are taken as the nearest inside; tokens of no sequence are left unwritten.
 *   lengths : i32 [sequences], contiguous: keys of a sequence with its new ones: its last token is at position lengths[s] - 1.  Taken as the
 *             nearest number between 0 and what the table's row holds.
 * A token that sees no key gets zeros.  Entries of the cache that a token does not see do not enter its result, whatever they hold; what it sees of infinities and NaN does, and
 * so do those of its query.
 * Scores, statistics and sums are f32, and for f32 queries so is everything else.  For 16-bit ones, on their way into matrix instructions, are rounded
 *   weights, with a value's scale : to 11 bits (over a cache of bf16 floats to 16; to 8 for prompts)
 *   queries of bf16 over a quantized cache : entries below 2^-14 of the largest of their head, to 2^-25 of it
 *   entries of a quantized cache, for prompts of bf16 : keys to 11 bits, values twice, by their scale and by the product
 * and what is 2^-18 of a token's largest weight, or 2^-12 of a step between two codes, is lost.  Where scales of a sequence lie further apart than 2^12 (zeros aside), tokens that
 * would lose more to others' scales than 2^-11 of the largest of 32 neighbouring entries of their result are taken once more, one by one, in f32: many times slower.
 *   workspace : optional device scratch of cq_attention_workspace_bytes() bytes, 16-byte aligned; lets few tokens over long
 *             sequences spread over the GPU.  Without it they are right, and slower.  It holds nothing between calls: calls whose kernels
 *             do not run at the same time may share it. */
cq_status cq_attention(cq_stream_t stream, const cq_cache* cache, const cq_tensor* q, const cq_tensor* y, const cq_tensor* table,
                       const cq_tensor* offsets, const cq_tensor* lengths, const cq_scores* scores, cq_dtype dtype, void* workspace,
                       size_t workspace_bytes);
size_t cq_attention_workspace_bytes(const cq_cache* cache, const cq_tensor* q, const cq_tensor* table, cq_dtype dtype);

/* Pages copied within each of `count` tensors, whose first dimension is that of the pages and whose others are contiguous: the bytes of page
 * pairs[i, 0] to page pairs[i, 1], for a sequence that forks (a source as often as one likes) or a pool that is compacted.
 *   pairs : i32 [n, 2] in device memory, contiguous.  A pair with a page outside of a tensor copies nothing in it.  A page that is the destination of
 *           two pairs, or source of one and destination of another, may hold parts of both afterwards.
 * The tensors are handed over in launches of up to 32.  A page has 64 GiB at most, where its bytes, address or stride are no multiples of four less than 16 GiB (64 GiB less
 * 4 KiB of fours). */
cq_status cq_cache_copy(cq_stream_t stream, const cq_tensor* tensors, uint32_t count, const cq_tensor* pairs);

/* hipError_t of the most recent failed HIP call of this library on the calling thread (0 if none). */
int cq_attention_last_hip_error(void);

#ifdef __cplusplus
}
#endif
#endif /* CUBEK_ATTENTION_H */
