// C ABI of libcubek_attention_hip.so (include/cubek_attention.h): argument checks, the choice of a kernel, launches.
#include "cq_abi_checks.hpp"
#include "cq_attention_internal.hpp"

namespace {

thread_local int g_last_hip_error = 0;

cq_status hip_status(hipError_t e) {
    if (e == hipSuccess) return CQ_OK;
    g_last_hip_error = static_cast<int>(e);
    return CQ_ERR_HIP;
}

// In front of the launches of a call: the launchers read hipGetLastError() after each launch, and an error that earlier HIP calls of the caller left
// would be taken for theirs; a stream of another device than the current one would get kernels of this one.
cq_status ready(cq_stream_t stream) {
    (void)hipGetLastError();
    if (stream == nullptr) return CQ_OK;  // the null stream is the current device's
    int device = -1;
    hipDevice_t of_stream = -1;
    hipError_t e = hipGetDevice(&device);
    if (e == hipSuccess) e = hipStreamGetDevice(stream, &of_stream);
    if (e != hipSuccess) return hip_status(e);
    return static_cast<int>(of_stream) == device ? CQ_OK : CQ_ERR_INVALID_ARGUMENT;
}

constexpr uint64_t kMostTokens = (1ull << 24) - 1;  // a workgroup of 256 threads each in one launch
constexpr uint64_t kMostHeads = 16383;

cq_status read_side(const cq_tensor* t, const cq_tensor* scales, cq::CacheArgs* c, uint32_t lead, uint64_t stored, cq::CacheSide* side) {
    if (!tensor_ok(t)) return CQ_ERR_INVALID_ARGUMENT;
    if (t->rank != 4 || t->elem_size != lead || t->shape[0] != c->pages || t->shape[1] != c->kv_heads || t->shape[2] != c->page_size || t->shape[3] != stored)
        return CQ_ERR_SHAPE_MISMATCH;
    if (stored > 1 && t->strides[3] != 1) return CQ_ERR_NON_CONTIGUOUS;
    if (c->code == cq::kCacheFloat && !aligned(t->ptr, lead)) return CQ_ERR_INVALID_ARGUMENT;
    side->base = static_cast<char*>(t->ptr);
    side->page = stride_of(t, 0) * lead;
    side->head = stride_of(t, 1) * lead;
    side->slot = stride_of(t, 2) * lead;
    if (c->code == cq::kCacheFloat) return scales ? CQ_ERR_INVALID_ARGUMENT : CQ_OK;
    if (!tensor_ok(scales) || !aligned(scales->ptr, dtype_size(c->param_dtype))) return CQ_ERR_INVALID_ARGUMENT;
    if (scales->rank != 4 || scales->elem_size != dtype_size(c->param_dtype) || scales->shape[3] != c->dim / c->block) return CQ_ERR_SHAPE_MISMATCH;
    for (uint32_t d = 0; d < 3; d++)
        if (scales->shape[d] != t->shape[d]) return CQ_ERR_SHAPE_MISMATCH;
    side->scales = static_cast<char*>(scales->ptr);
    side->scale_page = stride_of(scales, 0);
    side->scale_head = stride_of(scales, 1);
    side->scale_slot = stride_of(scales, 2);
    side->scale_block = stride_of(scales, 3);
    return CQ_OK;
}

// How a scheme stores the entries of a cache.
cq_status read_code(const cq_scheme* s, cq::CacheArgs* c) {
    const cq_status st = check_scheme(s);
    if (st != CQ_OK) return st;
    const bool native = s->store == CQ_STORE_NATIVE;
    switch (s->value) {
        case CQ_VALUE_Q8F: case CQ_VALUE_Q8S: c->code = cq::kCacheInt8; break;
        case CQ_VALUE_Q4F: case CQ_VALUE_Q4S: c->code = cq::kCacheInt4; break;
        case CQ_VALUE_E2M1: c->code = native ? cq::kCacheE2M1 : cq::kCacheInt4; break;
        case CQ_VALUE_E2M1_OCP: c->code = cq::kCacheE2M1; break;
        case CQ_VALUE_E4M3: c->code = cq::kCacheE4M3; break;
        case CQ_VALUE_E5M2: c->code = cq::kCacheE5M2; break;
        default: return CQ_ERR_UNSUPPORTED_SCHEME;
    }
    // fields of 8 bits that wrap hold no fp8 values
    if (!native && (s->value == CQ_VALUE_E4M3 || s->value == CQ_VALUE_E5M2)) return CQ_ERR_UNSUPPORTED_SCHEME;
    if (s->level != CQ_LEVEL_BLOCK) return CQ_ERR_UNSUPPORTED_SCHEME;
    for (uint32_t i = 0; i + 1 < s->block_rank; i++)
        if (s->block[i] != 1) return CQ_ERR_UNSUPPORTED_SCHEME;  // a scale belongs to one token
    c->block = s->block[s->block_rank - 1];
    if (c->block % cq_scheme_num_quants(s)) return CQ_ERR_BLOCK_NOT_DIVISIBLE;
    c->param_dtype = s->param == CQ_PARAM_F32 ? CQ_F32 : (s->param == CQ_PARAM_F16 ? CQ_F16 : CQ_BF16);
    c->unrounded = s->value == CQ_VALUE_E2M1_OCP;
    cq_value_range(s->value, &c->lo, &c->hi);
    return CQ_OK;
}

cq_status read_cache(const cq_cache* cache, cq_dtype dtype, cq::CacheArgs* c) {
    if (!cache || !tensor_ok(cache->keys)) return CQ_ERR_INVALID_ARGUMENT;
    uint64_t each = 1;
    uint32_t size = dtype_size(dtype);
    c->code = cq::kCacheFloat;
    if (cache->scheme) {
        const cq_status st = read_code(cache->scheme, c);
        if (st != CQ_OK) return st;
        each = cq_scheme_num_quants(cache->scheme);
        size = cache->scheme->store == CQ_STORE_NATIVE ? 1u : 4u;
    }
    const cq_tensor* const k = cache->keys;
    if (k->rank != 4 || k->shape[1] == 0 || k->shape[2] == 0 || k->shape[3] == 0) return CQ_ERR_SHAPE_MISMATCH;
    if (k->shape[0] > kMostExtent || k->shape[2] > kMostExtent || k->shape[0] * k->shape[2] > kMostExtent || k->shape[1] > kMostHeads ||
        k->shape[3] > CQ_MAX_HEAD_DIM / each)
        return CQ_ERR_TOO_LARGE;
    c->pages = static_cast<uint32_t>(k->shape[0]);
    c->kv_heads = static_cast<uint32_t>(k->shape[1]);
    c->page_size = static_cast<uint32_t>(k->shape[2]);
    c->dim = static_cast<uint32_t>(k->shape[3] * each);
    if (!cache->scheme) c->block = c->dim;
    if (c->dim % c->block) return CQ_ERR_SHAPE_MISMATCH;
    const cq_status st = read_side(k, cache->key_scales, c, size, k->shape[3], &c->keys);
    return st != CQ_OK ? st : read_side(cache->values, cache->value_scales, c, size, k->shape[3], &c->values);
}

// [tokens, heads, dim] typed `dtype`
cq_status read_heads(const cq_tensor* t, cq_dtype dtype, uint64_t tokens, uint64_t heads, uint64_t dim, const char** ptr, uint64_t* token, uint64_t* head) {
    if (!tensor_ok(t) || !aligned(t->ptr, dtype_size(dtype))) return CQ_ERR_INVALID_ARGUMENT;
    if (t->rank != 3 || t->elem_size != dtype_size(dtype) || t->shape[0] != tokens || t->shape[1] != heads || t->shape[2] != dim) return CQ_ERR_SHAPE_MISMATCH;
    if (dim > 1 && t->strides[2] != 1) return CQ_ERR_NON_CONTIGUOUS;
    *ptr = static_cast<const char*>(t->ptr);
    *token = stride_of(t, 0);
    *head = stride_of(t, 1);
    return CQ_OK;
}

// An f32 tensor [n], contiguous.
cq_status read_floats(const cq_tensor* t, uint64_t n, const float** out) {
    const int32_t* bits = nullptr;
    const cq_status st = read_indexes(t, n, &bits);
    *out = reinterpret_cast<const float*>(bits);
    return st;
}

// A tensor whose pages are copied.
cq_status read_pool(const cq_tensor* t, cq::CopyArgs::Pool* p) {
    if (!tensor_ok(t) || t->elem_size == 0) return CQ_ERR_INVALID_ARGUMENT;
    uint64_t elements = 1;
    for (uint32_t d = t->rank - 1; d > 0; d--) {
        if (t->shape[d] > 1 && has_elements(t) && t->strides[d] != elements) return CQ_ERR_NON_CONTIGUOUS;
        if (t->shape[d] > kMostExtent || elements > (1ull << 40) / (t->shape[d] ? t->shape[d] : 1)) return CQ_ERR_TOO_LARGE;
        elements *= t->shape[d];
    }
    if (t->shape[0] > kMostExtent || elements * t->elem_size > (1ull << 36)) return CQ_ERR_TOO_LARGE;
    p->base = static_cast<char*>(t->ptr);
    p->stride = stride_of(t, 0) * t->elem_size;
    p->bytes = elements * t->elem_size;
    p->pages = static_cast<uint32_t>(t->shape[0]);
    p->unit = 1;
    for (uint32_t unit : {16u, 4u})
        if (p->unit == 1 && aligned(p->base, unit) && p->stride % unit == 0 && p->bytes % unit == 0) p->unit = unit;
    return cq::copy_groups(*p) > cq::kMostCopyGroups ? CQ_ERR_TOO_LARGE : CQ_OK;
}

// What a call's kernels are chosen by: cache, queries, table.
cq_status read_shapes(const cq_cache* cache, const cq_tensor* q, const cq_tensor* table, cq_dtype dtype, cq::AttentionArgs* a) {
    if (!valid_dtype(dtype)) return CQ_ERR_INVALID_ARGUMENT;
    cq_status st = read_cache(cache, dtype, &a->cache);
    if (st != CQ_OK) return st;
    if (!tensor_ok(q) || !tensor_ok(table) || !aligned(table->ptr, 4)) return CQ_ERR_INVALID_ARGUMENT;
    if (q->rank != 3 || table->rank != 2 || table->elem_size != 4 || q->shape[1] % a->cache.kv_heads) return CQ_ERR_SHAPE_MISMATCH;
    if (q->shape[0] > kMostTokens || q->shape[1] > kMostHeads || table->shape[0] > kMostTokens || table->shape[1] > kMostExtent ||
        table->shape[1] * a->cache.page_size > kMostExtent)
        return CQ_ERR_TOO_LARGE;
    if (table->shape[1] > 1 && table->strides[1] != 1) return CQ_ERR_NON_CONTIGUOUS;
    a->dtype = dtype;
    a->tokens = static_cast<uint32_t>(q->shape[0]);
    a->heads = static_cast<uint32_t>(q->shape[1]);
    a->group = a->heads / a->cache.kv_heads;
    a->seqs = static_cast<uint32_t>(table->shape[0]);
    a->width = static_cast<uint32_t>(table->shape[1]);
    a->table = static_cast<const int32_t*>(table->ptr);
    a->table_row = stride_of(table, 0);
    return read_heads(q, dtype, a->tokens, a->heads, a->cache.dim, &a->q, &a->q_token, &a->q_head);
}

}  // namespace

extern "C" {

cq_status cq_cache_append(cq_stream_t stream, const cq_cache* cache, const cq_tensor* k, const cq_tensor* v, const cq_tensor* slots, const cq_tensor* q,
                          const cq_tensor* q_out, const cq_tensor* positions, const cq_rotary* rotary, cq_dtype dtype) {
    if (!valid_dtype(dtype)) return CQ_ERR_INVALID_ARGUMENT;
    cq::AppendArgs a{};
    cq_status st = read_cache(cache, dtype, &a.cache);
    if (st != CQ_OK) return st;
    if (!tensor_ok(k) || (q == nullptr) != (q_out == nullptr)) return CQ_ERR_INVALID_ARGUMENT;
    if (k->rank != 3) return CQ_ERR_SHAPE_MISMATCH;
    const uint64_t tokens = k->shape[0];
    if (tokens > kMostTokens) return CQ_ERR_TOO_LARGE;
    if ((st = read_heads(k, dtype, tokens, a.cache.kv_heads, a.cache.dim, &a.k, &a.k_token, &a.k_head)) != CQ_OK) return st;
    if ((st = read_heads(v, dtype, tokens, a.cache.kv_heads, a.cache.dim, &a.v, &a.v_token, &a.v_head)) != CQ_OK) return st;
    if ((st = read_indexes(slots, tokens, &a.slots)) != CQ_OK) return st;
    if (q) {
        if (!tensor_ok(q)) return CQ_ERR_INVALID_ARGUMENT;
        if (q->rank != 3) return CQ_ERR_SHAPE_MISMATCH;
        if (q->shape[1] > kMostHeads) return CQ_ERR_TOO_LARGE;
        const char* out = nullptr;
        if ((st = read_heads(q, dtype, tokens, q->shape[1], a.cache.dim, &a.q, &a.q_token, &a.q_head)) != CQ_OK) return st;
        if ((st = read_heads(q_out, dtype, tokens, q->shape[1], a.cache.dim, &out, &a.out_token, &a.out_head)) != CQ_OK) return st;
        a.q_out = const_cast<char*>(out);
        a.heads = static_cast<uint32_t>(q->shape[1]);
    }
    if (rotary) {
        if (!tensor_ok(rotary->frequencies) || rotary->interleaved > 1 || !positions) return CQ_ERR_INVALID_ARGUMENT;
        if (rotary->frequencies->rank != 1 || rotary->frequencies->shape[0] > a.cache.dim / 2) return CQ_ERR_SHAPE_MISMATCH;
        if ((st = read_floats(rotary->frequencies, rotary->frequencies->shape[0], &a.frequencies)) != CQ_OK) return st;
        if ((st = read_indexes(positions, tokens, &a.positions)) != CQ_OK) return st;
        a.pairs = static_cast<uint32_t>(rotary->frequencies->shape[0]);
        a.interleaved = rotary->interleaved;
        a.magnitude = rotary->magnitude;
    } else if (positions) {
        return CQ_ERR_INVALID_ARGUMENT;
    }
    if (tokens == 0) return CQ_OK;
    a.tokens = static_cast<uint32_t>(tokens);
    a.dtype = dtype;
    if ((st = ready(stream)) != CQ_OK) return st;
    return hip_status(cq::launch_append(stream, a));
}

size_t cq_attention_workspace_bytes(const cq_cache* cache, const cq_tensor* q, const cq_tensor* table, cq_dtype dtype) {
    cq::AttentionArgs a{};
    return read_shapes(cache, q, table, dtype, &a) == CQ_OK ? cq::attention_workspace_bytes(a) : 0;
}

cq_status cq_attention(cq_stream_t stream, const cq_cache* cache, const cq_tensor* q, const cq_tensor* y, const cq_tensor* table, const cq_tensor* offsets,
                       const cq_tensor* lengths, const cq_scores* scores, cq_dtype dtype, void* workspace, size_t workspace_bytes) {
    cq::AttentionArgs a{};
    cq_status st = read_shapes(cache, q, table, dtype, &a);
    if (st != CQ_OK) return st;
    const char* out = nullptr;
    if ((st = read_heads(y, dtype, a.tokens, a.heads, a.cache.dim, &out, &a.y_token, &a.y_head)) != CQ_OK) return st;
    a.y = const_cast<char*>(out);
    if ((st = read_indexes(offsets, a.seqs + 1ull, &a.offsets)) != CQ_OK) return st;
    if ((st = read_indexes(lengths, a.seqs, &a.lengths)) != CQ_OK) return st;
    if (!scores || scores->reserved != 0 || !(scores->cap >= 0.0f && scores->cap < __builtin_inff())) return CQ_ERR_INVALID_ARGUMENT;
    a.scale = scores->scale;
    a.cap = scores->cap;
    a.window = scores->window;
    if (scores->slopes && (st = read_floats(scores->slopes, a.heads, &a.slopes)) != CQ_OK) return st;
    if (scores->prefix && (st = read_indexes(scores->prefix, a.seqs, &a.prefix)) != CQ_OK) return st;
    if (a.tokens == 0 || a.heads == 0 || a.seqs == 0) return CQ_OK;
    a.workspace = aligned(workspace, 16) ? workspace : nullptr;
    a.workspace_bytes = a.workspace ? workspace_bytes : 0;
    if ((st = ready(stream)) != CQ_OK) return st;
    return hip_status(cq::launch_attention(stream, a));
}

cq_status cq_cache_copy(cq_stream_t stream, const cq_tensor* tensors, uint32_t count, const cq_tensor* pairs) {
    if ((!tensors && count) || !tensor_ok(pairs) || !aligned(pairs->ptr, 4)) return CQ_ERR_INVALID_ARGUMENT;
    if (pairs->rank != 2 || pairs->elem_size != 4 || pairs->shape[1] != 2) return CQ_ERR_SHAPE_MISMATCH;
    if (!is_contiguous(pairs)) return CQ_ERR_NON_CONTIGUOUS;
    if (pairs->shape[0] > kMostTokens) return CQ_ERR_TOO_LARGE;
    cq::CopyArgs::Pool pool;
    for (uint32_t i = 0; i < count; i++) {  // all of them before the first launch
        const cq_status st = read_pool(tensors + i, &pool);
        if (st != CQ_OK) return st;
    }
    if (pairs->shape[0] == 0 || count == 0) return CQ_OK;
    cq_status st = ready(stream);
    for (uint32_t first = 0; first < count && st == CQ_OK; first += cq::kCopyTensors) {
        cq::CopyArgs a{};
        const uint32_t n = count - first < cq::kCopyTensors ? count - first : cq::kCopyTensors;
        for (uint32_t i = 0; i < n; i++) (void)read_pool(tensors + first + i, &a.pools[i]);
        a.pairs = static_cast<const int32_t*>(pairs->ptr);
        a.count = static_cast<uint32_t>(pairs->shape[0]);
        st = hip_status(cq::launch_copy(stream, a, n));
    }
    return st;
}

int cq_attention_last_hip_error(void) { return g_last_hip_error; }

}  // extern "C"
