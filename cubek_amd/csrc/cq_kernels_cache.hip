// New tokens into a cache of pages.  An object per float type (CQ_TU_FLOAT).
//
// append_kernel: a workgroup takes some heads of one token, queries, keys and values alike: a lane asks for eight entries and their partners; meanwhile
// the first lanes work out cosine and sine of the token's angles, once for these heads; then each lane turns its entries and stores them, or quantizes them
// as the flat quantize kernels do, the maximum of a block by a butterfly over the lanes that hold it.  (Rows whose strides do not allow that go through
// LDS, an entry or a block a lane.)
//
// Angles and turning are in 64 bits: position * frequency is then exact to 2^-53 of itself (262144 positions: 2^-35), the turned entry is the
// exact one but for the one rounding to F, and so codes do not depend on how cosines are computed.
//
// Bound by a launch for single tokens (5.1-5.6 us), by vector instructions and the waits of short workgroups for prompts: 4093 tokens, 48 heads of 128 of bf16
// to e4m3, 92 MB, take 30 us (3.1 TB/s; a copy would 18), vector units busy 59 % with conversions to 64 bits and back, two FMAs an entry and the quantization.
#include <hip/hip_runtime.h>

#include "cq_attention_internal.hpp"
#include "cq_device.hpp"

namespace cq {
namespace {

// Cosine and sine of an angle: the angle less the nearest multiple n of pi / 2 (in two parts, the second what the first leaves of pi / 2), their
// Taylor polynomials on the rest (|r| <= pi / 4: the first term left out is below 2^-60), and the quarter turn that n stands for.
__device__ __forceinline__ void cos_sin(double angle, double* c, double* w) {
    const double n = __builtin_rint(angle * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489655800, angle);
    r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
    const double x = r * r;
    double s = 1.0 / 355687428096000.0, k = -1.0 / 6402373705728000.0;  // 1/17!, -1/18!
    s = __builtin_fma(s, x, -1.0 / 1307674368000.0);
    s = __builtin_fma(s, x, 1.0 / 6227020800.0);
    s = __builtin_fma(s, x, -1.0 / 39916800.0);
    s = __builtin_fma(s, x, 1.0 / 362880.0);
    s = __builtin_fma(s, x, -1.0 / 5040.0);
    s = __builtin_fma(s, x, 1.0 / 120.0);
    s = __builtin_fma(s, x, -1.0 / 6.0);
    s = __builtin_fma(s * x, r, r);
    k = __builtin_fma(k, x, 1.0 / 20922789888000.0);
    k = __builtin_fma(k, x, -1.0 / 87178291200.0);
    k = __builtin_fma(k, x, 1.0 / 479001600.0);
    k = __builtin_fma(k, x, -1.0 / 3628800.0);
    k = __builtin_fma(k, x, 1.0 / 40320.0);
    k = __builtin_fma(k, x, -1.0 / 720.0);
    k = __builtin_fma(k, x, 1.0 / 24.0);
    k = __builtin_fma(k, x, -0.5);
    k = __builtin_fma(k, x, 1.0);
    const uint32_t quarter = static_cast<uint32_t>(static_cast<int64_t>(n)) & 3u;
    const double even = quarter & 1u ? s : k, odd = quarter & 1u ? k : s;
    *c = quarter == 1u || quarter == 2u ? -even : even;
    *w = quarter & 2u ? -odd : odd;
}

// A 64-bit number to F, by way of f32: rounded as once but within 2^-25 of a tie of 16 bits.
template <class F>
__device__ __forceinline__ float narrowed(double v) {
    return F::round(static_cast<float>(v));
}

constexpr uint32_t kEach = 8;             // entries of a lane
constexpr uint32_t kWorkEntries = 256 * kEach;  // of a workgroup: with two lots a thread, 33 us where it is 30

// Eight entries, and eight to a 16-byte boundary.
template <class F>
__device__ __forceinline__ void unpack_each(const u32x4* w, float* v) {
#pragma unroll
    for (uint32_t c = 0; c < kEach / F::kPerChunk; c++) F::unpack(w[c], v + c * F::kPerChunk);
}
template <class F>
__device__ __forceinline__ void store_each(char* p, uint64_t i, const float* v) {
#pragma unroll
    for (uint32_t c = 0; c < kEach / F::kPerChunk; c++) reinterpret_cast<u32x4*>(p + i * F::kBytes)[c] = F::pack(v + c * F::kPerChunk);
}

// kEnc, kBits: encoding of the codes; kBits 0: floats.  kWide: rows on 16-byte boundaries, of whole lanes, blocks of 8, 16, 32 ... entries; else a lane
// takes one entry, or one block.
template <class F, int kEnc, int kBits, bool kWide>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    extern __shared__ char lds[];
    double2* const turn = reinterpret_cast<double2*>(lds);
    char* const rows = lds + a.pairs * sizeof(double2);  // not kWide
    const CacheArgs& c = a.cache;
    const uint32_t token = blockIdx.x, all = a.heads + 2u * c.kv_heads, row0 = blockIdx.y * a.rows, count = min(a.rows, all - row0), dim = c.dim;
    const int64_t slot = a.slots[token];
    const bool kept = slot >= 0 && slot < static_cast<int64_t>(c.pages) * c.page_size;
    if (row0 >= a.heads && !kept) return;

    const auto source = [&](uint32_t row, uint64_t* at) {
        if (row < a.heads) {
            *at = token * a.q_token + row * a.q_head;
            return a.q;
        }
        row -= a.heads;
        *at = row < c.kv_heads ? token * a.k_token + row * a.k_head : token * a.v_token + (row - c.kv_heads) * a.v_head;
        return row < c.kv_heads ? a.k : a.v;
    };
    constexpr uint32_t kStep = kWide ? kEach : 1u, kChunks = kEach / F::kPerChunk;
    const uint32_t of_row = dim / kStep, tasks = count * of_row;
    // an entry's partner, and whether it turns at all
    const auto partner_of = [&](uint32_t d) { return a.interleaved ? d ^ 1u : (d < a.pairs ? d + a.pairs : d - a.pairs); };
    u32x4 own[kChunks], partner[kChunks];
    if constexpr (kWide) {
        const uint32_t t = min(threadIdx.x, tasks - 1u), d = t % of_row * kEach;
        uint64_t at;
        const char* const from = source(row0 + t / of_row, &at);
#pragma unroll
        for (uint32_t e = 0; e < kChunks; e++) {
            own[e] = reinterpret_cast<const u32x4*>(from + (at + d) * F::kBytes)[e];
            partner[e] = reinterpret_cast<const u32x4*>(from + (at + (a.interleaved || d >= 2u * a.pairs ? d : partner_of(d))) * F::kBytes)[e];
        }
    } else {
        for (uint32_t t = threadIdx.x; t < tasks; t += 256) {
            uint64_t at;
            const char* const from = source(row0 + t / dim, &at);
            F::store(rows, t, F::load(from, at + t % dim));
        }
    }
    // A lane's eight entries begin with pair kPairs * n: pair k of them stands at n + k * stride, so that neighbouring lanes read neighbours.
    const uint32_t pairs_log2 = kWide ? (a.interleaved ? 2u : 3u) : 0u, stride = a.pairs >> pairs_log2;
    if (row0 < a.heads + c.kv_heads)
        for (uint32_t p = threadIdx.x; p < a.pairs; p += 256) {
            double cosine, sine;
            cos_sin(static_cast<double>(a.positions[token]) * static_cast<double>(a.frequencies[p]), &cosine, &sine);
            turn[(p & ((1u << pairs_log2) - 1u)) * stride + (p >> pairs_log2)] = double2{cosine * a.magnitude, sine * a.magnitude};
        }
    // all of the rows are read before any of them is written: q_out may be q
    if constexpr (kWide) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();

    const auto turned = [&](double2 z, float own, float partner, bool first) {
        const double x = own, p = partner;
        return narrowed<F>(__builtin_fma(first ? -p : p, z.y, x * z.x));
    };
    const auto entry = [&](uint32_t row, uint32_t d, bool turns) {
        const float own = F::load(rows, row * dim + d);
        if (!turns || d >= 2u * a.pairs) return own;
        const bool first = a.interleaved ? d % 2u == 0 : d < a.pairs;
        return turned(turn[a.interleaved ? d / 2u : (first ? d : d - a.pairs)], own, F::load(rows, row * dim + partner_of(d)), first);
    };

    const uint32_t page = kept ? static_cast<uint32_t>(slot) / c.page_size : 0u, place = kept ? static_cast<uint32_t>(slot) % c.page_size : 0u;
    QuantParams range;
    range.lo = c.lo, range.hi = c.hi, range.width = c.hi - c.lo, range.unrounded = c.unrounded;
    const uint32_t group_log2 = kBits && kWide ? 31u - static_cast<uint32_t>(__builtin_clz(c.block / kEach)) : 0u;
    const uint32_t block = kBits && !kWide ? c.block : kStep, of_row2 = dim / block, tasks2 = count * of_row2;
    // whole waves, so that butterflies have all their lanes; past the last the last again
    const auto task = [&](uint32_t t0) {
        const uint32_t t = min(t0, tasks2 - 1u), row = t / of_row2, d0 = t % of_row2 * block, from = row0 + row;
        const bool is_query = from < a.heads, is_key = !is_query && from < a.heads + c.kv_heads;
        const uint32_t head = is_query ? from : (from - a.heads) % c.kv_heads;
        const CacheSide& side = is_key ? c.keys : c.values;
        const uint64_t scale_at = page * side.scale_page + head * side.scale_head + place * side.scale_slot;
        char* const to = side.base + page * side.page + head * side.head + place * side.slot;
        if constexpr (kWide) {
            float v[kEach];
            unpack_each<F>(own, v);
            if ((is_query || is_key) && d0 < 2u * a.pairs) {
                if (a.interleaved) {
#pragma unroll
                    for (uint32_t e = 0; e < kEach; e += 2) {
                        const float x = v[e], y = v[e + 1];
                        v[e] = turned(turn[d0 / kEach + e / 2u * stride], x, y, true);
                        v[e + 1] = turned(turn[d0 / kEach + e / 2u * stride], y, x, false);
                    }
                } else {
                    const bool first = d0 < a.pairs;
                    float p[kEach];
                    unpack_each<F>(partner, p);
#pragma unroll
                    for (uint32_t e = 0; e < kEach; e++) v[e] = turned(turn[(first ? d0 : d0 - a.pairs) / kEach + e * stride], v[e], p[e], first);
                }
            }
            if constexpr (kBits == 0) {
                if (t0 >= tasks2) return;
                if (is_query)
                    store_each<F>(a.q_out, token * a.out_token + from * a.out_head + d0, v);
                else if (kept)
                    store_each<F>(to, d0, v);
            } else {
                float most = 0.0f;
#pragma unroll
                for (uint32_t e = 0; e < kEach; e++) most = fmaxf(most, fabsf(v[e]));
                most = group_max_rt(most, group_log2);
                if (t0 >= tasks2) return;
                if (is_query) {
                    store_each<F>(a.q_out, token * a.out_token + from * a.out_head + d0, v);
                } else if (kept) {
                    const float scale = F::round(scale_from_absmax(most, range.width)), divisor = F::round(round_to_dtype(c.param_dtype, scale));
                    float codes[kEach];
                    quantize_codes<F, kEach, kEnc>(v, divisor, divisor_is_tame(divisor), range.lo, range.hi, range.unrounded, codes);
                    uint32_t w[2];
                    if constexpr (kEnc == kEncInt)
                        pack_chunk_neg<kBits, kEach, false>(codes, w);
                    else
                        encode_chunk<kEnc, kEach>(codes, w);
                    if constexpr (kBits == 8)
                        *reinterpret_cast<u32x2*>(to + d0) = u32x2{w[0], w[1]};
                    else
                        *reinterpret_cast<uint32_t*>(to + d0 / 2u) = w[0];
                    if (d0 % c.block == 0) store_dtype(c.param_dtype, side.scales, scale_at + d0 / c.block * side.scale_block, scale);
                }
            }
        } else {
            if (t0 >= tasks2) return;
            if (is_query) {
                for (uint32_t d = d0; d < d0 + block; d++) F::store(a.q_out, token * a.out_token + from * a.out_head + d, entry(row, d, true));
            } else if (kept) {
                if constexpr (kBits == 0) {
                    F::store(to, d0, entry(row, d0, is_key));
                } else {
                    float most = 0.0f;
                    for (uint32_t d = d0; d < d0 + block; d++) most = fmaxf(most, fabsf(entry(row, d, is_key)));
                    const float scale = F::round(scale_from_absmax(most, range.width)), divisor = F::round(round_to_dtype(c.param_dtype, scale));
                    constexpr uint32_t kByte = 8 / kBits;  // entries of a byte
                    for (uint32_t d = d0; d < d0 + block; d += kByte) {
                        float v[4] = {entry(row, d, is_key), kByte == 2 ? entry(row, d + 1u, is_key) : 0.0f, 0.0f, 0.0f}, codes[4];
                        quantize_codes<F, 4, kEnc>(v, divisor, false, range.lo, range.hi, range.unrounded, codes);
                        uint32_t w[2];
                        if constexpr (kEnc == kEncInt)
                            pack_chunk_neg<kBits, 4, false>(codes, w);
                        else
                            encode_chunk<kEnc, 4>(codes, w);
                        to[d / kByte] = static_cast<char>(w[0] & 255u);
                    }
                    store_dtype(c.param_dtype, side.scales, scale_at + d0 / c.block * side.scale_block, scale);
                }
            }
        }
    };
    if constexpr (kWide) {
        if (threadIdx.x / 64u * 64u < tasks2) task(threadIdx.x);
    } else {
        for (uint32_t t = threadIdx.x; t < (tasks2 + 63u) / 64u * 64u; t += 256) task(t);
    }
}

bool on(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether rows of floats and of the cache can be taken eight entries at a time.
template <class F>
bool takes_wide(const AppendArgs& a, uint32_t bits) {
    const CacheArgs& c = a.cache;
    const uint64_t lanes = 16 / F::kBytes;
    const auto floats = [&](const void* p, uint64_t token, uint64_t head) { return on(p, 16) && token % lanes == 0 && head % lanes == 0; };
    const uint64_t row = bits ? bits : 16;  // bytes of a lane's store: eight codes, or 16 bytes of floats
    const auto stored = [&](const CacheSide& s) { return on(s.base, row) && s.page % row == 0 && s.head % row == 0 && s.slot % row == 0; };
    if (c.dim % kEach || !floats(a.k, a.k_token, a.k_head) || !floats(a.v, a.v_token, a.v_head) || !stored(c.keys) || !stored(c.values)) return false;
    if (a.heads && (!floats(a.q, a.q_token, a.q_head) || !floats(a.q_out, a.out_token, a.out_head))) return false;
    if (a.pairs % (a.interleaved ? kEach / 2 : kEach)) return false;
    return !bits || (c.block % kEach == 0 && (c.block & (c.block - 1u)) == 0 && c.block <= 64 * kEach);
}

template <class F, int kEnc, int kBits>
hipError_t launch_typed(hipStream_t s, AppendArgs a) {
    const uint32_t all = a.heads + 2u * a.cache.kv_heads;
    a.rows = kWorkEntries / a.cache.dim < all ? kWorkEntries / a.cache.dim : all;
    const dim3 grid(a.tokens, (all + a.rows - 1u) / a.rows);
    const uint32_t turns = a.pairs * sizeof(double2);
    if (takes_wide<F>(a, kBits))
        hipLaunchKernelGGL((append_kernel<F, kEnc, kBits, true>), grid, dim3(256), turns, s, a);
    else
        hipLaunchKernelGGL((append_kernel<F, kEnc, kBits, false>), grid, dim3(256), turns + a.rows * a.cache.dim * F::kBytes, s, a);
    return hipGetLastError();
}

template <class F>
hipError_t launch_append_of(hipStream_t s, const AppendArgs& a) {
    switch (a.cache.code) {
        case kCacheInt8: return launch_typed<F, kEncInt, 8>(s, a);
        case kCacheInt4: return launch_typed<F, kEncInt, 4>(s, a);
        case kCacheE4M3: return launch_typed<F, kEncE4M3, 8>(s, a);
        case kCacheE5M2: return launch_typed<F, kEncE5M2, 8>(s, a);
        case kCacheE2M1: return launch_typed<F, kEncE2M1, 4>(s, a);
        default: return launch_typed<F, kEncInt, 0>(s, a);
    }
}

}  // namespace

#define CQ_APPEND_NAME2(f) launch_append_##f
#define CQ_APPEND_NAME(f) CQ_APPEND_NAME2(f)
hipError_t CQ_APPEND_NAME(CQ_TU_FLOAT)(hipStream_t s, const AppendArgs& a) { return launch_append_of<CQ_TU_FLOAT>(s, a); }

}  // namespace cq
