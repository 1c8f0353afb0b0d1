// What stands behind a product, in f32: bias, activation, gate, residual, and the one rounding to the type of y.
#pragma once

#include "cq_matmul_internal.hpp"

namespace cq {
namespace {

__device__ __forceinline__ float load_float(int dtype, const char* p, uint64_t i) {
    if (dtype == CQ_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == CQ_F16) return static_cast<float>(reinterpret_cast<const _Float16*>(p)[i]);
    return static_cast<float>(reinterpret_cast<const __bf16*>(p)[i]);
}

__device__ __forceinline__ void store_float(int dtype, char* p, uint64_t i, float v) {
    if (dtype == CQ_F32)
        reinterpret_cast<float*>(p)[i] = v;
    else if (dtype == CQ_F16)
        reinterpret_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    else
        reinterpret_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
}

// 1 / (1 + exp(-v)), by the hardware's exp2 and reciprocal (one unit in the last place each).
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)); }

// erfc(x) for x >= 0 by Abramowitz and Stegun 7.1.26 (Hastings), a fifth-order polynomial in 1 / (1 + p x) times exp(-x^2): within 1.5e-7, and in
// the tail as small as erfc itself, so that a product with it loses nothing to cancellation (relative to itself it is off by 3e-3 where GELU is 1e-8 of v).  The library's erff takes three times the
// instructions (gelu of 4096 x 28672 values).
__device__ __forceinline__ float erfc_positive(float x) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
    float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    p = __builtin_fmaf(p, t, 1.421413741f);
    p = __builtin_fmaf(p, t, -0.284496736f);
    p = __builtin_fmaf(p, t, 0.254829592f);
    return p * t * __builtin_amdgcn_exp2f(x * x * -1.4426950408889634f);
}

// `activation` is uniform over the launch.
__device__ __forceinline__ float activated(uint32_t activation, float v) {
    switch (activation) {
        case CQ_ACT_RELU: return v < 0.0f ? 0.0f : v;
        case CQ_ACT_SILU: return v * sigmoid(v);
        case CQ_ACT_GELU: {
            // v times the share of it that counts: v less the share's complement would be inf - inf * 0 at infinity
            const float tail = 0.5f * erfc_positive(__builtin_fabsf(v) * 0.70710678118654752f);
            return v * (v < 0.0f ? tail : 1.0f - tail);
        }
        // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
        case CQ_ACT_GELU_TANH: return v * sigmoid(1.5957691216057308f * __builtin_fmaf(0.044715f * v * v, v, v));
        default: return v;
    }
}

// The workgroup's tile: positions first .. last - 1 of expert e.
struct TileOfPositions {
    uint32_t expert, first, last;
};

// Tile number `tile` when the positions of every expert are cut into tiles of 2^size_log2, expert by expert; false past the last one.  The
// offsets lie in device memory, where the host cannot check them: they are taken into 0 .. positions, and a range that runs
// backwards is empty.  Every wave looks at 64 experts at a time, so that 128 of them take two rounds of loads instead of 128.
__device__ __forceinline__ bool find_tile(const MatmulArgs& a, uint32_t tile, uint32_t size_log2, TileOfPositions* out) {
    const uint32_t round_up = (1u << size_log2) - 1u;
    if (a.offsets == nullptr) {
        out->expert = 0;
        out->first = tile << size_log2;
        out->last = min(a.positions, out->first + round_up + 1u);
        return out->first < a.positions;
    }
    const uint32_t lane = threadIdx.x & 63u;
    const int32_t most = static_cast<int32_t>(a.positions);
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 64) {
        const uint32_t e = min(e0 + lane, a.experts - 1u);
        const uint32_t first = static_cast<uint32_t>(min(max(a.offsets[e], 0), most)), last = static_cast<uint32_t>(min(max(a.offsets[e + 1], 0), most));
        const uint32_t tiles = e0 + lane < a.experts && last > first ? (last - first + round_up) >> size_log2 : 0u;
        uint32_t sum = tiles;
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t below = __shfl_up(sum, d);
            sum += lane >= d ? below : 0u;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(tile < sum);
        if (past != 0) {
            const uint32_t l = static_cast<uint32_t>(__builtin_ctzll(past));
            const uint32_t in = tile - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
            out->expert = e0 + l;
            out->first = __builtin_amdgcn_readlane(first, l) + (in << size_log2);
            out->last = min(static_cast<uint32_t>(__builtin_amdgcn_readlane(last, l)), out->first + round_up + 1u);
            return true;
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

__device__ __forceinline__ uint32_t row_of_position(const MatmulArgs& a, uint32_t p) {
    if (a.row_of == nullptr) return p;
    return static_cast<uint32_t>(min(max(a.row_of[p], 0), static_cast<int32_t>(a.tokens) - 1));
}

// Column col of position p from its sum, and the gated one's.
__device__ __forceinline__ void finish1(const MatmulArgs& a, uint32_t expert, uint32_t p, uint32_t col, float v, float up) {
    if (a.bias) {
        v += load_float(a.bias_dtype, a.bias, expert * a.bias_expert + col * a.bias_stride);
        if (a.gated) up += load_float(a.bias_dtype, a.bias, expert * a.bias_expert + (a.out_cols + col) * a.bias_stride);
    }
    v = activated(a.activation, v);
    if (a.gated) v *= up;
    if (a.residual) v += load_float(a.y_dtype, a.residual, p * a.residual_stride + col);
    store_float(a.y_dtype, a.y, p * a.y_stride + col, v);
}

typedef float f32x8 __attribute__((ext_vector_type(8)));

// Eight floats from a boundary of 16 bytes.
__device__ __forceinline__ f32x8 load8(const float* p) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const f32x4 low = *reinterpret_cast<const f32x4*>(p), high = *reinterpret_cast<const f32x4*>(p + 4);
    return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Eight floats of any type, from any of their addresses: 16-byte accesses need no boundary on gfx950 (element by element 10580 columns of f16 with a
// residual, 355 positions, took 38.7 us).
__device__ __forceinline__ f32x8 load_floats8(int dtype, const char* p, uint64_t i) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    if (dtype == CQ_F32) return load8(reinterpret_cast<const float*>(p) + i);
    const u32x4 bits = *reinterpret_cast<const u32x4*>(p + i * 2);
    if (dtype == CQ_F16) return __builtin_convertvector(__builtin_bit_cast(f16x8, bits), f32x8);
    f32x8 v;
#pragma unroll
    for (int k = 0; k < 4; k++) v[2 * k] = __builtin_bit_cast(float, bits[k] << 16), v[2 * k + 1] = __builtin_bit_cast(float, bits[k] & 0xffff0000u);
    return v;
}

// Eight columns, rounded once.
__device__ __forceinline__ void store8(int dtype, char* y, uint64_t at, f32x8 v) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    if (dtype == CQ_F32) {
        *reinterpret_cast<f32x4*>(y + at * 4) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(y + at * 4 + 16) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4*>(y + at * 2) = dtype == CQ_F16 ? __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8))
                                                                : __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
    }
}

// The bias of rows row .. row + 7 of W, as far as W has them; for all positions of a lane, which asks for it once.
__device__ __forceinline__ f32x8 load_bias8(const MatmulArgs& a, uint32_t expert, uint32_t row) {
    f32x8 v = {};
    if (a.bias == nullptr) return v;
    const uint64_t at = expert * a.bias_expert;
    if (a.bias_stride == 1 && row + 8u <= a.wide) return load_floats8(a.bias_dtype, a.bias, at + row);
#pragma unroll
    for (uint32_t k = 0; k < 8; k++) v[k] = load_float(a.bias_dtype, a.bias, at + min(row + k, a.wide - 1u) * a.bias_stride);
    return v;
}

// Columns col .. col + 7 of position p, as far as y has them, from their sums and those of the gated ones, bias and all.
__device__ __forceinline__ void finish8(const MatmulArgs& a, uint32_t p, uint32_t col, f32x8 v, f32x8 up) {
    const bool whole = col + 8 <= a.out_cols;
    if (a.activation != CQ_ACT_IDENTITY) {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) v[k] = activated(a.activation, v[k]);
    }
    if (a.gated) {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) v[k] *= up[k];
    }
    const uint64_t y_at = p * a.y_stride + col, r_at = p * a.residual_stride + col;
    if (whole) {
        if (a.residual) v += load_floats8(a.y_dtype, a.residual, r_at);
        store8(a.y_dtype, a.y, y_at, v);
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 8; k++)
        if (col + k < a.out_cols) {
            float out = v[k];
            if (a.residual) out += load_float(a.y_dtype, a.residual, r_at + k);
            store_float(a.y_dtype, a.y, y_at + k, out);
        }
}

}  // namespace
}  // namespace cq
