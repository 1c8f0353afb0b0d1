// What the products on the matrix cores share: codes and scales as they lie in memory and LDS, to operands of the instructions.
#pragma once

#include "cq_gemv_operand.hpp"

namespace cq {
namespace {

#define CQ_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

constexpr int bits_of(int code) { return code <= 8 ? code : (code == kCodeE2M1x2 ? 4 : 8); }

// A stored scale is loaded as the word around it and made a number later: a load is not waited for where it is issued.  By masks instead of
// branches, which would cut a step's instructions into pieces: all bits or none of a word, by the type of the scales (uniform over the launch).
struct ScaleMasks {
    uint32_t f32, bf16, f16;
    __device__ explicit ScaleMasks(int dtype) : f32(dtype == CQ_F32 ? ~0u : 0u), bf16(dtype == CQ_BF16 ? ~0u : 0u), f16(dtype == CQ_F16 ? ~0u : 0u) {}
};
__device__ __forceinline__ float scale_of(const ScaleMasks& m, uint32_t word, uint32_t offset) {
    const uint32_t half = word >> ((offset & 2u) * 8u);
    const uint32_t from_f16 = __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(half))));
    return __builtin_bit_cast(float, (word & m.f32) | (half << 16 & m.bf16) | (from_f16 & m.f16));
}

__device__ const char kZeros[16] __attribute__((aligned(16))) = {};

// The 32 codes of a lane's row in a step: 2, 4 or 8 words.
template <int kCode>
struct Codes {
    uint32_t word[bits_of(kCode)];
};

// Values 8 m .. 8 m + 7 of 16 bytes of codes as the matrix instruction takes them.
template <dev::Float kF, int kCode, bool kShort>
__device__ __forceinline__ u32x4 unit_slice(const u32x4& unit, uint32_t m, float scale) {
    if constexpr (kCode == 2) {
        uint32_t p[8];
        if constexpr (kShort)
            dev::dequantize_symmetric_packed_value_pairs_tame<kF, 2>(unit[m / 2], scale, p);
        else
            dev::dequantize_symmetric_packed_value_pairs<kF, 2>(unit[m / 2], scale, p);
        return m % 2 == 0 ? u32x4{p[0], p[1], p[2], p[3]} : u32x4{p[4], p[5], p[6], p[7]};
    } else {
        return operand<kF, kCode, kShort>(unit, m, scale);
    }
}

// Values 8 m .. 8 m + 7 of a lane's 32.
template <dev::Float kF, int kCode, bool kShort>
__device__ __forceinline__ u32x4 slice(const Codes<kCode>& c, uint32_t m, float scale) {
    if constexpr (kCode == 2) {
        return unit_slice<kF, kCode, kShort>(u32x4{c.word[0], c.word[1], 0, 0}, m, scale);
    } else if constexpr (bits_of(kCode) == 4) {
        return operand<kF, kCode, kShort>(u32x4{c.word[0], c.word[1], c.word[2], c.word[3]}, m, scale);
    } else {
        const uint32_t first = m / 2 * 4;
        return operand<kF, kCode, kShort>(u32x4{c.word[first], c.word[first + 1], c.word[first + 2], c.word[first + 3]}, m % 2, scale);
    }
}

// Whether the short dequantization takes a scale (2-bit fields have only the one range of tame scales).
template <dev::Float kF, int kCode>
__device__ __forceinline__ bool takes_short(float scale) {
    if constexpr (kCode > 8) return true;
    if constexpr (kCode == 2) return dev::pairs_scale_is_tame<kF>(scale);
    return (__builtin_bit_cast(uint32_t, scale) & 0x7fffffffu) < kShortBelow<kF, kCode>;
}

}  // namespace
}  // namespace cq
