// Products with quantized weights of any scheme, block, type and alignment: the kernel for what the matrix-core kernels do not
// take (x in f32, rows that do not start on 16-byte boundaries, blocks narrower than 16 bytes of codes).
//
// Every weight is decoded and rounded once per workgroup, F(F(scale) * F(code)), into LDS as f32, where a thread takes its numbers of x and of W
// with one access each for its FMAs; the next step's words are on their way meanwhile.  Bound by the decoding value by value and by the
// FMAs: 14 TFLOP/s of the vector units' 157, without the matrix instructions that there are for f32 (f32 x, [4096, 4096] 4 bits, 4096 positions 9.8 ms, 512 1.27 ms, 64 0.63 ms, 1 to 16 0.10 ms; with loads
// that waited for one another behind branches on the types 25.8, 3.2, 1.49 and 1.45 ms).
#include "../../include/cubek_quant_device.hpp"
#include "cq_matmul_epilogue.hpp"
#include "cq_matmul_weights.hpp"

namespace cq {
namespace {

// A number of 4 bytes or of 2, as the word around it and where in it: every load of a step is on its way before the first is looked at.
struct Around {
    const char* base;
    uint32_t in;
    __device__ explicit Around(const char* p) : base(p - (reinterpret_cast<uintptr_t>(p) & 3u)), in(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 3u)) {}
    __device__ uint32_t word(uint64_t offset) const { return *reinterpret_cast<const uint32_t*>(base + ((offset + in) & ~3ull)); }
    __device__ float number(const ScaleMasks& m, uint32_t word, uint64_t offset) const { return scale_of(m, word, static_cast<uint32_t>(offset) + in); }
};

// The number that value k of a stored row holds, from the byte that has it: no value crosses one.
__device__ __forceinline__ float decoded(const MatmulArgs& a, uint32_t byte, uint32_t k) {
    switch (a.native) {
        case 1: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte), 0);
        case 2: return __builtin_amdgcn_cvt_f32_bf8(static_cast<int>(byte), 0);
        case 3: return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((byte >> (4 * (k % 2))) & 15u, 1.0f, 0)[0];
    }
    const uint32_t field = byte >> (k * a.bits % 8);
    return static_cast<float>(static_cast<int32_t>(field << (32 - a.bits)) >> (32 - a.bits));
}

// 4 x 4 results of a thread in tiles of 64 positions x 64 columns, steps of 32 columns of W; for up to 16 positions one result of a thread in
// tiles of 16 x 16, steps of 128 columns: four times the workgroups, and a quarter of the products for nobody.
template <dev::Float kF, int kEach, int kStep>
__global__ __launch_bounds__(256) void matmul_general_kernel(MatmulArgs a, uint32_t first) {
    constexpr uint32_t kTile = 16 * kEach, kTileLog2 = kEach == 4 ? 6 : 4;
    typedef float vec __attribute__((ext_vector_type(kEach)));
    constexpr uint32_t kPitch = kTile + kEach;  // a thread's numbers are read at once
    __shared__ alignas(16) float xs[kStep][kPitch], gate[kStep][kPitch], up[kStep][kPitch];
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const uint32_t n0 = (first + blockIdx.x) * kTile;
    constexpr uint32_t kLoads = kTile * kStep / 256, kRowsApart = 256 / kStep;
    const uint32_t own_k = threadIdx.x % kStep, own_row = threadIdx.x / kStep;  // a thread brings the same column of kLoads rows in every step
    const Around x(a.x), scales(a.scales);
    const ScaleMasks x_masks(a.dtype), scale_masks(a.param_dtype);
    const uint32_t x_size = a.dtype == CQ_F32 ? 4 : 2, scale_size = a.param_dtype == CQ_F32 ? 4 : 2, code_bits = a.native == 3 ? 4 : a.native ? 8 : a.bits;
    TileOfPositions at;
    for (uint32_t tile = blockIdx.y; find_tile(a, tile, kTileLog2, &at); tile += gridDim.y) {
        const uint32_t e = at.expert;
        uint64_t x_at[kLoads], scale_at[2][kLoads], row_at[2][kLoads];  // in bytes
#pragma unroll
        for (uint32_t i = 0; i < kLoads; i++) {
            const uint32_t r = own_row + i * kRowsApart;
            x_at[i] = row_of_position(a, min(at.first + r, at.last - 1)) * a.x_stride * x_size;
#pragma unroll
            for (uint32_t u = 0; u < 2; u++) {
                const uint32_t n = min(n0 + r, a.out_cols - 1) + (a.gated ? u * a.out_cols : 0);
                row_at[u][i] = e * a.expert_bytes + n * a.row_bytes;
                scale_at[u][i] = a.block_rows == 0 ? 0 : (e * a.scale_expert + n / a.block_rows * a.scale_row) * scale_size;
            }
        }
        float v[kEach][kEach] = {}, w[kEach][kEach] = {};
        uint32_t x_word[kLoads], scale[2][kLoads], code[2][kLoads];
        const auto column = [&](uint32_t k0) { return min(k0 + own_k, a.cols - 1); };
        const auto scale_column = [&](uint32_t k) -> uint64_t { return a.block_rows == 0 ? 0 : k / a.block_cols * a.scale_col * scale_size; };
        const auto load = [&](uint32_t k) {
            const uint64_t scale_k = scale_column(k), code_k = static_cast<uint64_t>(k) * code_bits / 8;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; i++) x_word[i] = x.word(x_at[i] + static_cast<uint64_t>(k) * x_size);
#pragma unroll
            for (uint32_t u = 0; u < 2; u++)
                if (u == 0 || a.gated) {
#pragma unroll
                    for (uint32_t i = 0; i < kLoads; i++) {
                        scale[u][i] = scales.word(scale_at[u][i] + scale_k);
                        code[u][i] = reinterpret_cast<const uint8_t*>(a.words)[row_at[u][i] + code_k];
                    }
                }
        };
        if (a.cols) load(column(0));
        for (uint32_t k0 = 0; k0 < a.cols; k0 += kStep) {
            const uint32_t k = column(k0);
            const bool there = k0 + own_k < a.cols;
            const uint64_t scale_k = scale_column(k);
            const auto weight = [&](uint32_t u, uint32_t i) {
                const float s = scales.number(scale_masks, scale[u][i], scale_at[u][i] + scale_k);
                return there ? dev::round_to<kF>(dev::round_to<kF>(s) * decoded(a, code[u][i], k)) : 0.0f;
            };
#pragma unroll
            for (uint32_t i = 0; i < kLoads; i++) {
                const uint32_t r = own_row + i * kRowsApart;
                xs[own_k][r] = there ? x.number(x_masks, x_word[i], x_at[i] + static_cast<uint64_t>(k) * x_size) : 0.0f;
                gate[own_k][r] = weight(0, i);
                if (a.gated) up[own_k][r] = weight(1, i);
            }
            __syncthreads();
            if (k0 + kStep < a.cols) load(column(k0 + kStep));  // on their way during the products
            // a step's products are summed apart: a long row is rounded as often as it has steps, not as often as it has columns
            float dv[kEach][kEach] = {}, dw[kEach][kEach] = {};
            const auto multiply = [&](auto gated) {
#pragma unroll 8
                for (uint32_t c = 0; c < kStep; c++) {
                    const vec xv = *reinterpret_cast<const vec*>(&xs[c][ty * kEach]), gv = *reinterpret_cast<const vec*>(&gate[c][tx * kEach]);
                    const vec uv = decltype(gated)::value ? *reinterpret_cast<const vec*>(&up[c][tx * kEach]) : vec{};
#pragma unroll
                    for (uint32_t i = 0; i < kEach; i++)
#pragma unroll
                        for (uint32_t j = 0; j < kEach; j++) {
                            dv[i][j] = __builtin_fmaf(xv[i], gv[j], dv[i][j]);
                            if (decltype(gated)::value) dw[i][j] = __builtin_fmaf(xv[i], uv[j], dw[i][j]);
                        }
                }
            };
            if (a.gated)
                multiply(std::true_type{});
            else
                multiply(std::false_type{});
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++)
#pragma unroll
                for (uint32_t j = 0; j < kEach; j++) v[i][j] += dv[i][j], w[i][j] += dw[i][j];
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++)
#pragma unroll
            for (uint32_t j = 0; j < kEach; j++) {
                const uint32_t p = at.first + ty * kEach + i, n = n0 + tx * kEach + j;
                if (p >= at.last || n >= a.out_cols) continue;
                finish1(a, e, p, n, v[i][j], w[i][j]);
            }
    }
}

template <dev::Float kF, int kEach, int kStep>
hipError_t launch(hipStream_t s, const MatmulArgs& a) {
    constexpr uint32_t kTile = 16 * kEach;
    const uint64_t tiles = most_tiles(a, kEach == 4 ? 6 : 4);  // beyond what a launch's second dimension holds: some more each
    const uint32_t all = (a.out_cols + kTile - 1) / kTile, most = kLaunchThreads / 256 - 1;
    for (uint32_t first = 0; first < all; first += most) {
        hipLaunchKernelGGL((matmul_general_kernel<kF, kEach, kStep>), dim3(all - first < most ? all - first : most, static_cast<uint32_t>(tiles < 65535 ? tiles : 65535)),
                           dim3(256), 0, s, a, first);
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    return hipSuccess;
}

template <dev::Float kF>
hipError_t launch_tile(hipStream_t s, const MatmulArgs& a) {
    const uint64_t experts = a.offsets ? (a.experts < a.positions ? a.experts : a.positions) : 1;
    return a.positions <= 16 * experts ? launch<kF, 1, 128>(s, a) : launch<kF, 4, 32>(s, a);
}

}  // namespace

hipError_t launch_matmul_general(hipStream_t s, const MatmulArgs& a) {
    if (a.dtype == CQ_F32) return launch_tile<dev::Float::F32>(s, a);
    return a.dtype == CQ_F16 ? launch_tile<dev::Float::F16>(s, a) : launch_tile<dev::Float::BF16>(s, a);
}

}  // namespace cq
