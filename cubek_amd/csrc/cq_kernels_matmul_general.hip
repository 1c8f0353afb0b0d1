// Products with quantized weights of any scheme, block, type and alignment: the kernel for what the matrix-core kernels do not
// take (x in f32, rows that do not start on 16-byte boundaries, blocks narrower than 16 bytes of codes).
//
// A workgroup makes 64 positions x 64 columns of y, 32 columns of W at a time: every weight is decoded and rounded once per
// workgroup, F(F(scale) * F(code)), into LDS as f32, and a thread sums 4 x 4 products by FMAs.  Bound by the vector ALUs: 157 TFLOP/s
// would be their peak; what it reaches is 4.7 TFLOP/s ([28672, 8192], 4096 tokens: 0.41 s), most of it the decoding value by value.
#include "../../include/cubek_quant_device.hpp"
#include "cq_matmul_epilogue.hpp"

namespace cq {
namespace {

namespace dev = cubek_quant::device;

__device__ __forceinline__ float rounded(int dtype, float v) {
    if (dtype == CQ_F32) return v;
    return dtype == CQ_F16 ? dev::round_to<dev::Float::F16>(v) : dev::round_to<dev::Float::BF16>(v);
}

// The number that value k of a stored row holds.
__device__ __forceinline__ float decoded(const MatmulArgs& a, const char* row, uint32_t k) {
    const auto byte = [&](uint32_t at) { return static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(row)[at]); };
    switch (a.native) {
        case 1: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte(k)), 0);
        case 2: return __builtin_amdgcn_cvt_f32_bf8(static_cast<int>(byte(k)), 0);
        case 3: {
            const uint32_t nibble = (byte(k / 2) >> (4 * (k % 2))) & 15u;
            return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(nibble, 1.0f, 0)[0];
        }
    }
    const uint32_t at = k * a.bits;  // fields lie in ascending order in the bytes of a word, and no field crosses a byte
    const uint32_t field = byte(at / 8) >> (at % 8);
    return static_cast<float>(static_cast<int32_t>(field << (32 - a.bits)) >> (32 - a.bits));
}

constexpr uint32_t kTileLog2 = 6, kTile = 1u << kTileLog2, kStep = 32;

__global__ __launch_bounds__(256) void matmul_general_kernel(MatmulArgs a) {
    __shared__ float xs[kStep][kTile + 1], gate[kStep][kTile + 1], up[kStep][kTile + 1];
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const uint32_t n0 = blockIdx.x * kTile;
    TileOfPositions at;
    for (uint32_t tile = blockIdx.y; find_tile(a, tile, kTileLog2, &at); tile += gridDim.y) {
        const uint32_t e = at.expert;
        const char* const words = a.words + e * a.expert_bytes;
        const auto weight = [&](uint32_t n, uint32_t k) {
            const uint64_t i = a.block_rows == 0 ? 0 : e * a.scale_expert + n / a.block_rows * a.scale_row + k / a.block_cols * a.scale_col;
            return rounded(a.dtype, rounded(a.dtype, load_float(a.param_dtype, a.scales, i)) * decoded(a, words + n * a.row_bytes, k));
        };
        float v[4][4] = {}, w[4][4] = {};
        for (uint32_t k0 = 0; k0 < a.cols; k0 += kStep) {
#pragma unroll
            for (uint32_t i = 0; i < kTile * kStep / 256; i++) {
                const uint32_t l = i * 256 + threadIdx.x, k = l % kStep, r = l / kStep;
                const bool there = k0 + k < a.cols;
                const uint32_t p = min(at.first + r, at.last - 1), n = min(n0 + r, a.out_cols - 1);
                xs[k][r] = there ? load_float(a.dtype, a.x, row_of_position(a, p) * a.x_stride + k0 + k) : 0.0f;
                gate[k][r] = there ? weight(n, k0 + k) : 0.0f;
                if (a.gated) up[k][r] = there ? weight(a.out_cols + n, k0 + k) : 0.0f;
            }
            __syncthreads();
            // a step's products are summed apart: a long row is rounded as often as it has steps, not as often as it has columns
            float dv[4][4] = {}, dw[4][4] = {};
            for (uint32_t k = 0; k < kStep; k++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        dv[i][j] = __builtin_fmaf(xs[k][ty + 16 * i], gate[k][tx + 16 * j], dv[i][j]);
                        if (a.gated) dw[i][j] = __builtin_fmaf(xs[k][ty + 16 * i], up[k][tx + 16 * j], dw[i][j]);
                    }
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) v[i][j] += dv[i][j], w[i][j] += dw[i][j];
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t p = at.first + ty + 16 * i, n = n0 + tx + 16 * j;
                if (p >= at.last || n >= a.out_cols) continue;
                finish1(a, e, p, n, v[i][j], w[i][j]);
            }
    }
}

}  // namespace

hipError_t launch_matmul_general(hipStream_t s, const MatmulArgs& a) {
    const uint64_t tiles = most_tiles(a, kTileLog2);  // beyond what a launch's second dimension holds: some more each
    hipLaunchKernelGGL(matmul_general_kernel, dim3((a.out_cols + kTile - 1) / kTile, static_cast<uint32_t>(tiles < 65535 ? tiles : 65535)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace cq
