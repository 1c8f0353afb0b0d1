// The sums of workgroups that share the columns of a product (cq_kernels_matmul_tiles.hip), added up in their order, and what stands behind them.
#include "cq_matmul_epilogue.hpp"
#include "cq_matmul_tiles.hpp"

namespace cq {
namespace {

// A thread finishes eight columns of a position, whose expert decides on the bias: tiles of 32 positions, as the experts cut them.
__global__ __launch_bounds__(256) void matmul_finish_kernel(MatmulArgs a, uint32_t splits, uint32_t pitch) {
    TileOfPositions at;
    for (uint32_t tile = blockIdx.y; find_tile(a, tile, 5, &at); tile += gridDim.y) {
        const uint32_t eights = (a.out_cols + 7u) / 8u, all = eights * (at.last - at.first);
        for (uint32_t n = blockIdx.x * 256u + threadIdx.x; n < all; n += gridDim.x * 256u) {
            const uint32_t p = at.first + n / eights, col = n % eights * 8u;
            const float* from = static_cast<const float*>(a.workspace) + static_cast<uint64_t>(p) * pitch + col;
            f32x8 v = load8(from), up = a.gated ? load8(from + pitch / 2) : f32x8{};
            for (uint32_t s = 1; s < splits; s++) {
                from += static_cast<uint64_t>(a.positions) * pitch;
                v += load8(from);
                if (a.gated) up += load8(from + pitch / 2);
            }
            v += load_bias8(a, at.expert, col);
            if (a.gated) up += load_bias8(a, at.expert, a.out_cols + col);
            finish8(a, p, col, v, up);
        }
    }
}

}  // namespace

hipError_t launch_matmul_finish(hipStream_t s, const MatmulArgs& a, uint32_t splits) {
    const uint64_t tiles = most_tiles(a, 5);
    const uint32_t eights = (a.out_cols + 7) / 8, each = a.positions < 32 ? a.positions : 32;
    hipLaunchKernelGGL(matmul_finish_kernel, dim3((eights * each + 255) / 256, static_cast<uint32_t>(tiles < 65535 ? tiles : 65535)), dim3(256), 0, s, a, splits,
                       TilesGrid::sums_pitch(a));
    return hipGetLastError();
}

}  // namespace cq
