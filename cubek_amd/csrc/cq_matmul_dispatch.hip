// Which object holds the kernels for a product on the matrix cores.
#include "cq_matmul_tiles.hpp"

namespace cq {

hipError_t launch_matmul_tiles(hipStream_t s, const MatmulArgs& a) {
    const TilesShape shape = tiles_shape(a);
    const bool bf16 = a.dtype == CQ_BF16;
    switch (a.native) {
        case 1: return bf16 ? matmul_tiles_BF16_100(s, a, shape) : matmul_tiles_F16_100(s, a, shape);
        case 2: return bf16 ? matmul_tiles_BF16_101(s, a, shape) : matmul_tiles_F16_101(s, a, shape);
        case 3: return bf16 ? matmul_tiles_BF16_102(s, a, shape) : matmul_tiles_F16_102(s, a, shape);
    }
    switch (a.bits) {
        case 2: return bf16 ? matmul_tiles_BF16_2(s, a, shape) : matmul_tiles_F16_2(s, a, shape);
        case 4: return bf16 ? matmul_tiles_BF16_4(s, a, shape) : matmul_tiles_F16_4(s, a, shape);
        default: return bf16 ? matmul_tiles_BF16_8(s, a, shape) : matmul_tiles_F16_8(s, a, shape);
    }
}

}  // namespace cq
