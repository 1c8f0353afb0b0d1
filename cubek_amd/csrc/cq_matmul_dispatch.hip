// Which kernel on the matrix cores a product takes, and which object holds it.
#include "cq_matmul_tiles.hpp"

namespace cq {

#define CQ_BY_CODE(kernel, f, ...)                                                             \
    switch (a.native == 1 ? 100u : a.native == 2 ? 101u : a.native == 3 ? 102u : a.bits) {     \
        case 2: return kernel##_##f##_2(__VA_ARGS__);                                          \
        case 4: return kernel##_##f##_4(__VA_ARGS__);                                          \
        case 100: return kernel##_##f##_100(__VA_ARGS__);                                      \
        case 101: return kernel##_##f##_101(__VA_ARGS__);                                      \
        case 102: return kernel##_##f##_102(__VA_ARGS__);                                      \
        default: return kernel##_##f##_8(__VA_ARGS__);                                         \
    }

hipError_t launch_matmul_tiles(hipStream_t s, const MatmulArgs& a) {
    const MatmulChoice choice = matmul_choice(a);
    if (choice.few) {
        if (a.dtype == CQ_BF16) CQ_BY_CODE(matmul_few, BF16, s, a, choice.few_shape)
        CQ_BY_CODE(matmul_few, F16, s, a, choice.few_shape)
    }
    const auto product = [&]() -> hipError_t {
        if (a.dtype == CQ_BF16) CQ_BY_CODE(matmul_tiles, BF16, s, a, choice.tiles)
        CQ_BY_CODE(matmul_tiles, F16, s, a, choice.tiles)
    };
    const hipError_t err = product();
    return err != hipSuccess || choice.tiles.splits == 1 ? err : launch_matmul_finish(s, a, choice.tiles.splits);
}

}  // namespace cq
