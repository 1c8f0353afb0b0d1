// A workspace of the size that a product asks for gives the kernel for which it asked, and so does any larger one: walked over random shapes.
#include <cstdio>
#include <cstdlib>

#include "../../cubek_amd/csrc/cq_matmul_tiles.hpp"

using namespace cq;

static int32_t some_offsets[2];
static uint32_t up_to(uint32_t n) { return 1 + static_cast<uint32_t>(rand()) % n; }

static bool alike(const MatmulChoice& x, const MatmulChoice& y) {
    if (x.few != y.few) return false;
    if (!x.few) return x.tiles.shape == y.tiles.shape && x.tiles.splits == y.tiles.splits;
    return x.few_shape.tokens_log2 == y.few_shape.tokens_log2 && x.few_shape.shares_log2 == y.few_shape.shares_log2 && x.few_shape.units == y.few_shape.units;
}

int main() {
    srand(7);
    uint32_t shared = 0;
    for (int n = 0; n < 300000; n++) {
        MatmulArgs a{};
        a.dtype = CQ_BF16;
        a.positions = a.tokens = up_to(rand() % 3 ? 700 : 5000);
        a.gated = rand() % 2;
        a.out_cols = up_to(rand() % 3 ? 300 : 10000);
        a.wide = a.gated ? 2 * a.out_cols : a.out_cols;
        a.bits = 2u << rand() % 3;
        a.block_cols = 32u << rand() % 3;
        a.cols = a.block_cols * up_to(rand() % 3 ? 40 : 400);
        a.experts = 1;
        if (rand() % 3 == 0) a.offsets = some_offsets, a.experts = up_to(64);
        a.workspace_bytes = ~0ull;
        const MatmulChoice asked = matmul_choice(a);
        const uint64_t bytes = asked.few ? 0 : sums_bytes(a, asked.tiles.splits);
        shared += bytes != 0;
        for (const uint64_t more : {0ull, 4096ull, 1ull << 28}) {
            a.workspace_bytes = bytes + more;
            if (alike(matmul_choice(a), asked)) continue;
            printf("positions %u out %u cols %u bits %u gated %u experts %u: another kernel with %llu bytes and %llu more\n", a.positions, a.out_cols, a.cols, a.bits,
                   a.gated, a.experts, (unsigned long long)bytes, (unsigned long long)more);
            return 1;
        }
    }
    printf("%u of them share their columns\nok\n", shared);
    return shared > 1000 ? 0 : 1;
}
