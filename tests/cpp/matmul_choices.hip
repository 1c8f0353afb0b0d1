// The host's side of the products, walked over random shapes: every choice fits the compute unit's LDS, the loads that a wave may take
// part in and the workspace it was given, and every tile of a grid is dealt out once, whatever the experts and the shares of the columns.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../cubek_amd/csrc/cq_matmul_tiles.hpp"

using namespace cq;

static int32_t some_offsets[2];

static uint32_t up_to(uint32_t n) { return 1 + static_cast<uint32_t>(rand()) % n; }

static MatmulArgs random_args() {
    MatmulArgs a{};
    a.positions = a.tokens = up_to(rand() % 3 ? 300 : 9000);
    a.gated = rand() % 2;
    a.out_cols = up_to(rand() % 4 ? 2000 : 20000);
    a.wide = a.gated ? 2 * a.out_cols : a.out_cols;
    a.bits = 2u << rand() % 3;
    a.block_cols = 32u << rand() % 4;
    a.cols = a.block_cols * up_to(rand() % 4 ? 20 : 300);
    a.experts = 1;
    if (rand() % 2) a.offsets = some_offsets, a.experts = up_to(140);
    a.workspace_bytes = rand() % 2 ? 1ull << (10 + rand() % 22) : 0;
    return a;
}

#define CHECK(condition)                                                                                                                          \
    if (!(condition)) {                                                                                                                           \
        printf("%s: positions %u out %u cols %u bits %u block %u experts %u (%d) gated %u workspace %llu\n", #condition, a.positions, a.out_cols, \
               a.cols, a.bits, a.block_cols, a.experts, a.offsets != nullptr, a.gated, (unsigned long long)a.workspace_bytes);                    \
        return 1;                                                                                                                                 \
    }

int main() {
    srand(11);
    for (int n = 0; n < 20000; n++) {
        const MatmulArgs a = random_args();
        const MatmulChoice c = matmul_choice(a);
        CHECK(c.us < 1e30);
        if (c.few) {
            const FewShape& f = c.few_shape;
            CHECK(f.lds() <= 160 * 1024 && f.x_loads() <= 8 && f.shares_log2 <= 3 && a.block_cols % (128 / a.bits) == 0);
            CHECK(a.offsets || a.positions <= 1u << f.tokens_log2);
            CHECK((f.units == 4 || (f.units == 8 && a.bits > 2 && f.tokens_log2 < 5)) && f.x_bytes >= (a.positions < 1u << f.tokens_log2 ? a.positions : 1u << f.tokens_log2) * f.units * (128 / a.bits) * 2);
        } else {
            CHECK(c.tiles.splits >= 1 && sums_bytes(a, c.tiles.splits) <= a.workspace_bytes);
        }
        static const uint32_t rows[] = {256, 256, 128, 128, 32}, tokens[] = {128, 128, 64, 32, 32};
        const int shape = c.few ? rand() % 5 : static_cast<int>(c.tiles.shape);
        const TilesGrid g(a, rows[shape], tokens[shape], c.few ? 1u << rand() % 5 : c.tiles.splits);
        const uint32_t each = g.group * g.chunk, chunks = (g.n_tiles - g.wider_chunks) / g.chunk_width;
        std::vector<uint8_t> dealt(static_cast<size_t>(g.n_tiles) * g.p_tiles);
        for (uint32_t block = 0; block < g.workgroups(); block++) {  // as TilesGrid::tile divides on the device
            const uint32_t round = block / 8 / each, within = block / 8 % each, r = round * 8 + (block + round * g.turn) % 8;
            const uint32_t n_chunk = r % chunks, p_group = r / chunks, in_chunk = within / g.group, in_group = within % g.group;
            if (in_chunk >= g.chunk_width + (n_chunk < g.wider_chunks) || in_group >= g.group_width + (p_group < g.wider_groups)) continue;
            const uint32_t row_tile = n_chunk * g.chunk_width + std::min(n_chunk, g.wider_chunks) + in_chunk;
            const uint32_t tile = p_group * g.group_width + std::min(p_group, g.wider_groups) + in_group;
            CHECK(row_tile < g.n_tiles);
            if (tile < g.p_tiles) dealt[static_cast<size_t>(tile) * g.n_tiles + row_tile]++;
        }
        for (const uint8_t times : dealt) CHECK(times == 1);
    }
    printf("ok\n");
    return 0;
}
