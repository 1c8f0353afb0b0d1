// The products' limits, walked on the host: no product of 16-bit x with rows on boundaries leaves the kernels on the matrix cores for its number of
// positions or rows, what they launch has fewer than 2^32 threads along a dimension, and a scale's block is the quotient everywhere.
#include <cstdio>
#include <cstdlib>

#include "../../cubek_amd/csrc/cq_matmul_tiles.hpp"

using namespace cq;

#define CHECK(condition)                                                                                                                            \
    if (!(condition)) {                                                                                                                             \
        printf("%s: positions %u out %u cols %u bits %u block %u experts %u (%d) gated %u\n", #condition, a.positions, a.out_cols, a.cols, a.bits, \
               a.block_cols, a.experts, a.offsets != nullptr, a.gated);                                                                             \
        return 1;                                                                                                                                   \
    }

static uint64_t up_to(uint64_t n) { return 1 + (static_cast<uint64_t>(rand()) << 31 | static_cast<uint64_t>(rand())) % n; }
static uint64_t spread(uint32_t most_log2) { return up_to(1ull << (1 + rand() % most_log2)); }  // over its logarithm
static int32_t some_offsets[2];

static MatmulArgs product(uint64_t positions, uint64_t out_cols, uint32_t cols, uint32_t gated, uint32_t experts) {
    MatmulArgs a{};
    a.dtype = CQ_BF16;
    a.positions = a.tokens = static_cast<uint32_t>(positions);
    a.gated = gated;
    a.out_cols = static_cast<uint32_t>(out_cols);
    a.wide = gated ? 2 * a.out_cols : a.out_cols;
    a.cols = cols;
    a.bits = 2u << rand() % 3;
    a.block_cols = rand() % 4 ? 32u * (1 + rand() % 7) : 0;
    const uint32_t unit = a.block_cols ? 2 * a.block_cols : 64;  // whole blocks, and whole 16 bytes of 2-bit codes
    a.cols = (cols + unit - 1) / unit * unit;
    if (a.block_cols) a.block_rows = 1;
    a.row_bytes = a.cols * a.bits / 8ull;
    a.x_stride = a.cols;
    a.experts = experts ? experts : 1;
    if (experts) a.offsets = some_offsets;
    a.workspace_bytes = rand() % 2 ? 1ull << (10 + rand() % 22) : 0;
    return a;
}

int main() {
    srand(5);
    // a head of 128256 rows and of 151936, a projection of 28672, with prompts on both sides of what 2^22 workgroups of the smallest tile would hold
    const uint32_t heads[][2] = {{128256, 16384}, {128256, 17000}, {151936, 16384}, {28672, 74800}, {28672, 75000}, {28672, 1000000}, {1000000, 70000}};
    for (const auto& head : heads) {
        const MatmulArgs a = product(head[1], head[0], 4096, 0, 0);
        CHECK(tiles_take(a));
        CHECK(!matmul_choice(a).few && matmul_choice(a).tiles.shape == TilesShape::k256x128);
    }
    for (int n = 0; n < 200000; n++) {
        uint64_t positions, out_cols;
        const uint32_t gated = rand() % 2;
        do {  // results of up to 2^37 bytes
            positions = spread(28), out_cols = spread(26);
        } while (positions * out_cols > 1ull << 36);
        const MatmulArgs a = product(positions, out_cols, 512 + static_cast<uint32_t>(spread(14)), gated, rand() % 2 ? static_cast<uint32_t>(spread(11)) : 0);
        if (static_cast<uint64_t>(a.experts) * a.wide * a.row_bytes > 1ull << 38) continue;  // more than the card holds
        if (a.row_bytes >= (0xf0000000ull - a.row_bytes) / (256 + (gated ? a.out_cols : 0))) continue;  // distances within a tile: another limit
        CHECK(tiles_take(a));
        const MatmulChoice c = matmul_choice(a);
        CHECK(c.us < 1e30);
        if (c.few) {
            CHECK(c.few_shape.workgroups(a) < 1ull << 23 && most_tiles(a, c.few_shape.tokens_log2) <= 65535);
        } else {
            static const uint32_t rows[] = {256, 256, 128, 128, 32}, tokens[] = {128, 128, 64, 32, 32}, threads[] = {256, 512, 512, 512, 512};
            const int shape = static_cast<int>(c.tiles.shape);
            const TilesGrid g(a, rows[shape], tokens[shape], c.tiles.splits);
            const uint64_t each = static_cast<uint64_t>(g.group) * g.chunk, rectangles = (static_cast<uint64_t>(g.rectangles) + 7) / 8 * 8;
            CHECK(rectangles * each * threads[shape] < 1ull << 32);
            CHECK(static_cast<uint64_t>(g.rectangles) * each >= static_cast<uint64_t>(g.n_tiles) * g.p_tiles);
        }
    }
    {   // rows that overlap: the last one of a tile ends past 32 bits though their distances are within
        MatmulArgs a = product(4, 1000, 1u << 30, 0, 0);
        a.bits = 8, a.block_rows = a.block_cols = 0, a.cols = 1u << 30, a.row_bytes = 14u << 20, a.x_stride = 8;
        CHECK(!tiles_take(a));
        a.row_bytes = 4u << 20;
        CHECK(tiles_take(a));
    }
    // a block has at most 255 columns: up to 15 units of 16 bytes of codes, of which a row has fewer than 2^27
    const MatmulArgs a{};
    for (uint32_t each = 1; each <= 15; each++)
        for (uint32_t n = 0; n < 1u << 27; n += each * (n < 1u << 12 ? 1 : 4096))
            for (const uint32_t unit : {n, n + each - 1})
                if (unit < 1u << 27) CHECK(static_cast<uint32_t>((static_cast<uint64_t>(2u * unit) * magic_of(each)) >> 32) == unit / each);
    printf("ok\n");
    return 0;
}
