// The grid of the products on the matrix cores: which tile a workgroup takes, and which shape of tile a launch.
#pragma once

#include "../../include/cubek_quant_device.hpp"
#include "cq_matmul_internal.hpp"

namespace cq {

enum class TilesShape { k256x128, k256x128x2, k128x64, k128x32, k32x32 };  // rows of W x positions; x2: by twice the waves, along the columns
struct TilesChoice {
    TilesShape shape;
    uint32_t splits;  // workgroups that share the columns of a tile
};

// kNT, kTT: tiles of 32 rows and of 32 positions of a wave; kWN, kWK: waves along rows and along columns; kLine: bytes of a row in a chunk of
// codes.
template <int kNT, int kTT, int kWN, int kWK, int kLine>
struct TilesTraits {
    static constexpr uint32_t kRows = 32 * kNT * kWN, kTokens = 32 * kTT;
    static constexpr uint32_t kXBytes = kTokens * 128, kCodeBytes = kRows * kLine, kScaleBytes = kRows * 8;  // a step of x; a chunk of codes; a step's scales
    static constexpr uint32_t kXRing = 2, kCodeRing = 2, kScaleRing = 4;          // images of a step's x, a chunk's codes and a step's scales
    static constexpr uint32_t kPitch = 32 * kNT + 4;                              // of the sums on their way to y
    static constexpr uint32_t kImage = kXRing * kXBytes + kCodeRing * kCodeBytes + kScaleRing * kScaleBytes, kImages = kWK * kImage, kParts = kWN * kWK * 32 * kPitch * 4;
    static constexpr uint32_t kLds = kImages > kParts ? kImages : kParts;
    static_assert(kLds <= 160 * 1024, "a compute unit's LDS");
    static constexpr uint32_t kWaves = kWN * kWK, kFit = 160 * 1024 / kLds;
    static constexpr uint32_t kMost = kNT * kTT >= 8 ? 2 : 4;  // waves of a SIMD that the registers of the sums leave room for
    static constexpr uint32_t kWavesPerSimd = kWaves / 4 * kFit < kMost ? kWaves / 4 * kFit : kMost;
};

// n / each as 2 n ceil(2^31 / each) / 2^32, for n < 2^27 and each <= 15: a scheme's blocks have at most 255 columns, 15 units of 16 bytes of 8-bit codes.
// 0 for each = 0, one scale for everything.
inline uint32_t magic_of(uint32_t each) { return each ? (0x80000000u + each - 1u) / each : 0u; }

// Tiles of `size` positions that a launch may be taken to have: the experts' sizes lie in device memory, and as many end in half a tile as in a whole one.
inline double likely_tiles(const MatmulArgs& a, uint32_t size) {
    if (!a.offsets) return static_cast<double>((a.positions + static_cast<uint64_t>(size) - 1) / size);
    const double experts = a.experts < a.positions ? a.experts : a.positions, each = a.positions / experts;
    return experts * (each > 0.5 * size ? each / size + 0.5 : 1.0);
}

struct TilesGrid {
    uint32_t n_tiles, p_tiles, splits, pitch;  // pitch: floats of a position's sums in the workspace
    uint32_t scale_size, scale_col_bytes, block_magic;

    // Workgroups go round the dies, which have an L2 each, one by one.  Tiles are dealt out in rectangles of `group` tiles of positions by
    // `chunk` of rows, whose workgroups read few rows of x and few of W at a time: as many to each die as to any other, the same rows to the
    // same die.  Of experts the host does not know how many tiles there are: a die may have a rectangle more than another.  Where its compute
    // units do not hold all of its workgroups at once, that is kept to a sixteenth of them, and the next rectangles go one die further on, as the
    // narrower ones at the rows' end would all come to the same dies (64 experts, 6126 positions, 11 tiles of rows: 204 -> 177 us; of fewer
    // workgroups the larger rectangles' shared reads count for more: 4 experts of 324 positions, [1360, 11104] 8 bits, 152 us, and 230 in single tiles).
    static constexpr uint32_t kDies = 8, kSlots = 64, kGroup = 4, kChunk = 8, kParts = 16;
    uint32_t group, chunk, rectangles, turn = 0;
    uint32_t group_width, wider_groups, chunk_width, wider_chunks;  // groups and chunks are as even as can be: the first ones a tile wider
    cubek_quant::device::FastDivmod by_rectangle, by_chunks, by_group;

    TilesGrid(const MatmulArgs& a, uint32_t rows, uint32_t tokens, uint32_t splits)
        : n_tiles((a.out_cols + (a.gated ? rows / 2 : rows) - 1) / (a.gated ? rows / 2 : rows)), p_tiles(static_cast<uint32_t>(most_tiles(a, __builtin_ctz(tokens)))),
          splits(splits), pitch(sums_pitch(a)), scale_size(a.param_dtype == CQ_F32 ? 4u : 2u), scale_col_bytes(static_cast<uint32_t>(a.scale_col * scale_size)),
          block_magic(magic_of(a.block_cols / 32u)) {
        uint32_t area = kGroup * kChunk, widest = kGroup, even = kDies;  // chunks come in multiples of `even`, so that all rectangles do in multiples of kDies
        const double likely = likely_tiles(a, tokens) * n_tiles;
        if (a.offsets && likely * splits > kDies * kSlots) {
            const double fits = likely / (kDies * kParts);
            if (fits < area) area = fits < 1.0 ? 1u : static_cast<uint32_t>(fits);
            while (widest > area) widest /= 2;
            even = 1, turn = 1;
        }
        const uint32_t groups = (p_tiles + widest - 1) / widest;
        group = a.offsets ? (p_tiles < widest ? p_tiles : widest) : (p_tiles + groups - 1) / groups;
        group_width = a.offsets ? group : p_tiles / groups, wider_groups = a.offsets ? 0 : p_tiles % groups;
        const uint32_t most = area / group;
        while (even > 1 && groups % (kDies / even * 2) == 0) even /= 2;
        uint32_t chunks = ((n_tiles + most - 1) / most + even - 1) / even * even;
        if (chunks > n_tiles) chunks = n_tiles;
        chunk = (n_tiles + chunks - 1) / chunks, chunk_width = n_tiles / chunks, wider_chunks = n_tiles % chunks;
        rectangles = groups * chunks;
        by_rectangle = cubek_quant::device::FastDivmod(group * chunk);
        by_chunks = cubek_quant::device::FastDivmod(chunks);
        by_group = cubek_quant::device::FastDivmod(group);
    }

    __device__ uint32_t block_of(uint32_t half) const { return __umulhi(2u * half, block_magic); }
    uint32_t workgroups() const { return (rectangles + kDies - 1) / kDies * kDies * group * chunk; }

    // Floats of a position's sums: whole eights of columns, gated two of them.
    static uint32_t sums_pitch(const MatmulArgs& a) { return (a.out_cols + 7u) / 8u * 8u * (a.gated ? 2u : 1u); }

    // false: a workgroup beyond the last tile
    __device__ bool tile(uint32_t block, uint32_t* n, uint32_t* p) const {
        uint32_t round, within, p_group, n_chunk, in_chunk, in_group;
        by_rectangle.div_mod(block / kDies, &round, &within);
        by_chunks.div_mod(round * kDies + (block + round * turn) % kDies, &p_group, &n_chunk);
        by_group.div_mod(within, &in_chunk, &in_group);
        *n = n_chunk * chunk_width + min(n_chunk, wider_chunks) + in_chunk;
        *p = p_group * group_width + min(p_group, wider_groups) + in_group;
        return in_chunk < chunk_width + (n_chunk < wider_chunks) && in_group < group_width + (p_group < wider_groups) && *p < p_tiles;
    }
};

// Whether one launch holds the workgroups of a shape of tile.  Along each side less than half of a rectangle's places are empty, and seven rectangles may be.
inline bool tiles_fit(const MatmulArgs& a, uint32_t rows, uint32_t tokens, uint32_t threads, uint32_t splits) {
    const uint32_t columns = a.gated ? rows / 2 : rows;
    const uint64_t most = kLaunchThreads / threads, p_tiles = most_tiles(a, __builtin_ctz(tokens)), n_tiles = (a.out_cols + columns - 1) / columns;
    if (p_tiles >= most || n_tiles * p_tiles >= most) return false;
    return 4 * n_tiles * p_tiles + TilesGrid::kDies * TilesGrid::kGroup * TilesGrid::kChunk < most || TilesGrid(a, rows, tokens, splits).workgroups() < most;
}

// The kernel of a decode step (cq_kernels_matmul_few.hip): stages that a wave's loads are ahead.
constexpr uint32_t kFewAhead = 1;
// units: of 16 bytes of codes of a row in a stage, 8 for a line or 4 for half of one.  x of 32 positions or of 2-bit codes is so large that a compute
// unit would hold one workgroup of whole lines (32 positions [4096, 14336] 4 bits 35.5 -> 22.0 us, one position [8192, 8192] 2 bits 12.4 -> 10.0);
// otherwise halves leave room for more workgroups on a compute unit, whole lines are read faster ([28672, 8192] 4 bits, one position,
// 36.6 us and 40.8 in halves; eight experts [28672, 4096] gated, 32 positions, 153 us and 127 in halves).
struct FewShape {
    uint32_t groups, tokens_log2, shares_log2, units;  // groups of 16 rows of a wave; positions of a tile; shares of a row's columns; units of a stage
    uint32_t x_bytes;                                  // of a stage: whole loads of 1 KiB

    uint32_t x_loads() const { return (x_bytes / 1024 + (8 >> shares_log2) - 1) / (8 >> shares_log2); }  // of a wave
    uint32_t workgroups(const MatmulArgs& a) const {  // of a tile of positions
        const uint32_t columns = (8u >> shares_log2) * (a.gated ? 8u : 16u) * groups;
        return (a.out_cols + columns - 1) / columns;
    }
    uint32_t lds() const {
        const uint32_t images = (kFewAhead + 1) * ((x_bytes << shares_log2) + 8 * groups * 16 * units * 20);
        const uint32_t sums = 8 * groups * (tokens_log2 == 5 ? 2048u : 1024u);
        return images > sums ? images : sums;
    }
};

struct FewGrid {
    uint32_t shares_log2, tokens_log2, x_bytes, scale_size, scale_col_bytes, block_magic;

    FewGrid(const MatmulArgs& a, const FewShape& c)
        : shares_log2(c.shares_log2), tokens_log2(c.tokens_log2), x_bytes(c.x_bytes), scale_size(a.param_dtype == CQ_F32 ? 4u : 2u),
          scale_col_bytes(static_cast<uint32_t>(a.scale_col * scale_size)), block_magic(magic_of(a.block_cols * a.bits / 128)) {}
    __device__ uint32_t block_of(uint32_t unit) const { return __umulhi(2u * unit, block_magic); }
};

// Whether the kernels on the matrix cores take a product: 16-bit x, rows of whole 16-byte pieces on boundaries of 16 bytes, scales that serve
// 32 columns at least, and distances within a tile that fit 32 bits: half of a gated weight, and x where rows of it are picked, below 3.75 GiB.
inline bool tiles_take(const MatmulArgs& a) {
    const auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const uint64_t scale_size = a.param_dtype == CQ_F32 ? 4 : 2, rows = 256 + (a.gated ? a.out_cols : 0);
    const uint64_t x_rows = a.row_of ? a.tokens : 256, row = static_cast<uint64_t>(a.cols) * a.bits / 8;  // (rows of codes may overlap)
    constexpr uint64_t kFits = 0xf0000000ull;
    if (a.dtype == CQ_F32 || a.cols == 0 || a.cols % 32 || static_cast<uint64_t>(a.cols) * a.bits % 128 || a.block_cols % 32) return false;
    if (!on16(a.words) || !on16(a.x) || a.row_bytes % 16 || a.expert_bytes % 16 || a.x_stride % 8) return false;
    if (a.row_bytes >= (kFits - row) / rows || a.x_stride * 2 >= kFits / x_rows) return false;
    if (a.block_rows && (a.scale_row >= kFits / scale_size / 4 / (rows / a.block_rows + 2) ||
                         a.scale_col >= kFits / scale_size / 4 / (a.cols / a.block_cols + 1)))
        return false;
    return tiles_fit(a, 256, 128, 256, 1);  // the largest tiles; smaller ones are left out where a launch does not hold theirs
}

inline uint64_t sums_bytes(const MatmulArgs& a, uint32_t splits) { return splits > 1 ? 4ull * splits * a.positions * TilesGrid::sums_pitch(a) : 0; }

// Which kernel a product takes, by what it would take.  Times in microseconds, fitted to sweeps over shapes, splits and 1 to 2048 positions
// (blocks of 32, bf16; f16 and the other codes of a width alike): a launch is its rounds of steps, and a round costs little less when half
// of a compute unit's workgroups are there.  Measured against the model: [28672, 8192] 4 bits, tiles of 256 x 128, 2048 positions 833 us for 850,
// 1024 450 for 468, 128 in four parts 91 for 88; [4096, 4096] 512 positions, 256 x 128 in four parts 39.3 for 38.8, 128 x 64 in two 37.6 for 40.2;
// 128 positions, 128 x 64 in four parts 21.7 for 20.0, 32 x 32 23.7 for 22.4; a decode step of 16 on [28672, 8192] 36.3 for 36.
struct MatmulChoice {
    bool few = false;
    FewShape few_shape{};
    TilesChoice tiles{TilesShape::k256x128, 1};
    double us = 1e30;
};

// What `workgroups` take for a round of steps that takes `half` with one workgroup on a compute unit and `full` with two.
inline double rounds_us(double workgroups, double half, double full) {
    const double whole = static_cast<double>(static_cast<uint64_t>(workgroups / 512.0)), rest = workgroups - 512.0 * whole;
    return whole * full + (rest <= 0.0 ? 0.0 : rest <= 256.0 ? half : full);
}

// Experts of unlike sizes have more tiles than as many of the same size, though never more than one that is not full for each.
inline double uneven_tiles(const MatmulArgs& a, uint32_t size, double more) {
    const double likely = likely_tiles(a, size);
    if (!a.offsets) return likely;
    const double most = static_cast<double>(a.positions / size + (a.experts < a.positions ? a.experts : a.positions));
    return likely * more < most ? likely * more : most;
}

inline void consider_tiles(const MatmulArgs& a, TilesShape shape, uint32_t rows, uint32_t tokens, uint32_t along, uint32_t line, double start, double half, double full,
                           uint64_t room, MatmulChoice* best) {
    const uint32_t threads = (rows >= 128 ? 256 : 64) * along;
    const uint32_t columns = a.gated ? rows / 2 : rows, steps = line / 8 / a.bits, chunks = ((a.cols + 63) / 64 + steps - 1) / steps;
    const double row_tiles = (a.out_cols + columns - 1) / columns, tiles = row_tiles * uneven_tiles(a, tokens, 1.0), more = row_tiles * uneven_tiles(a, tokens, 1.25);
    // weights that only one or two tiles of positions share come from memory, later than out of the L2
    const double wait = a.offsets ? (rows == 256 ? 1.15 : rows == 32 ? 1.1 : tokens == 32 ? 1.2 : 1.0) : a.positions <= 32 ? 1.3 : 1.0;
    for (uint32_t splits = 1; splits <= 16; splits *= 2) {
        if (splits > 1 && (splits * along > chunks || sums_bytes(a, splits) > room)) break;
        if (!tiles_fit(a, rows, tokens, threads, splits)) break;
        const double rounds = static_cast<double>((chunks + splits * along - 1) / (splits * along) * steps);
        const double sums = splits > 1 ? 3.0 + 2.0 * static_cast<double>(sums_bytes(a, splits)) / 5e6 : 0.0;  // written and read at 5 TB/s
        const double us = (start + rounds * 0.5 * (rounds_us(tiles * splits, half, full) + rounds_us(more * splits, half, full))) * wait + sums;
        if (us < best->us * (splits > 1 ? 0.92 : 1.0)) {  // (workgroups of many rounds do not wait for one another)
            best->few = false;
            best->tiles = TilesChoice{shape, splits};
            best->us = us;
        }
    }
}

// The kernel of a decode step, where a unit of 16 bytes of codes has one scale: `round` is what a stage takes with one workgroup on a compute unit,
// every further one adds 0.45 of it, as many as LDS holds, up to four.  Fitted to 170 random products of up to 40 positions or experts of up to
// 400 each, for which every kernel was timed: what the model takes is 1.04 times the fastest in the geometric mean (70 positions of 16 experts,
// [5468, 3936] e2m1 gated 57 us, and 91 by whole lines).
inline void consider_few(const MatmulArgs& a, MatmulChoice* best) {
    const uint32_t unit = 128 / a.bits;
    if (a.block_cols % unit) return;
    const double experts = a.offsets ? (a.experts < a.positions ? a.experts : a.positions) : 1;
    const double read = experts * a.wide * a.cols * a.bits / 8 / 4.5e6;  // halves of lines at 4.5 TB/s
    for (uint32_t way = 0; way < 5; way++) {
        FewShape c{};
        c.tokens_log2 = way < 3 ? 3 + way : way, c.units = way < 2 ? 8 : 4;  // 8 and 16 positions by whole lines, 32, 8 and 16 by halves
        if (c.units == 8 && a.bits == 2) continue;
        const uint32_t most = 1u << c.tokens_log2, tokens = a.positions < most ? a.positions : most, columns = c.units * unit;
        const uint32_t stages = (a.cols / unit + c.units - 1) / c.units;
        // every further tile of positions reads the weights again: of experts as many have one more as one less
        if (a.positions > (a.offsets ? 1.5 * most * a.experts : most) || most_tiles(a, c.tokens_log2) > 65535) continue;
        c.x_bytes = (tokens * (columns * 2) + 1023) / 1024 * 1024;
        c.groups = a.gated ? 2 : 1;
        const double round = (c.tokens_log2 == 5 ? 0.35 + 0.0055 * columns : c.units == 8 ? 0.6 + 0.0031 * columns : c.tokens_log2 == 4 ? 0.4 + 0.0022 * columns : 0.45 + 0.0025 * columns) *
                             (c.groups == 2 ? 1.7 : 1.0);
        for (c.shares_log2 = 0; c.shares_log2 <= 3; c.shares_log2++) {
            if (c.shares_log2 && (1u << c.shares_log2) > stages) break;
            if (c.lds() > 160 * 1024 || c.x_loads() > 8) continue;
            if (c.workgroups(a) >= kLaunchThreads / 512) continue;
            const uint32_t held = 160 * 1024 / c.lds(), fit = held < 4 ? held : 4;
            const double stages_each = (stages + (1u << c.shares_log2) - 1) >> c.shares_log2;
            double us = 0.0;
            for (const double more : {1.0, 1.25}) {
                const double workgroups = (a.out_cols + 15) / 16 * uneven_tiles(a, most, more) * (1u << c.shares_log2) / 8;
                const double whole = static_cast<double>(static_cast<uint64_t>(workgroups / (256.0 * fit))), rest = (workgroups - whole * 256.0 * fit) / 256.0;
                us += 0.5 * round * (whole * (1.0 + 0.45 * (fit - 1)) + (rest <= 0.0 ? 0.0 : rest <= 1.0 ? 1.0 : rest <= 2.0 ? 1.45 : rest <= 3.0 ? 1.9 : 2.35));
            }
            us *= stages_each;
            if (c.units == 4 && us < read) us = read;
            if (a.offsets && c.tokens_log2 == 5) us *= 1.1;
            us += 2.5 + 0.5 * c.shares_log2;
            if (us < best->us) {
                best->few = true;
                best->few_shape = c;
                best->us = us;
            }
        }
    }
}

// The fastest within `room` bytes of workspace.
inline MatmulChoice choice_within(const MatmulArgs& a, uint64_t room) {
    MatmulChoice c;
    consider_few(a, &c);
    // start: a launch without its rounds, from the first loads to the last sums
    consider_tiles(a, TilesShape::k256x128, 256, 128, 1, 64, 6.0, 1.05, 1.75, room, &c);
    consider_tiles(a, TilesShape::k256x128x2, 256, 128, 2, 64, 9.0, 1.85, 3.7, room, &c);
    consider_tiles(a, TilesShape::k128x64, 128, 64, 2, 64, 5.0, 1.15, 1.65, room, &c);
    consider_tiles(a, TilesShape::k128x32, 128, 32, 2, 64, 4.5, 1.1, 1.75, room, &c);
    consider_tiles(a, TilesShape::k32x32, 32, 32, 8, 128, 4.0, 1.15, 2.3, room, &c);
    return c;
}

inline uint64_t room_of(const MatmulArgs& a, const MatmulChoice& c) { return c.few ? 0 : sums_bytes(a, c.tiles.splits); }

// The fastest of all where its sums find room, so that a workspace of the size that was asked for gives the kernel it was asked for: within that room alone
// another one may come out, as a smaller one in front of it sets another mark.
inline MatmulChoice matmul_choice(const MatmulArgs& a) {
    const MatmulChoice c = choice_within(a, ~0ull);
    return room_of(a, c) <= a.workspace_bytes ? c : choice_within(a, a.workspace_bytes);
}

hipError_t launch_matmul_finish(hipStream_t s, const MatmulArgs& a, uint32_t splits);
hipError_t launch_matmul_tiles(hipStream_t s, const MatmulArgs& a);

#define CQ_TILES_CODES(X, f) X(f, 2) X(f, 4) X(f, 8) X(f, 100) X(f, 101) X(f, 102)
#define CQ_TILES_DECLARE(f, c)                                                              \
    hipError_t matmul_tiles_##f##_##c(hipStream_t s, const MatmulArgs& a, const TilesChoice& choice); \
    hipError_t matmul_few_##f##_##c(hipStream_t s, const MatmulArgs& a, const FewShape& shape);
CQ_TILES_CODES(CQ_TILES_DECLARE, BF16)
CQ_TILES_CODES(CQ_TILES_DECLARE, F16)

}  // namespace cq
