// lt_cut.h -- how attention's work is cut: the kernel that takes a sequence, grids,
// workspaces, parts and counters.  Arithmetic alone, for the host, the kernels
// (lt_attention.hip: few rows, lt_attention_wide.hip: many) and a test on the CPU.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define LT_CUT __host__ __device__ __forceinline__
#else
#define LT_CUT inline
#endif

namespace lt {

// Rows (tokens times heads of a group) of a sequence up to which lt_attention.hip's
// kernel takes it; the other kernel takes those with more.  Few-row and many-row kernel in us, a sequence of
// 512 rows over 4,000 keys: heads of 64 (2 groups of 7) 16 and 33, of 128 (4 of 8) 29 and 64, 192 (4 of 4) 42 and 62,
// 256 (8 of 2) 61 and 86, 512 (2 of 8) 50 and 93.  The many-row kernel's tiles of 64 to 256 rows pay with many
// sequences: 8 of them of 512 rows 40 and 49, 104 and 87, 166 and 161, 407 and 338, 195 and 232; of 1,024 rows 69 and
// 66, 190 and 157, 322 and 280, 816 and 697, 377 and 403 (one of 1,024: 20 and 35, 51 and 66, 49 and 75, 108 and 118,
// 95 and 106).  One border for all, between what a sequence alone and what many would have.
constexpr uint32_t kThinMost = 512;

// The tokens of a sequence that are served: beyond max_new, as many as the grid has room for (and those get NaN).
LT_CUT uint32_t cut_tokens(uint32_t n, uint32_t max_new) { return max_new && n > max_new ? max_new : n; }

// A sequence's tiles in either kernel; in one of the two none.
LT_CUT uint32_t cut_tiles(uint32_t rows, uint32_t of) { return (rows + of - 1) / of; }

// ------------------------------------------------------------------- few rows
constexpr uint32_t kThinRows = 16;
constexpr size_t kAttnTickets = 8192;  // words of counters

// Parts that a launch is cut into, about, and blocks a round of a workgroup, which are the least that a part has.
constexpr uint32_t thin_target(uint32_t D) { return D <= 128 ? 512 : 256; }
constexpr uint32_t thin_least(uint32_t D) { return D <= 256 ? 8 : 4; }

// Parts of a tile that are joined at once (or 8 for each time that the workgroup's threads
// are more than a part's places); more are joined in groups first, and no tile has more than
// the square (less one: 2^24 blocks times parts stay in 32 bits).
constexpr uint32_t kThinJoin = 16, kMostParts = kThinJoin * kThinJoin - 1;

LT_CUT uint32_t thin_row_tiles(uint32_t n, uint32_t group) {
    return n * group > kThinMost ? 0 : cut_tiles(n * group, kThinRows);
}

// Blocks a part: all of the batch's (sum) over the launch's workgroups, evenly.
LT_CUT uint32_t thin_share(float sum, uint32_t n_kv, uint32_t target, uint32_t least) {
    const float each = ceilf(sum * (float)n_kv / (float)target);
    return each < (float)least ? least : each > 1e9f ? 1000000000u : (uint32_t)each;
}

// A tile's parts.  None where a workgroup has its blocks done before parts are joined; parts of
// `least` where there are few, for their latency; else no more parts than the chip has room for at once.
LT_CUT uint32_t thin_splits(uint32_t blocks, uint32_t share, uint32_t least) {
    if (blocks <= 3 * least || share == 0xffffffffu) return 1;
    uint32_t n = share > least ? blocks / share : (blocks + share - 1) / share;
    if (n == 0) n = 1;
    return n < kMostParts ? n : kMostParts;
}

// Parts of a group that is joined in one go; hands: threads that a part's place has.
LT_CUT uint32_t thin_in_group(uint32_t splits, uint32_t hands) {
    return splits <= kThinJoin || splits <= 8 * hands ? splits : (uint32_t)ceilf(sqrtf((float)splits));
}

// Tiles of a batch, at most.
LT_CUT uint32_t thin_tiles(uint32_t n_tokens, uint32_t n_seqs, uint32_t max_new, uint32_t group) {
    const uint64_t rows = (uint64_t)n_tokens * group;
    uint64_t tiles = rows / kThinRows + n_seqs;
    const uint64_t each = max_new && (uint64_t)max_new * group < kThinMost ? max_new * group : kThinMost;
    const uint64_t most = (uint64_t)n_seqs * ((each + kThinRows - 1) / kThinRows);
    if (most < tiles) tiles = most;
    if (rows < tiles) tiles = rows;
    return (uint32_t)tiles;
}

// Workgroups of a head: the tiles, and the parts of those that are split (at most the
// target and one more a tile).
LT_CUT uint32_t thin_grid(uint32_t tiles, uint32_t max_blocks, uint32_t n_kv, uint32_t target, uint32_t least) {
    const uint32_t each = (max_blocks + least - 1) / least;  // (a tile's parts, at most)
    uint64_t x = tiles + target / n_kv + 1;
    if ((uint64_t)tiles * each < x) x = (uint64_t)tiles * each;
    return (uint32_t)x;
}

// Places for a head's parts; as many for groups of them.
LT_CUT uint32_t thin_slots(uint32_t target, uint32_t n_kv) { return 2 * (target / n_kv + 1) + 2; }

// Their bytes: 16 rows of D sums, then m, l, mo of each.
LT_CUT size_t thin_workspace(uint32_t D, uint32_t n_kv) {
    return (size_t)n_kv * 2 * thin_slots(thin_target(D), n_kv) * kThinRows * (D + 4) * 4;
}

// ------------------------------------------------------------------- many rows
constexpr uint32_t kLeast = 8;        // blocks that a workgroup is worth having for
constexpr uint32_t kMaxTiles = 1024;  // of a head, whose blocks are counted in LDS

// Whether a sequence of the batch may have rows for the many-row kernel: not where max_new allows them and the
// batch has too few tokens (wide_tiles would be 0, and a launch empty).
LT_CUT bool any_wide(uint32_t n_tokens, uint32_t max_new, uint32_t group) {
    return (uint64_t)cut_tokens(n_tokens, max_new) * group > kThinMost;
}

LT_CUT uint32_t wide_row_tiles(uint32_t n, uint32_t group, uint32_t tile) {
    return n * group > kThinMost ? cut_tiles(n * group, tile) : 0;
}

// Tiles of a batch, at most.
LT_CUT uint32_t wide_tiles(uint32_t n_tokens, uint32_t n_seqs, uint32_t max_new, uint32_t group, uint32_t tile) {
    const uint64_t rows = (uint64_t)n_tokens * group;
    const uint64_t most_rows = rows / (kThinMost + 1);  // (sequences that this kernel takes, at most)
    uint64_t tiles = rows / tile + (most_rows < n_seqs ? most_rows : n_seqs);
    if (max_new) {
        const uint64_t most = (uint64_t)n_seqs * (((uint64_t)max_new * group + tile - 1) / tile);
        if (most < tiles) tiles = most;
    }
    return (uint32_t)tiles;
}

// Workgroups that the tiles' blocks are cut for (fit: as many as the chip holds); 0: whole tiles, two and more
// for every place, which the hardware's order evens out, or too many to be counted in LDS.
LT_CUT uint32_t wide_pieces(uint32_t tiles, uint32_t n_seqs, uint32_t n_kv, uint32_t fit) {
    return (uint64_t)tiles * n_kv >= 2 * fit || tiles > kMaxTiles || n_seqs > kMaxTiles ? 0 : fit;
}

// Pieces that `total` blocks are really cut into.
LT_CUT uint32_t wide_cut(uint64_t total, uint32_t pieces) {
    const uint32_t n = total / kLeast < pieces ? (uint32_t)(total / kLeast) : pieces;
    return n ? n : 1;
}

}  // namespace lt
