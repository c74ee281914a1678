// How attention's work is cut (csrc/lt_cut.h, the functions that its launches and kernels use): every block of every
// sequence once, as many workgroups, places and counters as there are.  CPU only.
#include "lt_cut.h"

#include <stdio.h>

#include <algorithm>
#include <random>
#include <string>
#include <vector>

using namespace lt;

static int failures = 0;
static std::string where;
#define CHECK(x)                                                                        \
    do {                                                                                \
        if (!(x)) {                                                                     \
            if (failures++ < 20) printf("FAILED %s: %s (line %d)\n", where.c_str(), #x, __LINE__); \
        }                                                                               \
    } while (0)

static std::mt19937_64 rng(7);
static uint32_t pick(uint32_t lo, uint32_t hi) { return lo + (uint32_t)(rng() % (hi - lo + 1)); }
static uint32_t pick_log(uint32_t lo, uint32_t hi) {
    const double u = (double)(rng() >> 11) / 9007199254740992.0;
    return std::min(hi, std::max(lo, (uint32_t)llround(exp(log((double)lo) + u * (log((double)hi) - log((double)lo))))));
}

struct Seq {
    uint32_t n, len;
};
struct Batch {
    std::vector<Seq> seqs;
    uint32_t n_tokens = 0, max_new = 0, max_blocks = 1, n_kv = 1, group = 1, window = 0;
};

// A sequence's blocks in sight, as the kernels count them.
static uint32_t blocks_of(const Batch &b, const Seq &s) {
    if (!s.n) return 1;
    const uint32_t begin = s.len - s.n;
    const uint32_t lo = b.window && begin + 1 > b.window ? (begin + 1 - b.window) / 32 : 0;
    return (s.len - 1) / 32 + 1 - lo;
}

static Batch draw() {
    Batch b;
    const uint32_t seqs = pick_log(1, 4096), most = pick_log(1, pick(0, 3) ? 40 : 3000), past = pick_log(1, 200000);
    const bool sparse = pick(0, 2) == 0, rare = pick(0, 3) == 0;  // (rare: a few tokens of all the sequences)
    uint32_t top = 0;
    for (uint32_t i = 0; i < seqs; i++) {
        const uint32_t n = (rare && pick(0, seqs) > 3) || (sparse && pick(0, 9)) ? 0 : pick(0, most);
        b.seqs.push_back({n, n + pick(0, past)});
        b.n_tokens += n;
        top = std::max(top, n);
        b.max_blocks = std::max(b.max_blocks, (b.seqs.back().len + 31) / 32);
    }
    b.n_tokens += pick(0, 3);
    b.max_blocks += pick(0, 5);
    const uint32_t kinds[] = {0, top, top + pick_log(1, 1u << 23)};
    b.max_new = kinds[pick(0, 2)];
    const uint32_t heads[] = {1, 2, 3, 4, 8, 17, 64, 256}, groups[] = {1, 2, 3, 7, 8, 16, 128};
    b.n_kv = heads[pick(0, 7)], b.group = groups[pick(0, 6)];
    b.window = pick(0, 2) ? 0 : pick_log(1, 5000);
    where = std::to_string(seqs) + " sequences, " + std::to_string(b.n_tokens) + " tokens, max_new " + std::to_string(b.max_new) +
            ", " + std::to_string(b.n_kv) + " x " + std::to_string(b.group) + " heads";
    return b;
}

// Few rows: the workgroups that the sequences take against the grid, places of parts and counters.
static void few(const Batch &b, uint32_t D) {
    const uint32_t target = thin_target(D), least = thin_least(D);
    float sum = 0;
    for (const Seq &s : b.seqs) sum += (float)thin_row_tiles(cut_tokens(s.n, b.max_new), b.group) * (float)blocks_of(b, s);
    const uint32_t share = thin_share(sum, b.n_kv, target, least);
    const uint32_t tiles = thin_tiles(b.n_tokens, (uint32_t)b.seqs.size(), b.max_new, b.group);
    const uint32_t grid = thin_grid(tiles, b.max_blocks, b.n_kv, target, least), slots = thin_slots(target, b.n_kv);
    uint64_t work = 0, parts = 0;
    for (const Seq &s : b.seqs) {
        const uint32_t n = thin_row_tiles(cut_tokens(s.n, b.max_new), b.group), blocks = blocks_of(b, s);
        const uint32_t splits = thin_splits(blocks, share, least);
        work += (uint64_t)n * splits;
        if (splits > 1) parts += (uint64_t)n * splits;
        for (uint32_t i = 0, at = 0; i < splits; i++) {
            const uint64_t b0 = (uint64_t)blocks * i / splits, b1 = (uint64_t)blocks * (i + 1) / splits;
            CHECK(b0 == at && (b1 > b0));
            CHECK((uint64_t)blocks * (i + 1) < 1ull << 32);  // (the kernel's 32 bits)
            at = (uint32_t)b1;
        }
        for (uint32_t hands : {1u, 2u, 4u, 32u}) {
            const uint32_t each = thin_in_group(splits, hands), groups = (splits + each - 1) / each;
            CHECK(each >= 1 && groups <= std::max(1u, kThinJoin));
        }
    }
    CHECK(work <= grid);
    CHECK(parts <= slots);
    CHECK((uint64_t)2 * slots * b.n_kv <= kAttnTickets);
    // (two places a slot, of which the kernel's last float is in 32 bits of bytes; no more than this head size's parts need)
    const uint64_t bytes = thin_workspace(D, b.n_kv), part = 16 * (D + 4) * 4;
    CHECK(bytes >= 2 * part * slots * b.n_kv && bytes < 1ull << 32);
    CHECK(bytes <= 2 * part * (2 * target + 4 * b.n_kv));
    // (no launch without a workgroup)
    CHECK(!b.n_tokens || grid > 0);
}

// Many rows.
static void many(const Batch &b, uint32_t tile, uint32_t per_cu) {
    const uint32_t seqs = (uint32_t)b.seqs.size(), fit = 256 * per_cu;
    std::vector<uint32_t> tiles;  // blocks of each
    for (const Seq &s : b.seqs) {
        const uint32_t n = cut_tokens(s.n, b.max_new), t = wide_row_tiles(n, b.group, tile);
        CHECK((t == 0) == (n * b.group <= kThinMost));
        for (uint32_t i = 0; i < t; i++) {
            const uint32_t begin = s.len - s.n, r1 = std::min(n * b.group, (i + 1) * tile) - 1;
            const uint32_t pos0 = begin + i * tile / b.group, pos1 = begin + r1 / b.group;
            const uint32_t lo = b.window && pos0 + 1 > b.window ? (pos0 + 1 - b.window) / 32 : 0;
            tiles.push_back(pos1 / 32 + 1 - lo);
        }
    }
    if (!any_wide(b.n_tokens, b.max_new, b.group)) {
        CHECK(tiles.empty());
        return;
    }
    const uint32_t room = wide_tiles(b.n_tokens, seqs, b.max_new, b.group, tile);
    CHECK(tiles.size() <= room);
    const uint32_t pieces = wide_pieces(room, seqs, b.n_kv, fit);
    CHECK(pieces || (uint64_t)room * b.n_kv > 0);  // (no launch without a workgroup)
    if (!pieces) return;
    CHECK(room <= kMaxTiles && seqs <= kMaxTiles && 3 * pieces <= kAttnTickets);
    uint64_t line = 0;
    std::vector<uint64_t> firsts;
    for (uint32_t t : tiles) firsts.push_back(line), line += t;
    const uint64_t total = line * b.n_kv;
    if (!total) return;
    const uint32_t cut = wide_cut(total, pieces);
    CHECK(cut >= 1 && cut <= pieces);
    for (uint32_t p = 0; p < cut; p++) CHECK(total * p / cut < total * (p + 1) / cut);
}

int main() {
    const struct { uint32_t tile, per_cu; } wide[] = {{128, 3}, {256, 1}, {64, 2}, {128, 1}, {64, 1}};
    for (int i = 0; i < 3000; i++) {
        const Batch b = draw();
        for (uint32_t D : {64u, 96u, 128u, 192u, 256u, 512u}) few(b, D);
        for (const auto &w : wide) many(b, w.tile, w.per_cu);
    }
    printf(failures ? "%d FAILED\n" : "ALL PASSED\n", failures);
    return failures != 0;
}
