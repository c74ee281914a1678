// lt_attention.hip -- attention over the 8-bit cache (lt_kv.h).
//
//   out = softmax(scale * q k^T) v   over the keys at positions max(0, p - window + 1) .. p
//
// for the queries at position p of every head; the heads of a group share a key
// and value head.
//
// A tile of 16 rows (tokens and heads of one group, of one sequence) is one
// operand of v_mfma_f32_16x16x32_f16, a block's codes the other.  Codes are
// exact in f16; queries and softmax weights go in as two f16 parts each (22 bits,
// the last half step 2^-23 of the largest), so a product keeps fp32's accuracy:
//   S^T [32 keys x 16 rows] = K q^T,   O^T [D x 16 rows] += V^T P^T
// S^T leaves its results where P^T is read, so the weights never leave the lane
// that made them; a lane holds 8 keys of one row.
//
// The softmax runs along: m is the largest logit so far (base 2), l the sum of
// 2^(s - m).  A block's value scale meets the weights, not the sums: with mo the
// largest of (block's largest logit + log2(scale)) so far, the weights are
// 2^(s + log2(scale) - mo), times 2^kBits to use f16's range; their sum
// times 2^(mo - log2(scale) - m) goes to l.  (Both are followed with some slack.)  (Two maxima, because a block of small
// values may have the largest logit.)
//
// Work: a sequence's tiles are cut along the keys into parts of about the same
// number of blocks, as many as fill the chip; the part that arrives last at a
// tile joins them.
//
// Bound by memory where the cache is large (48 sequences' caches of 220 MB: 54 us, 4.1 TB/s; one of 134 MB: 37 us, or 32
// where the last call's keys are still in the chip's last cache, of which the loads take 18 and the two rounds of
// joining 7); else by instructions (a block of heads of 64
// takes a wavefront about 250, of 128 400, of 256 650, 4 cycles each) and the chain of one launch: one
// token of 14 heads over 1,500 keys 7.6 us, of which lengths 1.3, table 0.7, queries 0.6, codes 0.9, products and the
// wavefronts' sums 1.5, arrival 0.9, joining 1.6 (taken with integer divisions in lengths, queries and joining; 0.35 less
// without: a graph of 12 layers 107.5 -> 103.2).
#include "llmtoy_hip.h"
#include "lt_attn.h"

namespace lt {

namespace {

// Wavefronts a workgroup, wavefronts that a block's channels are cut over, parts that a
// launch is cut into (more of them: 48 heads' caches of 220 MB 61.5 us with 512, 64 with 1,024; fewer:
// 79 with 256, whose workgroups leave half of the registers unused).
template <int D>
struct Shape {
    static constexpr int kWaves = 8, kSplit = D <= 256 ? 1 : 2, kTarget = thin_target(D);
    static constexpr int kThreads = kWaves * kWave, kBlocks = kWaves / kSplit;  // blocks a round
    static constexpr int DW = D / kSplit, C = DW / 32;
    static_assert(kBlocks == (int)thin_least(D), "");
    // (what a wavefront would not have the registers for: four on a SIMD up to heads of 128, then two)
    static constexpr bool kQueriesInLds = DW >= 128;
};

struct ThinArgs {
    const uint8_t *codes;
    const float2 *scales;
    uint32_t n_blocks, n_kv;
    KvBatchDev b;
    const float *q;
    float *out;
    size_t q_stride;
    uint32_t n_heads, group, window;
    float scale2;  // scale * log2(e)
    float per_group;  // 1 / group
    float *part;        // [n_kv][2][slots] of parts and of groups of them: [16][D] sums, then [16][4] m, l, mo
    uint32_t *tickets;  // [n_kv][slots][2]: groups, tiles; zero between launches
    uint32_t slots, target;  // parts of all heads that the work is cut into, about
    uint32_t least;          // blocks a part, at least
    uint32_t *err;
};

// How a sequence's rows are cut: `tiles` tiles of 16 rows, over the blocks lo ..
// lo + blocks - 1.
struct ThinRow {
    KvRow k;
    uint32_t tiles, lo, blocks;
};

__device__ __forceinline__ ThinRow thin_row(const ThinArgs &a, uint32_t r) {
    ThinRow t;
    t.k = kv_row_of(a.b, r);
    t.k.n = cut_tokens(t.k.n, a.b.max_new);
    t.tiles = thin_row_tiles(t.k.n, a.group);
    t.lo = 0;
    t.blocks = 1;
    if (!t.k.bad && t.k.n) {
        const uint32_t begin = t.k.len - t.k.n;
        if (a.window && begin + 1 > a.window) t.lo = (begin + 1 - a.window) / kKvBlock;
        t.blocks = (t.k.len - 1) / kKvBlock + 1 - t.lo;
    }
    return t;
}

// What workgroup `index` of a head takes: blocks b0 .. b1 - 1 for a tile of a
// row, as part `split` of `splits`; its place among the parts that are joined.
struct ThinWork {
    uint32_t row, tile, split, splits, b0, b1, slot;
    uint32_t first, n, len;
    bool any, bad;
};

// Every wavefront finds its work for itself from the lengths (one load and two sums for
// up to 64 sequences).
__device__ __forceinline__ ThinWork thin_work(const ThinArgs &a, uint32_t index) {
    ThinWork w{};
    const uint32_t lane = threadIdx.x % kWave;
    float sum = 0.0f;  // (a count beyond 2^24 need not be exact)
    bool falls = false;
    ThinRow t{};
    for (uint32_t r0 = 0; r0 < a.b.n_seqs; r0 += kWave) {
        const uint32_t r = r0 + lane;
        if (r >= a.b.n_seqs) break;
        t = thin_row(a, r);
        if ((t.k.falls || t.k.behind) && blockIdx.x == 0 && blockIdx.y == 0) kv_report(a.err, kKvErrRows, r);
        falls |= t.k.falls;
        sum += (float)t.tiles * (float)t.blocks;
    }
    if (a.b.n_seqs > 1) {
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    } else {
        sum = __uint_as_float(from_lane(__float_as_uint(sum), 0));
    }
    // (where start falls, sequences may overlap and have more tiles than the grid has workgroups for: whole
    // tiles, so that none waits for a part that nobody takes)
    const uint32_t share = __any(falls) ? 0xffffffffu : thin_share(sum, a.n_kv, a.target, a.least);
    uint32_t seen = 0, joined = 0;  // workgroups and joined parts of the rows before
    for (uint32_t r0 = 0; r0 < a.b.n_seqs; r0 += kWave) {
        const uint32_t r = r0 + lane;
        uint32_t splits = 0;
        if (a.b.n_seqs > kWave) t = r < a.b.n_seqs ? thin_row(a, r) : ThinRow{};
        if (r < a.b.n_seqs) {
            splits = thin_splits(t.blocks, share, a.least);
        }
        const uint32_t mine = t.tiles * splits, parts = splits > 1 ? mine : 0;
        uint32_t up = mine, pup = parts;
        if (a.b.n_seqs > 1) {
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const uint32_t p = __shfl_up(up, off, kWave), q = __shfl_up(pup, off, kWave);
                if ((int)lane >= off) up += p, pup += q;
            }
        }
        const uint32_t before = seen + up - mine;
        const uint64_t has = __ballot(index >= before && index < before + mine);
        if (has) {
            const int l = __builtin_ctzll(has);
            const uint32_t in = index - from_lane(before, l);
            w.any = true;
            w.row = r0 + l;
            w.splits = from_lane(splits, l);
            w.tile = w.splits == 1 ? in : in / w.splits;
            w.split = in - w.tile * w.splits;
            const uint32_t lo = from_lane(t.lo, l), blocks = from_lane(t.blocks, l);
            // as even as whole blocks go
            w.b0 = lo + (w.splits == 1 ? 0 : blocks * w.split / w.splits);
            w.b1 = lo + (w.splits == 1 ? blocks : blocks * (w.split + 1) / w.splits);
            w.slot = joined + from_lane(pup - parts, l) + in;
            w.first = from_lane(t.k.first, l), w.n = from_lane(t.k.n, l), w.len = from_lane(t.k.len, l);
            w.bad = from_lane(t.k.bad, l);
            return w;
        }
        seen += from_lane(up, kWave - 1);
        joined += from_lane(pup, kWave - 1);
    }
    return w;
}

// A row's token, among its sequence's.  (row + 1/2) / group is 1 / (2 group) from a whole number at
// least, and the product is off by (row + 1/2) / group * 2^-23 at most: exact for rows below 2^22, where
// kThinMost and a tile are the most.  (A quotient of integers takes some 20 instructions.)
__device__ __forceinline__ uint32_t token_of(const ThinArgs &a, uint32_t row) {
    return (uint32_t)(((float)row + 0.5f) * a.per_group);
}

// The largest of the four lanes that share a row.
__device__ __forceinline__ float row_max(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// Sums of parts and what they are sums to.
struct Joint {
    f32x4 sum;
    float m, l, mo;
    __device__ __forceinline__ void clear() { sum = f32x4{0, 0, 0, 0}, m = kNegInf, mo = kNegInf, l = 0.0f; }
    // `count` parts more (N at most): their m, l, mo and sums
    template <int N>
    __device__ __forceinline__ void add(const f32x4 (&st)[N], const f32x4 (&v)[N], uint32_t count) {
        float m1 = m, mo1 = mo;
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (i < count) m1 = fmaxf(m1, st[i][0]), mo1 = fmaxf(mo1, st[i][2]);
        l *= m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - m1);  // (l is 0 or NaN without a largest)
        sum *= mo == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mo - mo1);  // (sums of 0 or NaN)
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (i < count) {
                l += st[i][0] == kNegInf ? st[i][1] : st[i][1] * __builtin_amdgcn_exp2f(st[i][0] - m1);
                sum += v[i] * (st[i][2] == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(st[i][2] - mo1));
            }
        m = m1, mo = mo1;
    }
};

template <int D>
__global__ __launch_bounds__(Shape<D>::kThreads, (D <= 128 ? 4 : 2)) void k_attention_thin(ThinArgs a) {
    using Sh = Shape<D>;
    constexpr int W = Sh::kWaves, C = Sh::C, NT = Sh::kThreads, SPLIT = Sh::kSplit, NB = Sh::kBlocks;
    constexpr bool kQueriesInLds = Sh::kQueriesInLds;
    constexpr uint32_t kBatch = D <= 128 ? 8 : 16;  // parts that a thread reads at once
    constexpr uint32_t P = kThinRows * (D + 4);  // floats of a part
    // the wavefronts' sums; the queries lie there before, where they are in LDS
    __shared__ __align__(16) float s_o[NB][kThinRows][D + 4];
    __shared__ f32x4 s_m[NB][kThinRows];
    __shared__ float s_top[SPLIT > 1 ? W : 1][kThinRows];
    __shared__ uint32_t s_last;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, g = lane / 16, n = lane % 16;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / kWave), h = blockIdx.y;
    const uint32_t cut = wave % SPLIT, which = wave / SPLIT;  // channels, block of a round
    const ThinWork w = thin_work(a, blockIdx.x);
    if (!w.any) return;
    const uint32_t row = w.row;
    const uint32_t rows = w.n * a.group - w.tile * kThinRows;  // of this tile (more: 16)
    const uint32_t rho = w.tile * kThinRows + (n < rows ? n : 0);
    const uint32_t token = token_of(a, rho), head = h * a.group + rho - token * a.group;
    const int pos = (int)(w.len - w.n + token);
    const int low = a.window && (uint32_t)pos + 1 > a.window ? pos + 1 - (int)a.window : 0;
    // positions that every row of the tile sees the keys between
    const uint32_t tok0 = token_of(a, w.tile * kThinRows), rows_in = rows < kThinRows ? rows : kThinRows;
    const uint32_t tok1 = token_of(a, w.tile * kThinRows + rows_in - 1);
    const int pos0 = (int)(w.len - w.n + tok0), pos1 = (int)(w.len - w.n + tok1);
    const int low1 = a.window && (uint32_t)pos1 + 1 > a.window ? pos1 + 1 - (int)a.window : 0;
    const int low0 = a.window && (uint32_t)pos0 + 1 > a.window ? pos0 + 1 - (int)a.window : 0;
    uint32_t b0 = w.b0, b1 = w.b1;
    if (!w.bad) {
        b0 = max(b0, (uint32_t)low0 / kKvBlock);
        b1 = min(b1, (uint32_t)pos1 / kKvBlock + 1);
    } else {
        b1 = b0;
        if (tid == 0 && h == 0) kv_report(a.err, kKvErrRows, row);
    }
    const uint32_t *table = a.b.table + (size_t)row * a.b.max_blocks;

    const uint32_t mine = b0 + which < b1 ? (b1 - b0 - which + NB - 1) / NB : 0;  // blocks of this wavefront
    const uint32_t rounds = SPLIT == 1 ? mine : b0 < b1 ? (b1 - b0 + NB - 1) / NB : 0;
    // The pages and scales of a wavefront's next 64 blocks, a block a lane: i is block
    // b0 + which + NB * i.  lost: blocks that the cache does not have.
    uint32_t page_l = 0;
    float2 scales_n = make_float2(0.0f, 0.0f);
    float ks_l = 0.0f, lv_l = 0.0f;  // keys' scale, and log2 of the values'
    uint64_t lost_n = 0;
    const auto pages = [&](uint32_t i) {
        page_l = table[b0 + which + NB * (i < mine ? i : mine - 1)];
        lost_n = __ballot(page_l >= a.n_blocks);
        if (lost_n) {
            if (page_l >= a.n_blocks) {
                page_l = 0;
                if (h == 0) kv_report(a.err, kKvErrBlock, row);
            }
        }
        scales_n = a.scales[(size_t)page_l * a.n_kv + h];
    };
    const auto load = [&](uint4 *to, uint32_t i, int of) {
        const uint32_t page = from_lane(page_l, i % kWave);
        const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + (((size_t)page * a.n_kv + h) * 2 + of) * (kKvBlock * D)) +
                         cut * C * kWave + lane;
#pragma unroll
        for (int c = 0; c < C; c++) to[c] = p[c * kWave];
    };
    const float *qp = a.q + (size_t)(w.first + token) * a.q_stride + (size_t)head * D + 8 * g;
    float4 qx[C][2];
#pragma unroll
    for (int c = 0; c < C; c++) {
        qx[c][0] = *reinterpret_cast<const float4 *>(qp + 32 * (cut * C + c));
        qx[c][1] = *reinterpret_cast<const float4 *>(qp + 32 * (cut * C + c) + 4);
    }
    if (mine) pages(lane);
    uint4 kq[C], vq[C];
    if (mine) {
        load(kq, 0, 0);
        load(vq, 0, 1);
    }

    // the queries' two parts, scaled to 2^14 .. 2^15 by a power of two
    half8 qh[kQueriesInLds ? 1 : C], ql[kQueriesInLds ? 1 : C];
    half8 *s_q = reinterpret_cast<half8 *>(&s_o[0][0][0]);  // [SPLIT][C][2][64]
    f32x4 *s_x = reinterpret_cast<f32x4 *>(s_q + D * 4);    // parts of q k^T, two rounds in turn, [2][W][2][64]
    static_assert(SPLIT == 1 || sizeof s_o >= (D * 4 + 4 * W * kWave) * 16, "both lie in s_o");
    float c_row;
    {
        float top = 0.0f;
        bool fine = true;
        const auto look = [&](float4 v) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                top = fmaxf(top, fabsf(e[i]));
                fine &= fabsf(e[i]) <= 3.402823466e38f;
            }
        };
#pragma unroll
        for (int c = 0; c < C; c++) look(qx[c][0]), look(qx[c][1]);
        top = row_max(fine ? top : __builtin_inff());
        if (SPLIT > 1) {  // (the other wavefront's channels too)
            if (g == 0) s_top[wave][n] = top;
            lds_barrier();
            top = fmaxf(top, s_top[wave ^ 1][n]);
        }
        const bool bad = top > 3.402823466e38f;
        int e = 0;
        (void)frexpf(top, &e);
        e = top > 0.0f ? 15 - e : 0;
        c_row = bad ? __builtin_nanf("") : ldexpf(fabsf(a.scale2), -e);
        const bool minus = a.scale2 < 0.0f;  // (the logits' factor is not negative: the largest stays it)
#pragma unroll
        for (int c = 0; c < C; c++) {
            const float f[8] = {qx[c][0].x, qx[c][0].y, qx[c][0].z, qx[c][0].w, qx[c][1].x, qx[c][1].y, qx[c][1].z, qx[c][1].w};
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = bad ? 0.0f : ldexpf(minus ? -f[i] : f[i], e);
                hi[i] = (_Float16)y;
                lo[i] = (_Float16)(y - (float)hi[i]);
            }
            if (!kQueriesInLds) {
                qh[kQueriesInLds ? 0 : c] = hi, ql[kQueriesInLds ? 0 : c] = lo;
            } else if (c % NB == (int)which) {
                s_q[((cut * C + c) * 2) * kWave + lane] = hi, s_q[((cut * C + c) * 2 + 1) * kWave + lane] = lo;
            }
        }
    }
    if (kQueriesInLds) lds_barrier();

    f32x4 o[2 * C];
#pragma unroll
    for (int i = 0; i < 2 * C; i++) o[i] = f32x4{0, 0, 0, 0};
    float m = kNegInf, l = 0.0f, mo = kNegInf;

    for (uint32_t i = 0; i < rounds; i++) {
        const bool on = i < mine;
        if (i % kWave == 0) {
            const bool lost = lost_n >> lane & 1;
            ks_l = lost ? __builtin_nanf("") : scales_n.x;
            lv_l = lost ? __builtin_nanf("") : log2_scale(scales_n.y);
        }
        f32x4 sa[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
        if (on) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                const half8 k0 = codes8(kq[c].x, kq[c].y), k1 = codes8(kq[c].z, kq[c].w);
                const half8 hi = kQueriesInLds ? s_q[((cut * C + c) * 2) * kWave + lane] : qh[kQueriesInLds ? 0 : c];
                const half8 lo = kQueriesInLds ? s_q[((cut * C + c) * 2 + 1) * kWave + lane] : ql[kQueriesInLds ? 0 : c];
                sa[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, lo, sa[0], 0, 0, 0);
                sa[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, lo, sa[1], 0, 0, 0);
                sa[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, hi, sa[0], 0, 0, 0);
                sa[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, hi, sa[1], 0, 0, 0);
            }
        }
        // (64 blocks on, page_l holds the next 64)
        const bool more = i + 1 < mine;
        if (more && (i + 1) % kWave == 0) pages(i + 1 + lane);
        if (more) load(kq, i + 1, 0);
        if (SPLIT > 1) {
            f32x4 *x = s_x + i % 2 * (W * 2 * kWave) + lane;
            x[wave * 2 * kWave] = sa[0], x[(wave * 2 + 1) * kWave] = sa[1];
            lds_barrier();
            sa[0] += x[(wave ^ 1) * 2 * kWave], sa[1] += x[((wave ^ 1) * 2 + 1) * kWave];
        }
        if (!on) continue;
        // keys 32 j + 16 (e / 4) + 4 g + e % 4
        const uint32_t j = b0 + which + NB * i;
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = sa[e / 4][e % 4];
        const bool edge = (int)(j * kKvBlock + kKvBlock - 1) > pos0 || (int)(j * kKvBlock) < low1;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = (int)(j * kKvBlock + 4 * g) + 16 * (e / 4) + e % 4;
                if (key > pos || key < low) t[e] = kNegInf;
            }
        }
        const float ks = __uint_as_float(from_lane(__float_as_uint(ks_l), i % kWave));
        const float lv = __uint_as_float(from_lane(__float_as_uint(lv_l), i % kWave));
        const float c = c_row * ks;
        float mb = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        mb = row_max(mb);
        mb = mb == kNegInf ? mb : mb * c;
        if (__any(mb > m + kSlack || mb + lv > mo + kSlack)) {
            const float m1 = fmaxf(m, mb), mo1 = fmaxf(mo, mb + lv);
            if (i) {  // (no sums before the first block)
                l *= __builtin_amdgcn_exp2f(m - (m1 == kNegInf ? 0.0f : m1));  // (0 before the first key)
                const float fall = mo == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mo - mo1);
#pragma unroll
                for (int k = 0; k < 2 * C; k++) o[k] *= fall;
            }
            m = m1, mo = mo1;
        }
        const float ms = m == kNegInf ? 0.0f : m;  // (no key yet)
        // (a weight of less than 2^-60 of the largest need not be that small among the sums, but counts in l)
        float eb = fmaxf(lv - mo, -60.0f - ms) + kBits;
        if (lv != lv) eb = lv;
        float p[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(t[e], c, eb));
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (t[e] == kNegInf) p[e] = 0.0f;  // (what is not seen adds nothing, whatever its scale)
        }
#pragma unroll
        for (int e = 0; e < 8; e++) sum += p[e];
        if (sum != 0.0f) l += sum * __builtin_amdgcn_exp2f(-eb - ms);  // (0: none in sight, and eb may be NaN)
        half8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const half2v hi = pair(p[e], p[e + 1]), lo = pair(rest0(hi, p[e]), rest1(hi, p[e + 1]));
            ph[e] = hi[0], ph[e + 1] = hi[1];
            pl[e] = lo[0], pl[e + 1] = lo[1];
        }
#pragma unroll
        for (int k = 0; k < C; k++) {
            const half8 v0 = codes8(vq[k].x, vq[k].y), v1 = codes8(vq[k].z, vq[k].w);
            o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * k], 0, 0, 0);
            o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * k + 1], 0, 0, 0);
            o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl, o[2 * k], 0, 0, 0);
            o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl, o[2 * k + 1], 0, 0, 0);
        }
        if (more) load(vq, i + 1, 1);
    }
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);

    // the wavefronts' parts joined through LDS
    if (g == 0 && cut == 0) s_m[which][n] = f32x4{m, l, mo, 0.0f};
    if (kQueriesInLds) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * C; i++) *reinterpret_cast<f32x4 *>(&s_o[which][n][cut * Sh::DW + 16 * i + 4 * g]) = o[i];
    __syncthreads();
    // Row rr's place among the sums and the outputs: its channels in fours, over the workgroup.
    const auto out_of = [&](uint32_t rr) {
        const uint32_t r1 = w.tile * kThinRows + rr, t = token_of(a, r1);
        return a.out + ((size_t)(w.first + t) * a.n_heads + h * a.group + r1 - t * a.group) * D;
    };
    const Shared shared(a.part, a.n_kv * 2 * a.slots * P);
    const auto place = [&](uint32_t slot) { return (h * 2 * a.slots + slot) * P; };
    // A row's four channels, to a part's place or to the outputs.
    constexpr uint32_t kOut = 0xffffffffu;
    const auto put = [&](const Joint &x, uint32_t rr, uint32_t d, uint32_t to) {
        if (to != kOut) {
            shared.put(to + rr * D + d, x.sum);
            if (d == 0) shared.put(to + kThinRows * D + 4 * rr, f32x4{x.m, x.l, x.mo, 0.0f});
        } else {
            const float scale = w.bad ? __builtin_nanf("") : out_scale(x.m, x.l, x.mo, kBits);
            *reinterpret_cast<f32x4 *>(out_of(rr) + d) = x.sum * scale;
        }
    };
    const uint32_t all = rows_in * (D / 4);
    for (uint32_t at = tid; at < all; at += NT) {
        const uint32_t rr = at / (D / 4), d = at % (D / 4) * 4;
        f32x4 st[NB], v[NB];
#pragma unroll
        for (int i = 0; i < NB; i++) st[i] = s_m[i][rr], v[i] = *reinterpret_cast<const f32x4 *>(&s_o[i][rr][d]);
        Joint x;
        x.clear();
        x.add(st, v, NB);
        put(x, rr, d, w.splits > 1 ? place(w.slot) : kOut);
    }
    if (w.splits == 1) return;

    // The part that is last at its group joins the group, the group that is last at its
    // tile the tile.  A part's stores are acknowledged before it counts; the one that
    // counts last reads past the L2s, and leaves the counters at zero.
    const uint32_t most_hands = all < (uint32_t)NT ? NT / all : 1;
    const uint32_t in_group = thin_in_group(w.splits, most_hands);
    const bool one = in_group == w.splits;
    const uint32_t grp = one ? 0 : w.split / in_group, slot0 = w.slot - w.split, g0 = slot0 + grp * in_group;
    const uint32_t gn = w.splits - grp * in_group < in_group ? w.splits - grp * in_group : in_group;
    const uint32_t groups = one ? 1 : (w.splits + in_group - 1) / in_group;
    uint32_t *tickets = a.tickets + (size_t)h * a.slots * 2;
    const auto last = [&](uint32_t *t, uint32_t count) -> bool {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const bool is = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
            if (is) __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = is;
        }
        __syncthreads();
        return s_last;
    };
    // Parts slot, slot + step, ..: their sums to `to`, or to the outputs.  Where there are more
    // threads than a part has places, the parts are dealt out to `hands` of them, and what
    // those make of them is joined through LDS.
    const auto join = [&](uint32_t slot, uint32_t step, uint32_t count, uint32_t to) {
        const uint32_t hands = count <= kBatch ? 1 : most_hands;  // (one after the other: a thread reads them all at once)
        const uint32_t hand = hands > 1 ? tid / all : 0;
        for (uint32_t at0 = 0; at0 < all; at0 += NT) {
            const uint32_t at = hands > 1 ? tid - hand * all : at0 + tid;
            const uint32_t rr = at / (D / 4), d = at % (D / 4) * 4;
            Joint x;
            x.clear();
            if (hand < hands && at < all)
                for (uint32_t u0 = hand; u0 < count; u0 += kBatch * hands) {
                    f32x4 st[kBatch], v[kBatch];
                    const uint32_t n_here = (count - u0 + hands - 1) / hands;
#pragma unroll
                    for (uint32_t u = 0; u < kBatch; u++) {
                        if (u % 4 == 0 && u >= n_here) break;
                        const uint32_t p = place(slot + (u < n_here ? u0 + u * hands : u0) * step);
                        st[u] = shared.get(p + kThinRows * D + 4 * rr), v[u] = shared.get(p + 4 * at);
                    }
                    x.add(st, v, n_here);
                }
            if (hands > 1) {
                f32x4 *s_part = reinterpret_cast<f32x4 *>(&s_o[0][0][0]);
                if (hand < hands) s_part[tid] = x.sum, s_part[NT + tid] = f32x4{x.m, x.l, x.mo, 0.0f};
                __syncthreads();
                if (hand) continue;  // (the only round)
                for (uint32_t k = 1; k < hands; k++) {
                    const f32x4 st[1] = {s_part[NT + k * all + at]}, v[1] = {s_part[k * all + at]};
                    x.add(st, v, 1);
                }
            }
            if (at < all) put(x, rr, d, to);
        }
    };
    if (!last(tickets + 2 * g0, gn)) return;
    if (groups == 1) {
        join(g0, 1, gn, kOut);
        return;
    }
    join(g0, 1, gn, place(a.slots + g0));
    if (last(tickets + 2 * slot0 + 1, groups)) join(a.slots + slot0, in_group, groups, kOut);
}

template <int D>
void go(ThinArgs t, uint32_t tiles, hipStream_t s) {
    using Sh = Shape<D>;
    t.target = Sh::kTarget, t.slots = thin_slots(t.target, t.n_kv), t.least = Sh::kBlocks;
    const uint32_t x = thin_grid(tiles, t.b.max_blocks, t.n_kv, t.target, t.least);
    hipLaunchKernelGGL(k_attention_thin<D>, dim3(x, t.n_kv), dim3(Sh::kThreads), 0, s, t);
}
}  // namespace

bool attention_head_dim(uint32_t D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256 || D == 512; }

static bool wide(const AttnArgs &a) { return any_wide(a.b.n_tokens, a.b.max_new, a.group); }

size_t attention_workspace(const AttnArgs &a) {
    const size_t thin = thin_workspace(a.kv.D, a.kv.n_kv);
    const size_t more = wide(a) ? attention_wide_workspace(a.kv.D) : 0;
    return thin < more ? more : thin;
}

hipError_t launch_attention(const AttnArgs &a, hipStream_t s) {
    if (wide(a)) {
        const hipError_t e = launch_attention_wide(a, s);
        if (e != hipSuccess) return e;
    }
    ThinArgs t{};
    t.codes = a.kv.codes, t.scales = a.kv.scales, t.n_blocks = a.kv.n_blocks, t.n_kv = a.kv.n_kv, t.b = a.b;
    t.q = a.q, t.out = a.out, t.q_stride = a.q_stride, t.n_heads = a.n_heads, t.group = a.group, t.window = a.window;
    t.scale2 = a.scale * 1.4426950408889634f, t.per_group = 1.0f / (float)a.group;
    t.part = (float *)a.work, t.tickets = a.tickets, t.err = a.err;
    const uint32_t tiles = thin_tiles(a.b.n_tokens, a.b.n_seqs, a.b.max_new, a.group);
    switch (a.kv.D) {
    case 64: go<64>(t, tiles, s); break;
    case 96: go<96>(t, tiles, s); break;
    case 128: go<128>(t, tiles, s); break;
    case 192: go<192>(t, tiles, s); break;
    case 256: go<256>(t, tiles, s); break;
    case 512: go<512>(t, tiles, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace lt
