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
// 2^(s + log2(scale) - mo), at most 1, times 2^15 to use f16's range; their sum
// times 2^(mo - log2(scale) - m) goes to l.  (Two maxima, because a block of small
// values may have the largest logit.)
//
// Work: a sequence's tiles are cut along the keys into parts of about the same
// number of blocks, as many as fill the chip; the part that arrives last at a
// tile joins them.
#include "llmtoy_hip.h"
#include "lt_attn.h"

namespace lt {

namespace {

constexpr int kThinRows = 16;
// Wavefronts of a workgroup: eight take a tile's blocks in turn; heads of 512
// need the registers and the LDS of twice as much.
template <int D>
constexpr int kThinWaves = D <= 256 ? 8 : 4;
// Workgroups that a launch's work is split into, where there are fewer tiles: one
// on each CU.
constexpr uint32_t kThinTarget = 256;
// Parts of a tile that are joined at once; more are joined in groups first.
constexpr uint32_t kJoin = 16;

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
    float *part;        // [n_kv][slots][16][D + 4]: sums, then m, l, mo
    uint32_t *tickets;  // [n_kv][slots][2]: groups, tiles; zero between launches
    uint32_t slots;
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
    // (beyond max_new: as many as the grid has room for, and those get NaN)
    const uint32_t n = a.b.max_new && t.k.n > a.b.max_new ? a.b.max_new : t.k.n;
    t.tiles = n * a.group > kThinMost ? 0 : (n * a.group + kThinRows - 1) / kThinRows;
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

// Blocks a part: all of the batch's over the launch's workgroups, evenly, and one
// a wavefront at least.  Every wavefront finds it for itself from the lengths
// (one load and a sum for up to 64 sequences).
__device__ __forceinline__ uint32_t thin_share(const ThinArgs &a, uint32_t least) {
    float sum = 0.0f;  // (a count beyond 2^24 need not be exact)
    for (uint32_t r = threadIdx.x % kWave; r < a.b.n_seqs; r += kWave) {
        const ThinRow t = thin_row(a, r);
        if (t.k.falls && blockIdx.x == 0 && blockIdx.y == 0) kv_report(a.err, kKvErrRows, r);
        sum += (float)t.tiles * (float)t.blocks;
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    const float each = ceilf(sum * (float)a.n_kv / (float)kThinTarget);
    return each < (float)least ? least : each > 1e9f ? 1000000000u : (uint32_t)each;
}

__device__ __forceinline__ ThinWork thin_work(const ThinArgs &a, uint32_t index, uint32_t least) {
    ThinWork w{};
    const uint32_t lane = threadIdx.x % kWave, share = thin_share(a, least);
    uint32_t seen = 0, joined = 0;  // workgroups and joined parts of the rows before
    for (uint32_t r0 = 0; r0 < a.b.n_seqs; r0 += kWave) {
        const uint32_t r = r0 + lane;
        ThinRow t{};
        uint32_t splits = 0;
        if (r < a.b.n_seqs) {
            t = thin_row(a, r);
            splits = (t.blocks + share - 1) / share;
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
            w.tile = in / w.splits;
            w.split = in % w.splits;
            const uint32_t lo = from_lane(t.lo, l), blocks = from_lane(t.blocks, l);
            // as even as whole blocks go
            w.b0 = lo + (uint32_t)((uint64_t)blocks * w.split / w.splits);
            w.b1 = lo + (uint32_t)((uint64_t)blocks * (w.split + 1) / w.splits);
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

// The largest of the four lanes that share a row.
__device__ __forceinline__ float row_max(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// Joins `count` partial results that lie `step` floats apart into a row's sums: T
// threads a row, thread `part` the channels 4 part + 4 T i.
template <int D, int T>
struct Joined {
    static constexpr int N = (D + 4 * T - 1) / (4 * T);
    f32x4 sum[N];
    float m, l, mo;
    __device__ __forceinline__ void run(const float *from, uint32_t count, size_t step, uint32_t part) {
        m = kNegInf, mo = kNegInf, l = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] = f32x4{0, 0, 0, 0};
        // (the largest so far, as the softmax runs: one pass, four parts' loads at once)
        for (uint32_t i = 0; i < count; i += 4) {
            f32x4 st[4], v[4][N];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float *p = from + (size_t)(i + u < count ? i + u : i) * step;
                st[u] = get4(p + D);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const uint32_t d = 4 * (part + T * k);
                    v[u][k] = get4(p + (d < D ? d : 0));
                }
            }
            float m1 = m, mo1 = mo;
#pragma unroll
            for (int u = 0; u < 4; u++) m1 = fmaxf(m1, st[u][0]), mo1 = fmaxf(mo1, st[u][2]);
            l *= m == kNegInf ? 1.0f : exp2f(m - m1);  // (l is 0 or NaN then)
            const float fall = mo == kNegInf ? 1.0f : exp2f(mo - mo1);
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] *= fall;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (i + u >= count) break;
                l += st[u][0] == kNegInf ? st[u][1] : st[u][1] * exp2f(st[u][0] - m1);
                const float f = st[u][2] == kNegInf ? 1.0f : exp2f(st[u][2] - mo1);  // (sums of 0 or NaN)
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] += v[u][k] * f;
            }
            m = m1, mo = mo1;
        }
    }
};

template <int D>
__global__ __launch_bounds__(kThinWaves<D> *kWave, D <= 256 ? 2 : 1) void k_attention_thin(ThinArgs a) {
    constexpr int C = D / 32, P = D + 4, W = kThinWaves<D>, T = W * kWave / kThinRows;  // P: floats of a joined row
    // the wavefronts' sums; with heads of 256 and more the queries lie there before
    constexpr bool kQueriesInLds = D >= 256;
    __shared__ __align__(16) float s_o[W][kThinRows][D + 4];
    __shared__ float s_m[3][W][kThinRows];
    __shared__ uint32_t s_last;
    const uint32_t lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), h = blockIdx.y;
    const ThinWork w = thin_work(a, blockIdx.x, W);
    if (!w.any) return;
    const uint32_t row = w.row;
    const uint32_t rows = w.n * a.group - w.tile * kThinRows;  // of this tile (more: 16)
    const uint32_t rho = w.tile * kThinRows + (n < rows ? n : 0);
    const uint32_t token = rho / a.group, head = h * a.group + rho % a.group;
    const int pos = (int)(w.len - w.n + token);
    const int low = a.window && (uint32_t)pos + 1 > a.window ? pos + 1 - (int)a.window : 0;
    // positions that every row of the tile sees the keys between
    const uint32_t tok0 = w.tile * kThinRows / a.group, rows_in = rows < kThinRows ? rows : kThinRows;
    const uint32_t tok1 = (w.tile * kThinRows + rows_in - 1) / a.group;
    const int pos0 = (int)(w.len - w.n + tok0), pos1 = (int)(w.len - w.n + tok1);
    const int low1 = a.window && (uint32_t)pos1 + 1 > a.window ? pos1 + 1 - (int)a.window : 0;
    const int low0 = a.window && (uint32_t)pos0 + 1 > a.window ? pos0 + 1 - (int)a.window : 0;
    uint32_t b0 = w.b0, b1 = w.b1;
    if (!w.bad) {
        b0 = max(b0, (uint32_t)low0 / kKvBlock);
        b1 = min(b1, (uint32_t)pos1 / kKvBlock + 1);
    } else {
        b1 = b0;
        if (threadIdx.x == 0 && h == 0) kv_report(a.err, kKvErrRows, row);
    }
    const uint32_t *table = a.b.table + (size_t)row * a.b.max_blocks;

    // The pages and scales of a wavefront's next 64 blocks, a block a lane: i is block
    // b0 + wave + W * i.  Keys' scale, and log2 of the values' (a block of zeros: any).
    uint32_t page_l = 0;
    float ks_l = 0.0f, lv_l = 0.0f;
    const auto pages = [&](uint32_t i) {
        const uint32_t j = b0 + wave + W * i;
        if (j >= b1) return;
        page_l = table[j];
        const bool lost = page_l >= a.n_blocks;
        if (lost) {
            page_l = 0;
            if (h == 0) kv_report(a.err, kKvErrBlock, row);
        }
        const float2 s = a.scales[(size_t)page_l * a.n_kv + h];
        ks_l = lost ? __builtin_nanf("") : s.x;
        lv_l = lost ? __builtin_nanf("") : s.y == 0.0f ? 0.0f : log2f(s.y);
    };
    pages(lane);

    // the queries' two parts, scaled to 2^14 .. 2^15 by a power of two
    half8 qh[kQueriesInLds ? 1 : C], ql[kQueriesInLds ? 1 : C];
    half8 *s_q = reinterpret_cast<half8 *>(&s_o[0][0][0]);  // [C][2][64]
    float c_row;
    {
        const float *qp = a.q + (size_t)(w.first + token) * a.q_stride + (size_t)head * D + 8 * g;
        float top = 0.0f;
        bool fine = true;
        float x[C][8];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const float4 u = *reinterpret_cast<const float4 *>(qp + 32 * c), v = *reinterpret_cast<const float4 *>(qp + 32 * c + 4);
            const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = e[i];
                top = fmaxf(top, fabsf(e[i]));
                fine &= fabsf(e[i]) <= 3.402823466e38f;
            }
        }
        const bool bad = row_max(fine ? 0.0f : 1.0f) > 0.0f;
        top = row_max(top);
        int e = 0;
        (void)frexpf(top, &e);
        e = top > 0.0f ? 15 - e : 0;
        c_row = bad ? __builtin_nanf("") : ldexpf(fabsf(a.scale2), -e);
        const bool minus = a.scale2 < 0.0f;  // (the logits' factor is not negative: the largest stays it)
#pragma unroll
        for (int c = 0; c < C; c++) {
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = bad ? 0.0f : ldexpf(minus ? -x[c][i] : x[c][i], e);
                hi[i] = (_Float16)y;
                lo[i] = (_Float16)(y - (float)hi[i]);
            }
            if (!kQueriesInLds) {
                qh[kQueriesInLds ? 0 : c] = hi, ql[kQueriesInLds ? 0 : c] = lo;
            } else if (c % W == (int)wave) {
                s_q[(c * 2) * kWave + lane] = hi, s_q[(c * 2 + 1) * kWave + lane] = lo;
            }
        }
    }
    if (kQueriesInLds) __syncthreads();

    f32x4 o[2 * C];
#pragma unroll
    for (int i = 0; i < 2 * C; i++) o[i] = f32x4{0, 0, 0, 0};
    float m = kNegInf, l = 0.0f, mo = kNegInf;

    uint4 kq[C], vq[C];
    const auto load = [&](uint4 *to, uint32_t page, int which) {
        const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + (((size_t)page * a.n_kv + h) * 2 + which) * (kKvBlock * D)) + lane;
#pragma unroll
        for (int c = 0; c < C; c++) to[c] = p[c * kWave];
    };
    const uint32_t mine = b0 + wave < b1 ? (b1 - b0 - wave + W - 1) / W : 0;  // blocks of this wavefront
    for (uint32_t i0 = 0; i0 < mine; i0 += kWave) {
        if (i0) pages(i0 + lane);
        const uint32_t here = mine - i0 < kWave ? mine - i0 : kWave;
        load(kq, from_lane(page_l, 0), 0);
        load(vq, from_lane(page_l, 0), 1);
        for (uint32_t i = 0; i < here; i++) {
            const uint32_t next = from_lane(page_l, i + 1 < here ? i + 1 : i);
            const float ks = __uint_as_float(from_lane(__float_as_uint(ks_l), i));
            const float lv = __uint_as_float(from_lane(__float_as_uint(lv_l), i));
            f32x4 sa[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}, sb[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int c = 0; c < C; c++) {
                const half8 k0 = codes8(kq[c].x, kq[c].y), k1 = codes8(kq[c].z, kq[c].w);
                const half8 hi = kQueriesInLds ? s_q[(c * 2) * kWave + lane] : qh[kQueriesInLds ? 0 : c];
                const half8 lo = kQueriesInLds ? s_q[(c * 2 + 1) * kWave + lane] : ql[kQueriesInLds ? 0 : c];
                sa[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, hi, sa[0], 0, 0, 0);
                sa[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, hi, sa[1], 0, 0, 0);
                sb[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, lo, sb[0], 0, 0, 0);
                sb[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, lo, sb[1], 0, 0, 0);
            }
            if (i + 1 < here) load(kq, next, 0);
            // keys 32 j + 16 (e / 4) + 4 g + e % 4
            const uint32_t j = b0 + wave + W * (i0 + i);
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) t[e] = sa[e / 4][e % 4] + sb[e / 4][e % 4];
            const bool edge = (int)(j * kKvBlock + kKvBlock - 1) > pos0 || (int)(j * kKvBlock) < low1;
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = (int)(j * kKvBlock + 4 * g) + 16 * (e / 4) + e % 4;
                    if (key > pos || key < low) t[e] = kNegInf;
                }
            }
            const float c = c_row * ks;
            float mb = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
            mb = row_max(mb);
            mb = mb == kNegInf ? mb : mb * c;
            const float m1 = fmaxf(m, mb), mo1 = fmaxf(mo, mb + lv);
            const float ms = m1 == kNegInf ? 0.0f : m1;  // (no key yet)
            if (__any(m1 > m || mo1 > mo)) {
                l *= __builtin_amdgcn_exp2f(m - ms);  // (0 before the first key)
                const float fall = mo == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mo - mo1);
#pragma unroll
                for (int k = 0; k < 2 * C; k++) o[k] *= fall;
            }
            m = m1, mo = mo1;
            // (a weight of less than 2^-60 of the largest need not be that small among the sums, but counts in l)
            float e15 = fmaxf(lv - mo1, -60.0f - ms) + 15.0f;
            if (lv != lv) e15 = lv;
            float p[8], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(t[e], c, e15));
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (t[e] == kNegInf) p[e] = 0.0f;  // (what is not seen adds nothing, whatever its scale)
            }
#pragma unroll
            for (int e = 0; e < 8; e++) sum += p[e];
            if (mo1 != kNegInf || sum != sum) l += sum * __builtin_amdgcn_exp2f(-e15 - ms);
            half8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const _Float16 hi = (_Float16)p[e];
                ph[e] = hi;
                pl[e] = (_Float16)(p[e] - (float)hi);
            }
#pragma unroll
            for (int k = 0; k < C; k++) {
                const half8 v0 = codes8(vq[k].x, vq[k].y), v1 = codes8(vq[k].z, vq[k].w);
                o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * k], 0, 0, 0);
                o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * k + 1], 0, 0, 0);
                o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl, o[2 * k], 0, 0, 0);
                o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl, o[2 * k + 1], 0, 0, 0);
            }
            if (i + 1 < here) load(vq, next, 1);
        }
    }
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);

    // the wavefronts' parts joined through LDS
    if (g == 0) s_m[0][wave][n] = m, s_m[1][wave][n] = l, s_m[2][wave][n] = mo;
    if (kQueriesInLds) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * C; i++) *reinterpret_cast<f32x4 *>(&s_o[wave][n][16 * i + 4 * g]) = o[i];
    __syncthreads();
    // a row's channels over T threads
    const uint32_t rr = threadIdx.x / T, part = threadIdx.x % T;
    const uint32_t r1 = w.tile * kThinRows + rr;
    float *out = a.out + ((size_t)(w.first + r1 / a.group) * a.n_heads + h * a.group + r1 % a.group) * D;
    float *mine_p = a.part + (((size_t)h * a.slots + w.slot) * kThinRows + rr) * P;
    if (rr < rows_in) {
        float mt = kNegInf, mot = kNegInf, lt_ = 0.0f, fo[W];
#pragma unroll
        for (int i = 0; i < W; i++) mt = fmaxf(mt, s_m[0][i][rr]), mot = fmaxf(mot, s_m[2][i][rr]);
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float mi = s_m[0][i][rr], moi = s_m[2][i][rr], li = s_m[1][i][rr];
            lt_ += mi == kNegInf ? li : li * exp2f(mi - mt);  // (l is 0 or NaN without a largest)
            fo[i] = moi == kNegInf ? 1.0f : exp2f(moi - mot);
        }
        const float scale = w.splits > 1 ? 1.0f : w.bad ? __builtin_nanf("") : out_scale(mt, lt_, mot, 15.0f);
#pragma unroll
        for (int i = 0; i < (D + 4 * T - 1) / (4 * T); i++) {
            const uint32_t d = 4 * (part + T * i);
            if (d >= D) break;
            f32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < W; u++) sum += *reinterpret_cast<const f32x4 *>(&s_o[u][rr][d]) * fo[u];
            if (w.splits > 1) put4(mine_p + d, sum);
            else *reinterpret_cast<f32x4 *>(out + d) = sum * scale;
        }
        if (w.splits > 1 && part == 0) put4(mine_p + D, f32x4{mt, lt_, mot, 0});
    }
    if (w.splits == 1) return;

    // The part that is last at its group joins the group, the group that is last at its
    // tile the tile.  A part's stores are acknowledged before it counts; the one that
    // counts last reads past the L2s, and leaves the counters at zero.
    const uint32_t groups = (w.splits + kJoin - 1) / kJoin, in_group = (w.splits + groups - 1) / groups;
    const uint32_t grp = w.split / in_group, slot0 = w.slot - w.split;
    const uint32_t g0 = slot0 + grp * in_group;
    const uint32_t gn = w.splits - grp * in_group < in_group ? w.splits - grp * in_group : in_group;
    const uint32_t used_groups = (w.splits + in_group - 1) / in_group;
    uint32_t *tickets = a.tickets + (size_t)h * a.slots * 2;
    const auto last = [&](uint32_t *t, uint32_t count) -> bool {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            const bool is = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
            if (is) __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = is;
        }
        __syncthreads();
        return s_last;
    };
    if (!last(tickets + 2 * g0, gn)) return;
    Joined<D, T> sums;
    const size_t step = (size_t)kThinRows * P;
    const float *from = a.part + (((size_t)h * a.slots + g0) * kThinRows + rr) * P;
    if (rr < rows_in) sums.run(from, gn, step, part);
    if (used_groups > 1) {
        // (the group's first part's place now holds the group's sums)
        float *to = const_cast<float *>(from);
        __syncthreads();
        if (rr < rows_in) {
#pragma unroll
            for (int k = 0; k < Joined<D, T>::N; k++) {
                const uint32_t d = 4 * (part + T * k);
                if (d < D) put4(to + d, sums.sum[k]);
            }
            if (part == 0) put4(to + D, f32x4{sums.m, sums.l, sums.mo, 0});
        }
        if (!last(tickets + 2 * slot0 + 1, used_groups)) return;
        from = a.part + (((size_t)h * a.slots + slot0) * kThinRows + rr) * P;
        if (rr < rows_in) sums.run(from, used_groups, step * in_group, part);
    }
    if (rr < rows_in) {
        const float scale = out_scale(sums.m, sums.l, sums.mo, 15.0f);
#pragma unroll
        for (int k = 0; k < Joined<D, T>::N; k++) {
            const uint32_t d = 4 * (part + T * k);
            if (d < D) *reinterpret_cast<f32x4 *>(out + d) = sums.sum[k] * scale;
        }
    }
}

// Workgroups of a head: a tile more or less a sequence, and the parts of those
// that are split (at most the target and one more a tile).
uint32_t thin_tiles(const AttnArgs &a) {
    const uint64_t rows = (uint64_t)a.b.n_tokens * a.group;
    uint64_t tiles = rows / kThinRows + a.b.n_seqs;
    const uint64_t each = a.b.max_new && (uint64_t)a.b.max_new * a.group < kThinMost ? a.b.max_new * a.group : kThinMost;
    const uint64_t most = (uint64_t)a.b.n_seqs * ((each + kThinRows - 1) / kThinRows);
    if (most < tiles) tiles = most;
    if (rows < tiles) tiles = rows;
    return (uint32_t)tiles;
}
uint32_t thin_slots(uint32_t n_kv) { return 2 * (kThinTarget / n_kv + 1) + 2; }

template <int D>
void go(const ThinArgs &t, uint32_t tiles, hipStream_t s) {
    const dim3 grid(tiles + kThinTarget / t.n_kv + 1, t.n_kv);
    hipLaunchKernelGGL(k_attention_thin<D>, grid, dim3(kThinWaves<D> * kWave), 0, s, t);
}

}  // namespace

bool attention_head_dim(uint32_t D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256 || D == 512; }

// Whether a sequence may have rows for the wide kernel.
static bool wide(const AttnArgs &a) { return (uint64_t)(a.b.max_new ? a.b.max_new : a.b.n_tokens) * a.group > kThinMost; }

size_t attention_workspace(const AttnArgs &a) {
    const size_t thin = (size_t)a.kv.n_kv * thin_slots(a.kv.n_kv) * kThinRows * (a.kv.D + 4) * 4;
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
    t.scale2 = a.scale * 1.4426950408889634f;
    t.part = (float *)a.work, t.tickets = a.tickets, t.slots = thin_slots(t.n_kv), t.err = a.err;
    const uint32_t tiles = thin_tiles(a);
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
