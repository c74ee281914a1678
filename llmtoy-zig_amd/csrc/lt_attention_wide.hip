// lt_attention_wide.hip -- attention over the 8-bit cache (lt_kv.h) for
// sequences with many tokens in the batch: prompts and parts of prompts.  The
// mathematics, the two parts of queries and weights and the softmax's two
// maxima are lt_attention.hip's.
//
// A wavefront has 32 rows (tokens and heads of one group): queries in registers,
// sums in registers, v_mfma_f32_32x32x16_f16.  The codes of a block are
// converted once a workgroup, into LDS, in the order of the operands: each
// wavefront converts its share of the next block while it computes with this one.
// Wide heads are cut over SPLIT wavefronts, which add their parts of q k^T
// through LDS and each find the same weights.
//
// With two parts of queries and of weights a block takes 4 D / 16 of these
// instructions a wavefront, 1,024 cycles with heads of 128, and about 180 vector instructions (a
// sixth of them exponentials), 940 cycles.  The two do not run side by side here: together they are
// what a CU is busy for, with two wavefronts a SIMD of one workgroup or of two, with and
// without priorities, and with the next block's products between this one's exponentials.  4,095
// tokens of 32 heads of 128: 262 us, 1.05 PFLOP/s of f16 products (a library's product of 8192^3: 1.14).
//
// Work: whole tiles, the longest first, where there are enough of them; else all
// tiles' blocks in one line, cut into as many equal pieces as workgroups fit on
// the chip.  A tile's pieces leave their sums in memory, and the one that is last joins them.
#include "llmtoy_hip.h"
#include "lt_attn.h"

namespace lt {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t kJoin = 16;      // parts joined at once; more are joined in groups first

struct WideArgs {
    const uint8_t *codes;
    const float2 *scales;
    uint32_t n_blocks, n_kv;
    KvBatchDev b;
    const float *q;
    float *out;
    size_t q_stride;
    uint32_t n_heads, group, window;
    float scale2;       // scale * log2(e)
    uint32_t tiles;     // of a head, at most
    uint32_t pieces;    // workgroups that the tiles' blocks are cut for; 0: whole tiles
    float *part;        // [2 pieces] parts of tiles
    uint32_t *tickets;  // [3 pieces], zero between launches
    uint32_t *err;
};

// Wavefronts a head is cut over, wavefronts a workgroup, workgroups a CU.  Measured on
// 512 queries of 16 or 32 heads (us): heads of 64 4 wavefronts three times a CU 319, twice 335, 8 345;
// of 96 8 230, 4 twice a CU 238; of 128 8 501, 4 twice 523; of 192 cut, 4 twice 280, 8 288;
// of 256 whole 363, cut 475.  (Products of the next block between this one's
// exponentials: slower for 64 to 128 and 512, 5% faster for 192.)
template <int D>
struct Shape {
    static constexpr int kSplit = D == 192 || D == 512 ? 2 : 1, kWaves = D == 96 || D == 128 ? 8 : 4;
    static constexpr int kPerCu = D == 64 ? 3 : D == 192 ? 2 : 1;
    static constexpr int kThreads = kWaves * kWave, kRows = 32 * kWaves / kSplit;
    static constexpr int DW = D / kSplit, S = DW / 16, CB = DW / 32;
    static constexpr uint32_t kPart = kWaves * (CB * 4 + 1) * kWave * 4;  // floats
};

struct Tile {
    KvRow k;
    uint32_t r0, rows;  // its first row among the sequence's, its rows
    uint32_t lo, hi;    // blocks lo .. hi - 1
};

template <int R>
__device__ __forceinline__ uint32_t row_tiles(const WideArgs &a, uint32_t row) {
    return wide_row_tiles(cut_tokens(kv_row_of(a.b, row).n, a.b.max_new), a.group, R);
}

template <int R>
__device__ __forceinline__ Tile tile_of(const WideArgs &a, uint32_t row, uint32_t t) {
    Tile x;
    x.k = kv_row_of(a.b, row);
    const uint32_t all = cut_tokens(x.k.n, a.b.max_new) * a.group;
    x.r0 = t * R;
    x.rows = all - x.r0 < R ? all - x.r0 : R;
    x.lo = 0, x.hi = 1;
    if (!x.k.bad) {
        const uint32_t begin = x.k.len - x.k.n, pos0 = begin + x.r0 / a.group, pos1 = begin + (x.r0 + x.rows - 1) / a.group;
        if (a.window && pos0 + 1 > a.window) x.lo = (pos0 + 1 - a.window) / kKvBlock;
        x.hi = pos1 / kKvBlock + 1;
    }
    return x;
}

// The sum of v over the threads before this one, and over all.
template <int WAVES>
__device__ __forceinline__ uint64_t scan(uint64_t v, uint64_t *s_sum, uint64_t &all) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint64_t up = v;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint64_t p = __shfl_up(up, off, kWave);
        if ((int)lane >= off) up += p;
    }
    __syncthreads();
    if (lane == kWave - 1) s_sum[wave] = up;
    __syncthreads();
    uint64_t before = up - v;
    all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w < (int)wave) before += s_sum[w];
        all += s_sum[w];
    }
    return before;
}

// The last i < n with first[i] <= u, first not falling, first[0] <= u.
template <typename T>
__device__ __forceinline__ uint32_t last_at(const T *first, uint32_t n, T u) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Larger of the two lanes that share a row.
__device__ __forceinline__ float row_max2(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// v, but what is computed from it stays in its branch (the compiler would rather always do it and select).
template <typename T>
__device__ __forceinline__ T in_branch(T v) {
    asm volatile("" : "+v"(v));
    return v;
}

// N operands read from LDS one after the other, the i-th for use(i, operand): kAhead of
// them under way before the first product (the compiler, short of registers, would
// read one and wait for it).
constexpr int kAhead = 4;
struct Feed {
    half8 x[kAhead];
    const half8 *from;
    __device__ __forceinline__ void open(const half8 *f) {
        from = f;
#pragma unroll
        for (int i = 0; i < kAhead; i++) x[i] = from[i * kWave];
    }
    template <int N, typename F>
    __device__ __forceinline__ void run(F use) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            __builtin_amdgcn_sched_barrier(0);
            use(i, x[i % kAhead]);
            __builtin_amdgcn_sched_barrier(0);
            if (i + kAhead < N) x[i % kAhead] = from[(i + kAhead) * kWave];
        }
    }
};

template <int D>
__global__ __launch_bounds__(Shape<D>::kThreads, Shape<D>::kPerCu) void k_attention_wide(WideArgs a) {
    using Sh = Shape<D>;
    constexpr int SPLIT = Sh::kSplit, W = Sh::kWaves, NT = Sh::kThreads, R = Sh::kRows, S = Sh::S, CB = Sh::CB;
    constexpr int NG = D / 16, GPW = (NG + W - 1) / W;  // KiB of codes a block, a wavefront
    __shared__ half8 s_kv[2][8 * D];
    __shared__ f32x4 s_x[SPLIT > 1 ? W * 4 * kWave : 1];
    __shared__ uint64_t s_first[kMaxTiles], s_sum[W];
    __shared__ uint32_t s_base[kMaxTiles], s_hit[2], s_last;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, half = lane / 32, n = lane % 32;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / kWave), cut = wave % SPLIT, rg = wave / SPLIT;

    // ---- the rows' tiles
    const uint32_t per = (a.b.n_seqs + NT - 1) / NT;
    uint64_t mine = 0, every;  // (sequences that overlap may have 2^32 tiles and more)
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t r = tid * per + i;
        if (r >= a.b.n_seqs) break;
        const KvRow k = kv_row_of(a.b, r);
        mine += wide_row_tiles(cut_tokens(k.n, a.b.max_new), a.group, R);
        if (k.falls && blockIdx.x == 0) kv_report(a.err, kKvErrRows, r);
    }
    const uint64_t before0 = scan<W>(mine, s_sum, every);
    if (every > a.tiles) return;  // (start falls, sequences overlap; reported)
    const uint32_t all_tiles = (uint32_t)every;
    uint32_t at = (uint32_t)before0;
    // ---- what this workgroup takes: blocks u .. u1 - 1 of the line of heads and tiles, or a tile
    uint64_t u = 0, u1 = 1, line = 0, total = 0;
    uint32_t pieces = 1, piece = 0, head_kv = 0;
    if (!a.pieces) {
        // (the longest are the last)
        const uint32_t t = a.tiles - 1 - blockIdx.x / a.n_kv;
        head_kv = blockIdx.x % a.n_kv;
        if (t >= all_tiles) return;
        for (uint32_t i = 0; i < per; i++) {
            const uint32_t r = tid * per + i;
            if (r >= a.b.n_seqs) break;
            const uint32_t c = row_tiles<R>(a, r);
            if (t >= at && t < at + c) s_hit[0] = r, s_hit[1] = t - at;
            at += c;
        }
        __syncthreads();
    } else {
        // (a.tiles <= kMaxTiles, and a sequence counts as one at least)
        for (uint32_t i = 0; i < per; i++) {
            const uint32_t r = tid * per + i;
            if (r >= a.b.n_seqs) break;
            s_base[r] = at;
            at += row_tiles<R>(a, r);
        }
        __syncthreads();
        const uint32_t per2 = (all_tiles + NT - 1) / NT;
        uint64_t blocks = 0;
        for (uint32_t i = 0; i < per2; i++) {
            const uint32_t t = tid * per2 + i;
            if (t >= all_tiles) break;
            const uint32_t r = last_at(s_base, a.b.n_seqs, t);
            const Tile x = tile_of<R>(a, r, t - s_base[r]);
            s_first[t] = blocks;
            blocks += x.hi - x.lo;
        }
        const uint64_t before = scan<W>(blocks, s_sum, line);
        for (uint32_t i = 0; i < per2; i++)
            if (tid * per2 + i < all_tiles) s_first[tid * per2 + i] += before;
        __syncthreads();
        total = line * a.n_kv;
        pieces = wide_cut(total, a.pieces);
        // (an XCD's workgroups side by side in the line: their L2 has the blocks)
        piece = blockIdx.x;
        if (pieces == a.pieces && pieces % 8 == 0) piece = piece % 8 * (pieces / 8) + piece / 8;
        if (piece >= pieces) return;
        u = total * piece / pieces;
        u1 = total * (piece + 1) / pieces;
    }

    while (u < u1) {
        uint32_t tile = 0, row, t;
        uint64_t first = 0;  // the tile's place in the line
        if (a.pieces) {
            head_kv = (uint32_t)(u / line);
            tile = last_at(s_first, all_tiles, u - head_kv * line);
            row = last_at(s_base, a.b.n_seqs, tile);
            t = tile - s_base[row];
            first = head_kv * line + s_first[tile];
        } else {
            row = s_hit[0], t = s_hit[1];
        }
        row = __builtin_amdgcn_readfirstlane(row), t = __builtin_amdgcn_readfirstlane(t);
        head_kv = __builtin_amdgcn_readfirstlane(head_kv);
        const Tile x = tile_of<R>(a, row, t);
        uint32_t b0 = x.lo, b1 = x.hi;
        uint64_t next = u1;
        bool whole = true;
        if (a.pieces) {
            const uint64_t end = first + (x.hi - x.lo);
            next = end < u1 ? end : u1;
            b0 = x.lo + (uint32_t)(u - first);
            b1 = x.lo + (uint32_t)(next - first);
            whole = u == first && next == end;
        }
        b0 = __builtin_amdgcn_readfirstlane(b0), b1 = __builtin_amdgcn_readfirstlane(b1);
        if (x.k.bad) {
            if (tid == 0 && head_kv == 0) kv_report(a.err, kKvErrRows, row);
            b1 = b0;
        }
        const uint32_t h = head_kv;
        const uint32_t *table = a.b.table + (size_t)row * a.b.max_blocks;

        // ---- this lane's row; positions that all rows of the wavefront see the keys between
        const uint32_t begin = x.k.len - x.k.n;
        const uint32_t in = rg * 32 + n < x.rows ? rg * 32 + n : 0;  // (rows behind the tile's: its first once more)
        const uint32_t token = (x.r0 + in) / a.group, head = h * a.group + (x.r0 + in) % a.group;
        const int pos = (int)(begin + token);
        const int low = a.window && (uint32_t)pos + 1 > a.window ? pos + 1 - (int)a.window : 0;
        const bool idle = rg * 32 >= x.rows;
        const uint32_t wlast = rg * 32 + 31 < x.rows ? rg * 32 + 31 : x.rows - 1;
        // (with rows behind the tile's in it, a wavefront also has the tile's first)
        const uint32_t wfirst = rg * 32 + 31 < x.rows ? rg * 32 : 0;
        const int pos0 = (int)(begin + (x.r0 + wfirst) / a.group), pos1 = (int)(begin + (x.r0 + wlast) / a.group);
        const int low0 = a.window && (uint32_t)pos0 + 1 > a.window ? pos0 + 1 - (int)a.window : 0;
        const int low1 = a.window && (uint32_t)pos1 + 1 > a.window ? pos1 + 1 - (int)a.window : 0;

        // ---- pages and scales of 64 blocks, a block a lane; keys' scale and log2 of the values'
        uint32_t page_l = 0;
        float ks_n = 0.0f, lv_n = 0.0f, ks_l = 0.0f, lv_l = 0.0f;
        const auto pages = [&](uint32_t j) {
            if (j >= b1) return;
            page_l = table[j];
            const bool lost = page_l >= a.n_blocks;
            if (lost) {
                page_l = 0;
                if (h == 0) kv_report(a.err, kKvErrBlock, row);
            }
            const float2 s = a.scales[(size_t)page_l * a.n_kv + h];
            ks_n = lost ? __builtin_nanf("") : s.x;
            lv_n = lost ? __builtin_nanf("") : log2_scale(s.y);
        };
        uint4 raw[GPW];
        const auto fetch = [&](uint32_t j) {
            if (j >= b1) return;
            if ((j - b0) % kWave == 0) pages(j + lane);
            const uint32_t page = from_lane(page_l, (j - b0) % kWave);
            const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + ((size_t)page * a.n_kv + h) * (2 * kKvBlock * D)) + lane;
#pragma unroll
            for (int i = 0; i < GPW; i++)
                if (NG % W == 0 || wave + i * W < NG) raw[i] = p[(wave + i * W) * kWave];
        };
        const uint32_t lds_at = (lane / 32) * kWave + (lane / 16 % 2) * 32 + lane % 16;
        const auto stage = [&](uint32_t j) {
            if (j >= b1) return;
            half8 *to = s_kv[(j - b0) % 2] + lds_at;
#pragma unroll
            for (int i = 0; i < GPW; i++)
                if (NG % W == 0 || wave + i * W < NG) {
                    to[(wave + i * W) * 2 * kWave] = codes8(raw[i].x, raw[i].y);
                    to[(wave + i * W) * 2 * kWave + 16] = codes8(raw[i].z, raw[i].w);
                }
        };
        fetch(b0);

        // ---- the queries' two parts, scaled to 2^14 .. 2^15 by a power of two
        half8 qh[S], ql[S];
        float c_row = 0.0f;
        {
            const float *qp = a.q + (size_t)(x.k.first + token) * a.q_stride + (size_t)head * D + 8 * half;
            float top = 0.0f;
            bool fine = true;
#pragma unroll
            for (int s = 0; s < D / 16; s++) {
                const float4 v = *reinterpret_cast<const float4 *>(qp + 16 * s), w = *reinterpret_cast<const float4 *>(qp + 16 * s + 4);
                const float e[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    top = fmaxf(top, fabsf(e[i]));
                    fine &= fabsf(e[i]) <= 3.402823466e38f;
                }
            }
            const bool bad = row_max2(fine ? 0.0f : 1.0f) > 0.0f;
            top = row_max2(top);
            int e = 0;
            (void)frexpf(top, &e);
            e = top > 0.0f ? 15 - e : 0;
            c_row = bad ? __builtin_nanf("") : ldexpf(fabsf(a.scale2), -e);
            const bool minus = a.scale2 < 0.0f;  // (the logits' factor is not negative: the largest stays it)
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float *p = qp + 16 * (cut * S + s);
                const float4 v = *reinterpret_cast<const float4 *>(p), w = *reinterpret_cast<const float4 *>(p + 4);
                const float f[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = bad ? 0.0f : ldexpf(minus ? -f[i] : f[i], e);
                    qh[s][i] = (_Float16)y;
                    ql[s][i] = (_Float16)(y - (float)qh[s][i]);
                }
            }
        }
        f32x16 o[CB];
#pragma unroll
        for (int i = 0; i < CB; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[i][j] = 0.0f;
        float m = kNegInf, l = 0.0f, mo = kNegInf;

        lds_barrier();  // (the last segment's readers of s_kv)
        stage(b0);
        ks_l = ks_n, lv_l = lv_n;
        fetch(b0 + 1);
        lds_barrier();
        for (uint32_t j = b0; j < b1; j++) {
            if ((j - b0) % kWave == 0) ks_l = ks_n, lv_l = lv_n;
            stage(j + 1);
            fetch(j + 2);
            const half8 *kv = s_kv[(j - b0) % 2];
            const bool on = !idle && (int)(j * kKvBlock) <= pos1 && (int)(j * kKvBlock + kKvBlock) > low0;
            f32x16 acc;
            Feed keys, values;
#pragma unroll
            for (int e = 0; e < 16; e++) acc[e] = 0.0f;
            if (on) {
                keys.open(kv + cut * S * kWave + lane);
                keys.run<S>([&](int s, half8 k) {
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[s], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[s], acc, 0, 0, 0);
                });
            }
            if (SPLIT > 1) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s_x[(wave * 4 + e) * kWave + lane] = f32x4{acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]};
                lds_barrier();
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f32x4 v = s_x[((wave ^ 1) * 4 + e) * kWave + lane];
#pragma unroll
                    for (int f = 0; f < 4; f++) acc[4 * e + f] += v[f];
                }
            }
            if (on) {
                values.open(kv + 4 * D + cut * CB * 2 * kWave + lane);  // (there by the time of the weights)
                const float ks = __uint_as_float(from_lane(__float_as_uint(ks_l), (j - b0) % kWave));
                const float lv = __uint_as_float(from_lane(__float_as_uint(lv_l), (j - b0) % kWave));
                // keys 32 j + 4 half + 8 (e / 4) + e % 4
                const bool edge = (int)(j * kKvBlock + kKvBlock - 1) > pos0 || (int)(j * kKvBlock) < low1;
                if (edge) {
                    const int key0 = in_branch((int)(j * kKvBlock + 4 * half));
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int key = key0 + 8 * (e / 4) + e % 4;
                        if (key > pos || key < low) acc[e] = kNegInf;
                    }
                }
                const float c = c_row * ks;
                float mb = acc[0];
#pragma unroll
                for (int e = 1; e < 16; e++) mb = fmaxf(mb, acc[e]);
                mb = row_max2(mb);
                mb = mb == kNegInf ? mb : mb * c;
                if (__any(mb > m + kSlack || mb + lv > mo + kSlack)) {
                    const float m1 = fmaxf(m, mb), mo1 = fmaxf(mo, mb + lv);
                    l *= __builtin_amdgcn_exp2f(m - (m1 == kNegInf ? 0.0f : m1));  // (0 before the first key)
                    const float fall = mo == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mo - mo1);
#pragma unroll
                    for (int k = 0; k < CB; k++) o[k] *= fall;
                    m = m1, mo = mo1;
                }
                const float ms = m == kNegInf ? 0.0f : m;  // (no key yet)
                // (a weight of less than 2^-60 of the largest need not be that small among the sums, but counts in l)
                float eb = fmaxf(lv - mo, -60.0f - ms) + kBits;
                if (lv != lv) eb = lv;
                float p[16], sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(acc[e], c, eb));
                if (edge) {
                    const float none = in_branch(kNegInf);
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (acc[e] == none) p[e] = 0.0f;  // (what is not seen adds nothing, whatever its scale)
                }
#pragma unroll
                for (int e = 0; e < 16; e++) sum += p[e];
                if (sum != 0.0f) l += sum * __builtin_amdgcn_exp2f(-eb - ms);  // (0: none in sight, and eb may be NaN)
                // operand u: the keys 4 half + 16 u' + 8 u .. + 3 for u' = 0, 1, as a value's codes lie
                half8 ph[2], pl[2];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int w = e / 4 % 2, i = e % 4 + 4 * (e / 8);
                    const half2v hi = pair(p[e], p[e + 1]);
                    const half2v lo = pair(rest0(hi, p[e]), rest1(hi, p[e + 1]));
                    ph[w][i] = hi[0], ph[w][i + 1] = hi[1];
                    pl[w][i] = lo[0], pl[w][i + 1] = lo[1];
                }
                values.run<2 * CB>([&](int i, half8 v) {
                    o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[i % 2], o[i / 2], 0, 0, 0);
                    o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[i % 2], o[i / 2], 0, 0, 0);
                });
            }
            lds_barrier();
        }
        l += __shfl_xor(l, 32, kWave);

        // ---- a row's channels: 32 k + 8 i + 4 half .. + 3 of the wavefront's
        const bool valid = rg * 32 + n < x.rows;
        float *out = a.out + ((size_t)(x.k.first + token) * a.n_heads + head) * D + cut * Sh::DW + 4 * half;
        const auto write = [&](float scale) {
            if (!valid) return;
#pragma unroll
            for (int k = 0; k < CB; k++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<f32x4 *>(out + 32 * k + 8 * i) =
                        f32x4{o[k][4 * i], o[k][4 * i + 1], o[k][4 * i + 2], o[k][4 * i + 3]} * scale;
        };
        if (whole) {
            write(x.k.bad ? __builtin_nanf("") : out_scale(m, l, mo, kBits));
            u = next;
            continue;
        }
        // ---- a part: piece f's is its second place, later ones' their first
        const uint64_t end = first + (x.hi - x.lo);
        uint32_t f = (uint32_t)(first * pieces / total), g = (uint32_t)((end - 1) * pieces / total);
        while (f + 1 < pieces && total * (f + 1) / pieces <= first) f++;
        while (g + 1 < pieces && total * (g + 1) / pieces <= end - 1) g++;
        const uint32_t parts = g - f + 1, me = piece - f;
        const Shared shared(a.part, 2 * a.pieces * Sh::kPart);
        const auto place = [&](uint32_t i) { return 2 * (f + i) + (i == 0); };
        const auto put = [&](uint32_t slot) {
            const uint32_t to = slot * Sh::kPart + wave * ((CB * 4 + 1) * kWave * 4) + lane * 4;
#pragma unroll
            for (int k = 0; k < CB; k++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    shared.put(to + (k * 4 + i) * (kWave * 4), f32x4{o[k][4 * i], o[k][4 * i + 1], o[k][4 * i + 2], o[k][4 * i + 3]});
            shared.put(to + CB * 4 * (kWave * 4), f32x4{m, l, mo, 0.0f});
        };
        const auto join = [&](uint32_t from, uint32_t step, uint32_t count) {
#pragma unroll
            for (int k = 0; k < CB; k++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[k][j] = 0.0f;
            m = kNegInf, mo = kNegInf, l = 0.0f;
            for (uint32_t i = 0; i < count; i++) {
                const uint32_t p = place(from + i * step) * Sh::kPart + wave * ((CB * 4 + 1) * kWave * 4) + lane * 4;
                f32x4 v[CB * 4];
#pragma unroll
                for (int k = 0; k < CB * 4; k++) v[k] = shared.get(p + k * (kWave * 4));
                const f32x4 st = shared.get(p + CB * 4 * (kWave * 4));
                const float m1 = fmaxf(m, st[0]), mo1 = fmaxf(mo, st[2]);
                l *= m == kNegInf ? 1.0f : exp2f(m - m1);  // (l is 0 or NaN then)
                l += st[0] == kNegInf ? st[1] : st[1] * exp2f(st[0] - m1);
                const float fa = mo == kNegInf ? 1.0f : exp2f(mo - mo1), fb = st[2] == kNegInf ? 1.0f : exp2f(st[2] - mo1);
#pragma unroll
                for (int k = 0; k < CB * 4; k++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[k / 4][k % 4 * 4 + e] = o[k / 4][k % 4 * 4 + e] * fa + v[k][e] * fb;
                m = m1, mo = mo1;
            }
        };
        // A part's stores are acknowledged before it counts; the one that counts last reads
        // past the L2s, and leaves the counter at zero.
        const auto last = [&](uint32_t *ticket, uint32_t count) -> bool {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                const bool is = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
                if (is) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                s_last = is;
            }
            __syncthreads();
            const bool is = s_last;
            __syncthreads();
            return is;
        };
        put(place(me));
        const uint32_t groups = (parts + kJoin - 1) / kJoin, each = (parts + groups - 1) / groups;
        const uint32_t g0 = me / each * each, count = parts - g0 < each ? parts - g0 : each;
        const uint32_t used = (parts + each - 1) / each;
        if (last(a.tickets + place(g0), count)) {
            join(g0, 1, count);
            bool done = used == 1;
            if (!done) {  // (the group's first place now holds the group's sums: every wavefront has read its own there)
                put(place(g0));
                done = last(a.tickets + 2 * a.pieces + f, used);
                if (done) join(0, each, used);
            }
            if (done) write(out_scale(m, l, mo, kBits));
        }
        u = next;
    }
}

template <int D>
hipError_t go(const AttnArgs &a, hipStream_t s) {
    WideArgs t{};
    t.codes = a.kv.codes, t.scales = a.kv.scales, t.n_blocks = a.kv.n_blocks, t.n_kv = a.kv.n_kv, t.b = a.b;
    t.q = a.q, t.out = a.out, t.q_stride = a.q_stride, t.n_heads = a.n_heads, t.group = a.group, t.window = a.window;
    t.scale2 = a.scale * 1.4426950408889634f;
    t.part = (float *)a.work, t.tickets = a.tickets, t.err = a.err;
    t.tiles = wide_tiles(a.b.n_tokens, a.b.n_seqs, a.b.max_new, a.group, Shape<D>::kRows);
    const uint32_t fit = 256 * Shape<D>::kPerCu;
    const uint64_t all = (uint64_t)t.tiles * t.n_kv;
    t.pieces = wide_pieces(t.tiles, a.b.n_seqs, t.n_kv, fit);
    if (all * Shape<D>::kThreads >= (1ull << 32)) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(k_attention_wide<D>, dim3(t.pieces ? fit : (uint32_t)all), dim3(Shape<D>::kThreads), 0, s, t);
    return hipGetLastError();
}

template <int D>
size_t workspace() { return 2ull * 256 * Shape<D>::kPerCu * Shape<D>::kPart * 4; }

}  // namespace

size_t attention_wide_workspace(uint32_t D) {
    switch (D) {
    case 64: return workspace<64>();
    case 96: return workspace<96>();
    case 128: return workspace<128>();
    case 192: return workspace<192>();
    case 256: return workspace<256>();
    case 512: return workspace<512>();
    default: return 0;
    }
}

hipError_t launch_attention_wide(const AttnArgs &a, hipStream_t s) {
    switch (a.kv.D) {
    case 64: return go<64>(a, s);
    case 96: return go<96>(a, s);
    case 128: return go<128>(a, s);
    case 192: return go<192>(a, s);
    case 256: return go<256>(a, s);
    case 512: return go<512>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lt
