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
// 2^(s - m) * 2^(m + log2(scale) - mo), at most 1, times 2^15 to use f16's range.
#include "llmtoy_hip.h"
#include "lt_kv.h"

namespace lt {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kThinWaves = 4, kThinRows = 16;
// Workgroups that a launch's work is split into, where there are fewer tiles: two
// on each CU.
constexpr uint32_t kThinTarget = 512;
// Blocks a workgroup takes at least: one a wavefront.
constexpr uint32_t kThinBlocks = kThinWaves;

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
    float *part;   // [slots][16][D + 4]: sums, then m, l, mo
    uint32_t slots;
    uint32_t *err;
};

// A byte code + 128 is the f16 number 1024 + 128 + code with the byte 0x64 above it.
__device__ __forceinline__ half8 codes8(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        half2v h[4];
        half8 v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - off;
    return r.v;
}

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
    t.tiles = (n * a.group + kThinRows - 1) / kThinRows;
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
    bool any;
};

// Blocks a part: all of the batch's over the launch's workgroups, evenly.  Every
// wavefront finds it for itself from the lengths (one load and a sum for up to 64
// sequences).
__device__ __forceinline__ uint32_t thin_share(const ThinArgs &a) {
    float sum = 0.0f;  // (a count beyond 2^24 need not be exact)
    for (uint32_t r = threadIdx.x % kWave; r < a.b.n_seqs; r += kWave) {
        const ThinRow t = thin_row(a, r);
        if (t.k.falls && blockIdx.x == 0 && blockIdx.y == 0) kv_report(a.err, kKvErrRows, r);
        sum += (float)t.tiles * (float)t.blocks;
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    const float each = ceilf(sum * (float)a.n_kv / (float)kThinTarget);
    return each < (float)kThinBlocks ? kThinBlocks : each > 1e9f ? 1000000000u : (uint32_t)each;
}

__device__ __forceinline__ ThinWork thin_work(const ThinArgs &a, uint32_t index) {
    ThinWork w{};
    const uint32_t lane = threadIdx.x % kWave, share = thin_share(a);
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
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const uint32_t p = __shfl_up(up, off, kWave), q = __shfl_up(pup, off, kWave);
            if ((int)lane >= off) up += p, pup += q;
        }
        const uint32_t before = seen + up - mine;
        const uint64_t has = __ballot(index >= before && index < before + mine);
        if (has) {
            const int l = __builtin_ctzll(has);
            const uint32_t in = index - __shfl(before, l, kWave);
            w.any = true;
            w.row = r0 + l;
            w.splits = __shfl(splits, l, kWave);
            w.tile = in / w.splits;
            w.split = in % w.splits;
            const uint32_t lo = __shfl(t.lo, l, kWave), blocks = __shfl(t.blocks, l, kWave);
            // as even as whole blocks go
            w.b0 = lo + (uint32_t)((uint64_t)blocks * w.split / w.splits);
            w.b1 = lo + (uint32_t)((uint64_t)blocks * (w.split + 1) / w.splits);
            w.slot = joined + __shfl(pup - parts, l, kWave) + in;
            return w;
        }
        seen += __shfl(up, kWave - 1, kWave);
        joined += __shfl(pup, kWave - 1, kWave);
    }
    return w;
}

template <int D>
__global__ __launch_bounds__(kThinWaves *kWave, D <= 128 ? 2 : 1) void k_attention_thin(ThinArgs a) {
    constexpr int C = D / 32, P = D + 4;  // P: floats of a joined row
    __shared__ __align__(16) float s_o[kThinWaves][kThinRows][D + 4];
    __shared__ float s_m[3][kThinWaves][kThinRows];
    const uint32_t lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), h = blockIdx.y;
    ThinWork w = thin_work(a, blockIdx.x);
    if (!w.any) return;
    w.tile = __builtin_amdgcn_readfirstlane(w.tile), w.b0 = __builtin_amdgcn_readfirstlane(w.b0);
    w.b1 = __builtin_amdgcn_readfirstlane(w.b1);
    const uint32_t row = __builtin_amdgcn_readfirstlane(w.row);
    const ThinRow tr = thin_row(a, row);
    const uint32_t rows = tr.k.n * a.group - w.tile * kThinRows;  // of this tile (more: 16)
    const uint32_t rho = w.tile * kThinRows + (n < rows ? n : 0);
    const uint32_t token = rho / a.group, head = h * a.group + rho % a.group;
    const int pos = (int)(tr.k.len - tr.k.n + token);
    const int low = a.window && (uint32_t)pos + 1 > a.window ? pos + 1 - (int)a.window : 0;
    // positions that every row of the tile sees the keys between
    const uint32_t tok0 = w.tile * kThinRows / a.group, rows_in = rows < kThinRows ? rows : kThinRows;
    const uint32_t tok1 = (w.tile * kThinRows + rows_in - 1) / a.group;
    const int pos0 = (int)(tr.k.len - tr.k.n + tok0), pos1 = (int)(tr.k.len - tr.k.n + tok1);
    const int low1 = a.window && (uint32_t)pos1 + 1 > a.window ? pos1 + 1 - (int)a.window : 0;
    const int low0 = a.window && (uint32_t)pos0 + 1 > a.window ? pos0 + 1 - (int)a.window : 0;
    uint32_t b0 = w.b0, b1 = w.b1;
    if (!tr.k.bad) {
        b0 = max(b0, (uint32_t)low0 / kKvBlock);
        b1 = min(b1, (uint32_t)pos1 / kKvBlock + 1);
    } else {
        b1 = b0;
        if (threadIdx.x == 0 && h == 0) kv_report(a.err, kKvErrRows, row);
    }
    const uint32_t *table = a.b.table + (size_t)row * a.b.max_blocks;

    // the queries' two parts, scaled to 2^14 .. 2^15 by a power of two
    half8 qh[C], ql[C];
    float c_row;
    {
        const float *qp = a.q + (size_t)(tr.k.first + token) * a.q_stride + (size_t)head * D + 8 * g;
        float x[C][8];
        float top = 0.0f;
        bool fine = true;
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
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        int bad = !fine;
        bad |= __shfl_xor(bad, 16, kWave);
        bad |= __shfl_xor(bad, 32, kWave);
        int e = 0;
        (void)frexpf(top, &e);
        e = top > 0.0f ? 15 - e : 0;
        c_row = bad ? __builtin_nanf("") : ldexpf(a.scale2, -e);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = bad ? 0.0f : ldexpf(x[c][i], e);
                const _Float16 hi = (_Float16)y;
                qh[c][i] = hi;
                ql[c][i] = (_Float16)(y - (float)hi);
            }
    }

    f32x4 o[2 * C];
#pragma unroll
    for (int i = 0; i < 2 * C; i++) o[i] = f32x4{0, 0, 0, 0};
    float m = kNegInf, l = 0.0f, mo = kNegInf;

    const auto page_of = [&](uint32_t j) -> uint32_t { return j < b1 ? __builtin_amdgcn_readfirstlane(table[j]) : 0; };
    uint4 kq[C], vq[C];
    float2 sc;
    const auto at = [&](uint32_t page) {
        const size_t b = (size_t)(page < a.n_blocks ? page : 0) * a.n_kv + h;
        return b;
    };
    const auto load = [&](uint4 *to, size_t b, int which) {
        const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + (b * 2 + which) * (kKvBlock * D)) + lane;
#pragma unroll
        for (int c = 0; c < C; c++) to[c] = p[c * kWave];
    };
    uint32_t j = b0 + wave;
    uint32_t page = page_of(j), next = page_of(j + kThinWaves);
    if (j < b1) {
        sc = a.scales[at(page)];
        load(kq, at(page), 0);
        load(vq, at(page), 1);
    }
    for (; j < b1; j += kThinWaves) {
        const bool more = j + kThinWaves < b1;
        float2 s = sc;
        if (page >= a.n_blocks) {
            s.x = s.y = __builtin_nanf("");
            if (lane == 0 && h == 0) kv_report(a.err, kKvErrBlock, row);
        }
        f32x4 sa[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}, sb[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int c = 0; c < C; c++) {
            const half8 k0 = codes8(kq[c].x, kq[c].y), k1 = codes8(kq[c].z, kq[c].w);
            sa[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[c], sa[0], 0, 0, 0);
            sa[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[c], sa[1], 0, 0, 0);
            sb[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[c], sb[0], 0, 0, 0);
            sb[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[c], sb[1], 0, 0, 0);
        }
        const uint32_t after = page_of(j + 2 * kThinWaves);
        if (more) {
            sc = a.scales[at(next)];
            load(kq, at(next), 0);
        }
        // logits of keys 32 j + 16 (e / 4) + 4 g + e % 4, base 2
        float t[8];
        const float c = c_row * s.x;
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = (sa[e / 4][e % 4] + sb[e / 4][e % 4]) * c;
        const int key = (int)(j * kKvBlock + 4 * g);
        const bool edge = (int)(j * kKvBlock + kKvBlock - 1) > pos0 || (int)(j * kKvBlock) < low1;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at_key = key + 16 * (e / 4) + e % 4;
                if (at_key > pos || at_key < low) t[e] = kNegInf;
            }
        }
        float mb = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        mb = fmaxf(mb, __shfl_xor(mb, 16, kWave));
        mb = fmaxf(mb, __shfl_xor(mb, 32, kWave));
        const float m1 = fmaxf(m, mb);
        const float ms = m1 == kNegInf ? 0.0f : m1;  // (no key yet)
        const float lv = log2f(s.y);
        const float mo1 = fmaxf(mo, mb + lv);
        float p[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = exp2f(t[e] - ms);
            sum += p[e];
        }
        l = l * exp2f(m - ms) + sum;
        m = m1;
        // weights' factor: at most 2^15 for the largest; a block of zeros adds nothing
        const float up = ms + lv - mo1;
        float f = mo1 == kNegInf ? 0.0f : exp2f(fminf(up, 126.0f)) * 32768.0f;
        if (s.y != s.y) f = s.y;
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] *= f;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (t[e] == kNegInf) p[e] = 0.0f;  // (what is not seen adds nothing, whatever its scale)
        }
        if (__any(mo1 > mo)) {
            const float fall = mo == kNegInf ? 0.0f : exp2f(mo - mo1);
#pragma unroll
            for (int i = 0; i < 2 * C; i++) o[i] *= fall;
        }
        mo = mo1;
        half8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const _Float16 hi = (_Float16)p[e];
            ph[e] = hi;
            pl[e] = (_Float16)(p[e] - (float)hi);
        }
#pragma unroll
        for (int i = 0; i < C; i++) {
            const half8 v0 = codes8(vq[i].x, vq[i].y), v1 = codes8(vq[i].z, vq[i].w);
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * i], 0, 0, 0);
            o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * i + 1], 0, 0, 0);
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl, o[2 * i], 0, 0, 0);
            o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl, o[2 * i + 1], 0, 0, 0);
        }
        if (more) load(vq, at(next), 1);
        page = next;
        next = after;
    }
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);

    // the four wavefronts' parts joined through LDS
    if (g == 0) s_m[0][wave][n] = m, s_m[1][wave][n] = l, s_m[2][wave][n] = mo;
#pragma unroll
    for (int i = 0; i < 2 * C; i++) *reinterpret_cast<f32x4 *>(&s_o[wave][n][16 * i + 4 * g]) = o[i];
    __syncthreads();
    // a row's channels over 16 threads
    const uint32_t rr = threadIdx.x / 16, part = threadIdx.x % 16;
    if (rr >= rows_in) return;
    float mt = kNegInf, mot = kNegInf;
#pragma unroll
    for (int i = 0; i < kThinWaves; i++) mt = fmaxf(mt, s_m[0][i][rr]), mot = fmaxf(mot, s_m[2][i][rr]);
    float lt_ = 0.0f, fo[kThinWaves];
#pragma unroll
    for (int i = 0; i < kThinWaves; i++) {
        const float mi = s_m[0][i][rr], moi = s_m[2][i][rr], li = s_m[1][i][rr];
        lt_ += mi == kNegInf ? (li != li ? li : 0.0f) : li * exp2f(mi - mt);
        fo[i] = moi == kNegInf ? 0.0f : exp2f(moi - mot);
    }
    // (a NaN among the sums goes through: 0 times it is NaN)
    const uint32_t r1 = w.tile * kThinRows + rr;
    float *out = a.out + ((size_t)(tr.k.first + r1 / a.group) * a.n_heads + h * a.group + r1 % a.group) * D;
    float *to = w.splits > 1 ? a.part + (((size_t)h * a.slots + w.slot) * kThinRows + rr) * P : out;
    float scale = 1.0f;
    if (w.splits == 1) scale = tr.k.bad ? __builtin_nanf("") : lt_ > 0.0f || lt_ != lt_ ? (mot == kNegInf ? 0.0f : exp2f(mot - mt - 15.0f)) / lt_ : 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
        const uint32_t d = 4 * (part + 16 * i);
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < kThinWaves; u++) sum += *reinterpret_cast<const f32x4 *>(&s_o[u][rr][d]) * fo[u];
        *reinterpret_cast<f32x4 *>(to + d) = sum * scale;
    }
    if (D % 64 && part < 8) {
        const uint32_t d = D / 64 * 64 + 4 * part;
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < kThinWaves; u++) sum += *reinterpret_cast<const f32x4 *>(&s_o[u][rr][d]) * fo[u];
        *reinterpret_cast<f32x4 *>(to + d) = sum * scale;
    }
    if (w.splits > 1 && part == 0) to[D] = mt, to[D + 1] = lt_, to[D + 2] = mot;
}

// Joins the parts of the tiles that were split: a workgroup a tile (the one that
// would have been its first part) and head, 16 threads a row.
template <int D>
__global__ __launch_bounds__(256) void k_attention_join(ThinArgs a) {
    constexpr int P = D + 4;
    const uint32_t h = blockIdx.y;
    const ThinWork w = thin_work(a, blockIdx.x);
    if (!w.any || w.splits < 2 || w.split) return;
    const ThinRow tr = thin_row(a, w.row);
    const uint32_t rows = tr.k.n * a.group - w.tile * kThinRows, rr = threadIdx.x / 16, part = threadIdx.x % 16;
    if (rr >= rows) return;
    const float *from = a.part + (((size_t)h * a.slots + w.slot) * kThinRows + rr) * P;
    float mt = kNegInf, mot = kNegInf;
    for (uint32_t i = 0; i < w.splits; i++) {
        const float *p = from + (size_t)i * kThinRows * P;
        mt = fmaxf(mt, p[D]), mot = fmaxf(mot, p[D + 2]);
    }
    f32x4 sum[(D + 63) / 64];
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; k++) sum[k] = f32x4{0, 0, 0, 0};
    float l = 0.0f;
    for (uint32_t i = 0; i < w.splits; i++) {
        const float *p = from + (size_t)i * kThinRows * P;
        const float mi = p[D], li = p[D + 1], moi = p[D + 2];
        l += mi == kNegInf ? (li != li ? li : 0.0f) : li * exp2f(mi - mt);
        const float f = moi == kNegInf ? 0.0f : exp2f(moi - mot);
#pragma unroll
        for (int k = 0; k < (D + 63) / 64; k++) {
            const uint32_t d = 4 * (part + 16 * k);
            if (d < D) sum[k] += *reinterpret_cast<const f32x4 *>(p + d) * f;
        }
    }
    const float scale = l > 0.0f || l != l ? (mot == kNegInf ? 0.0f : exp2f(mot - mt - 15.0f)) / l : 0.0f;
    const uint32_t r1 = w.tile * kThinRows + rr;
    float *out = a.out + ((size_t)(tr.k.first + r1 / a.group) * a.n_heads + h * a.group + r1 % a.group) * D;
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; k++) {
        const uint32_t d = 4 * (part + 16 * k);
        if (d < D) *reinterpret_cast<f32x4 *>(out + d) = sum[k] * scale;
    }
}

// Workgroups of a head: a tile more or less a sequence, and the parts of those
// that are split (at most the target and one more a tile).
uint32_t thin_tiles(const AttnArgs &a) {
    const uint64_t rows = (uint64_t)a.b.n_tokens * a.group;
    uint64_t tiles = rows / kThinRows + a.b.n_seqs;
    if (a.b.max_new) {
        const uint64_t most = (uint64_t)a.b.n_seqs * (((uint64_t)a.b.max_new * a.group + kThinRows - 1) / kThinRows);
        if (most < tiles) tiles = most;
    }
    if (rows < tiles) tiles = rows;
    return (uint32_t)tiles;
}
uint32_t thin_slots(uint32_t n_kv) { return 2 * (kThinTarget / n_kv + 1) + 2; }

template <int D>
void go(const ThinArgs &t, uint32_t tiles, hipStream_t s) {
    const dim3 grid(tiles + kThinTarget / t.n_kv + 1, t.n_kv);
    hipLaunchKernelGGL(k_attention_thin<D>, grid, dim3(kThinWaves * kWave), 0, s, t);
    hipLaunchKernelGGL(k_attention_join<D>, grid, dim3(256), 0, s, t);
}

}  // namespace

bool attention_head_dim(uint32_t D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256 || D == 512; }

size_t attention_workspace(const AttnArgs &a) {
    return (size_t)a.kv.n_kv * thin_slots(a.kv.n_kv) * kThinRows * (a.kv.D + 4) * 4;
}

hipError_t launch_attention(const AttnArgs &a, hipStream_t s) {
    ThinArgs t{};
    t.codes = a.kv.codes, t.scales = a.kv.scales, t.n_blocks = a.kv.n_blocks, t.n_kv = a.kv.n_kv, t.b = a.b;
    t.q = a.q, t.out = a.out, t.q_stride = a.q_stride, t.n_heads = a.n_heads, t.group = a.group, t.window = a.window;
    t.scale2 = a.scale * 1.4426950408889634f;
    t.part = (float *)a.work, t.slots = thin_slots(t.n_kv), t.err = a.err;
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
