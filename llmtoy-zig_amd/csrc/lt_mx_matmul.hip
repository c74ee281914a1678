// lt_mx_matmul.hip -- products of an MXFP4 matrix with many vectors:
// out[t][r] = sum_c W[r][c] X[t][c].
//
// X in fp32: a first launch turns its blocks into limbs (lt_mx.h) laid out as
// matrix operands, and the product runs one matrix instruction a limb into the
// same sums.  X as an MXFP4 tensor: its codes and scales are an operand already.
// (Up to five vectors of fp32 that fit the LDS go to the matvec's kernel.)
//
// What bounds it.  4096 vectors by 8192 x 4096: 1.37 PFLOP of FP6 x FP4
// products; the instructions alone, their operands held in registers, take 238
// us at the clock that the card holds under them (5.8 PFLOP/s; 8.9 with
// constant operands), the product with its loads from LDS 253 us, the whole
// kernel 294 to 309 us (cards differ), and the limbs 21 us before it (130 MB, 6.2
// TB/s).  With 4-bit X 82 us, of which the instructions alone take 61.  Middle sizes
// are bound by how their tiles fall on the CUs: 509 x 4864 x 2816 is 152 of them on
// 256 CUs, 27 us and the limbs 7 (smaller tiles, which need more waves or leave a
// SIMD with one, 32.5 to 56 us in all against 31.6).
//
// What made it fast, on that size: both operands through LDS by direct loads
// instead of registers (1570 -> 335 us); uniform addresses that move on by one
// addition a load, where computing each address anew had cost more issue slots
// than the matrix instructions (a 256 x 64 tile's stage from 0.80 to 0.60 us);
// 512 x 128 tiles with three stages (326 -> 316).  Holding the next stage's
// operands in registers besides, s_setprio and forced interleaving changed
// nothing or cost.
#include "llmtoy_hip.h"
#include "lt_internal.h"
#include "lt_mx.h"

#include <type_traits>

namespace lt {

namespace {

// The workspace of T vectors, in tiles of 64: the limbs as operands of
// v_mfma_scale_f32_32x32x64 (a lane holds one block of one vector),
//   [tile][pair of blocks][2 halves of the tile][5 limbs][64 lanes] 16 B, then the same of 8 B
// 15 KiB for a pair, in a row; and scale words as a tensor's.
constexpr size_t kPairBytes = 2 * kMxLimbs * 64 * 24;
constexpr size_t kPairLo = 2 * kMxLimbs * 64 * 16;
struct MxLimbs {
    uint8_t *data;    // [tile][2 kg] pairs
    uint8_t *scales;  // [tile of 16][kq][64][4]
};
__host__ __device__ inline size_t limb_tiles(size_t T) { return (T + 63) / 64; }
size_t limb_data_bytes(const MxDims &d, size_t T) { return limb_tiles(T) * 2 * d.kg * kPairBytes; }
// the last loads of a product run past the data by up to kStages pairs
constexpr int kStages = 4;
size_t limb_scales_at(const MxDims &d, size_t T) { return limb_data_bytes(d, T) + kStages * kPairBytes; }
size_t limb_bytes(const MxDims &d, size_t T) { return limb_scales_at(d, T) + limb_tiles(T) * 4 * d.kq * 256 + kStages * 256; }

// A thread a block; vectors from T on and blocks from nb on are zeros.  One wave a
// workgroup: few vectors reach more CUs (509 x 2816 6.4 -> 6.0 us, 7 x 4096 2.2 ->
// 1.8).  Coalesced loads through LDS and stores past the caches gave nothing.
constexpr int kLimbThreads = 64;
__global__ __launch_bounds__(kLimbThreads) void k_mx_limbs(const float *__restrict__ X, uint32_t T, MxDims d, MxLimbs p) {
    const size_t id = (size_t)blockIdx.x * kLimbThreads + threadIdx.x;
    const uint32_t lane = (uint32_t)(id % 64), half = (uint32_t)(id / 64 % 2);
    const size_t pair = id / 128;  // over tiles and pairs
    if (pair >= limb_tiles(T) * 2 * d.kg) return;
    const uint32_t b = (uint32_t)(pair % (2 * d.kg)) * 2 + lane / 32;
    const size_t t = pair / (2 * d.kg) * 64 + half * 32 + lane % 32;
    mx_f32x16 lo = {}, hi = {};
    if (t < T && b < d.nb) mx_load_block(X + (t * d.nb + b) * 32, lo, hi);
    const uint32_t s = mx_limb_scale(mx_top(lo, hi));
    p.scales[mx_scale_at(d, t / 16, (uint32_t)(t % 16), b)] = (uint8_t)s;
    uint8_t *at = p.data + pair * kPairBytes;
    mx_u32x4 *w16 = reinterpret_cast<mx_u32x4 *>(at) + half * kMxLimbs * 64 + lane;
    mx_u32x2 *w8 = reinterpret_cast<mx_u32x2 *>(at + kPairLo) + half * kMxLimbs * 64 + lane;
    mx_limbs(lo, hi, s, [&](int j, const mx_u32x6 &q) {
        w16[j * 64] = mx_u32x4{q[0], q[1], q[2], q[3]};
        w8[j * 64] = mx_u32x2{q[4], q[5]};
    });
}

typedef const __attribute__((address_space(1))) void *mx_gptr;
typedef __attribute__((address_space(3))) void *mx_lptr;
// 64 lanes x 16 bytes from each lane's address to LDS at dst (the wave's), in lane order.
__device__ __forceinline__ void to_lds(const uint8_t *src, uint8_t *dst) {
    __builtin_amdgcn_global_load_lds((mx_gptr)src, (mx_lptr)dst, 16, 0, 0);
}

// One operand of the product: a tensor's codes, or the limbs; and its scales.
struct MxSide {
    const uint8_t *data, *scales;
    uint32_t last;  // the last tile of 32 rows (its second half may be past the rows: allocated, not used)
};

// out[t][r]: a workgroup of WR x WC waves computes 32 WR MI rows of W by 32 WC NI
// vectors, a wave MI x NI tiles of 32 x 32; a stage is a pair of blocks (64
// columns) of both sides, of which NST are in LDS.  The vectors are the
// instruction's rows and W's rows its columns: a store of sums is then 32
// neighbouring rows of out for each of two vectors, whatever rows % 4 is.
template <int NL, int WR, int WC, int MI, int NI, int NST>
struct MxTile {
    static constexpr int kWaves = WR * WC, kRows = WR * MI, kVecs = WC * NI;  // tiles of 32
    // a stage in KiB: W's codes, its scale words (256 B a tile), X's operands, its scale words
    static constexpr int kWS = kRows, kX = kWS + (kRows + 3) / 4;
    static constexpr int kXS = kX + (NL == 1 ? kVecs : (kVecs + 1) / 2 * 15), kChunks = kXS + (kVecs + 3) / 4;
    static constexpr int kEach = (kChunks + kWaves - 1) / kWaves;  // loads of a wave for a stage
    static_assert((NST - 2) * kEach < 64, "the count of loads in flight");
    static_assert(NST <= kStages, "the memory that the last loads run into");
};

constexpr size_t kStageSums = 12 << 20;  // 48 MiB

// Until this wave has at most N loads in flight and no LDS access; then, behind
// the barrier, every wave of the workgroup.
template <int N>
__device__ __forceinline__ void arrive() {
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | N >> 4 << 14);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int NL, int WR, int WC, int MI, int NI, int NST>
__global__ __launch_bounds__(64 * WR * WC, 2) void k_mx_gemm(MxSide w, MxSide x, uint32_t kg, uint32_t kq, uint32_t rows,
                                                             uint32_t T, uint32_t grid_m, uint32_t grid_n, float *out) {
    using L = MxTile<NL, WR, WC, MI, NI, NST>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[NST * L::kChunks * 1024];
    const uint32_t lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wc = wave / WR;
    // blocks of one XCD (equal index % 8) take neighbouring tiles, 8 of W's by as many of X's
    const uint32_t per = (grid_m * grid_n + 7) / 8;
    const uint32_t id = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (id >= grid_m * grid_n) return;
    const uint32_t band = id / (8 * grid_n) * 8, wide = min(8u, grid_m - band), in = id % (8 * grid_n);
    const uint32_t m0 = (band + in % wide) * L::kRows, n0 = in / wide * L::kVecs;  // in tiles of 32
    const uint32_t steps = 2 * kg;

    // This wave's loads of a stage: a uniform address that moves on from stage
    // to stage, and each lane's offset.
    const uint8_t *src[L::kEach];
    uint32_t off[L::kEach];
    int stride[L::kEach], to[L::kEach];  // stride 0: scale words
#pragma unroll
    for (int i = 0; i < L::kEach; i++) {
        const int c = min(wave + i * L::kWaves, L::kChunks - 1);  // (the last one again, the same bytes)
        to[i] = c * 1024;
        if (c < L::kWS || (NL == 1 && c >= L::kX && c < L::kXS)) {  // codes of a tile of 32
            const MxSide &p = c < L::kWS ? w : x;
            const uint32_t t32 = min(c < L::kWS ? m0 + c : n0 + c - L::kX, p.last);
            src[i] = p.data + (size_t)2 * t32 * kg * 1024;
            off[i] = lane % 32 / 16 * kg * 1024 + lane / 32 * 256 + lane % 16 * 16;
            stride[i] = 512;
        } else if (c >= L::kX && c < L::kXS) {  // limbs: 15 chunks a tile of 64
            const uint32_t t64 = min(n0 / 2 + (c - L::kX) / 15, x.last / 2);
            src[i] = x.data + (size_t)t64 * steps * kPairBytes + (c - L::kX) % 15 * 1024;
            off[i] = lane * 16;
            stride[i] = (int)kPairBytes;
        } else {  // scale words: 16 lanes a tile of 32, [block][row] of the pair
            const bool isw = c < L::kX;
            const MxSide &p = isw ? w : x;
            const uint32_t first = min(isw ? m0 + (c - L::kWS) * 4 : n0 + (c - L::kXS) * 4, p.last);
            const uint32_t in = min(lane / 16, p.last - first);
            src[i] = p.scales + (size_t)2 * first * kq * 256;
            off[i] = (2 * in + lane / 4 % 2) * kq * 256 + lane / 8 % 2 * 64 + lane % 4 * 16;
            stride[i] = 0;
        }
    }
    // (the last stages' loads run past the end by up to NST stages: allocated, not used)
    uint32_t fetched = 0;
    auto fetch_one = [&](int i, uint8_t *dst) { to_lds(src[i] + off[i], dst + to[i]); };
    auto fetch_next = [&](bool odd) {  // odd: the stage just fetched was odd
        fetched++;
        const int sc = !odd || fetched % 8 == 0 ? 128 : -128;
#pragma unroll
        for (int i = 0; i < L::kEach; i++) off[i] += stride[i] ? stride[i] : sc;
    };

    mx_acc32 acc[MI][NI] = {};
    auto operand = [&](const uint8_t *st, int v, int j) {
        if (NL == 1) return mx_op4(*reinterpret_cast<const mx_u32x4 *>(st + (L::kX + v) * 1024 + lane * 16));
        const uint8_t *u = st + L::kX * 1024 + v / 2 * (int)kPairBytes;
        const int o = (v % 2 * kMxLimbs + j) * 64 + lane;
        return mx_op6(reinterpret_cast<const mx_u32x4 *>(u)[o], reinterpret_cast<const mx_u32x2 *>(u + kPairLo)[o]);
    };
    auto step = [&](auto odd, uint32_t pair, const uint8_t *st, uint8_t *dst) {
        constexpr int ODD = decltype(odd)::value;
        const uint32_t shift = pair / 2 % 4 * 8;
        const uint32_t at = lane * 4;  // a lane's scale word
        mx_op b[MI], a[NI], an[NI];
        int sb[MI], sa[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            sa[i] = (int)(*reinterpret_cast<const uint32_t *>(st + L::kXS * 1024 + (wc * NI + i) * 256 + at) >> shift & 255u);
            a[i] = operand(st, wc * NI + i, 0);
        }
#pragma unroll
        for (int i = 0; i < MI; i++) {
            b[i] = mx_op4(*reinterpret_cast<const mx_u32x4 *>(st + (wr * MI + i) * 1024 + lane * 16));
            sb[i] = (int)(*reinterpret_cast<const uint32_t *>(st + L::kWS * 1024 + (wr * MI + i) * 256 + at) >> shift);
        }
#pragma unroll
        for (int j = 0; j < NL; j++) {
            if (j + 1 < NL)
#pragma unroll
                for (int i = 0; i < NI; i++) an[i] = operand(st, wc * NI + i, j + 1);
#pragma unroll
            for (int n = 0; n < NI; n++)
#pragma unroll
                for (int m = 0; m < MI; m++) {
                    acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        a[n], b[m], acc[m][n], NL == 1 ? kMxCbszFp4 : kMxCbszFp6, kMxCbszFp4, 0,
                        sa[n] - (NL == 1 ? 0 : (int)kMxLimbShift[j]), 0, sb[m]);
                    const int k = (j * NI + n) * MI + m + 1, total = NL * NI * MI;
                    if (k * L::kEach / total > (k - 1) * L::kEach / total) {
#pragma unroll
                        for (int i = (k - 1) * L::kEach / total; i < k * L::kEach / total; i++) fetch_one(i, dst);
                    }
                }
#pragma unroll
            for (int i = 0; i < NI; i++) a[i] = an[i];
        }
        fetch_next((NST - 1 + ODD) % 2);
    };

    constexpr int kAhead = (NST - 2) * L::kEach, kStage = L::kChunks * 1024;
    for (int i = 0; i < NST - 1; i++) {
#pragma unroll
        for (int c = 0; c < L::kEach; c++) fetch_one(c, lds + i * kStage);
        fetch_next(i % 2);
    }
    int now = 0, free = NST - 1;
    auto turn = [&](auto odd, uint32_t s) {
        // stage s is in LDS, and every wave is past stage s - 1, whose memory the
        // loads of stage s + NST - 1 take
        arrive<kAhead>();
        step(odd, s, lds + now * kStage, lds + free * kStage);
        free = now;
        now = now + 1 == NST ? 0 : now + 1;
    };
    for (uint32_t s = 0; s < steps; s += 2) {
        turn(std::integral_constant<int, 0>{}, s);
        turn(std::integral_constant<int, 1>{}, s + 1);
    }
    arrive<0>();  // no load into LDS outlives the workgroup

    // Past the caches where the stores are whole lines (4096 x 8192 x 4096 324 ->
    // 316 us, 1024 x 4096 x 4096 with 4-bit X 20.1 -> 19.2).
    const bool lines = rows % 32 == 0 && ((uintptr_t)out & 127) == 0;
    auto store = [&](auto past) {
#pragma unroll
        for (int n = 0; n < NI; n++)
#pragma unroll
            for (int m = 0; m < MI; m++) {
                const uint32_t r = (m0 + wr * MI + m) * 32 + lane % 32;
                if (r >= rows) continue;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const uint32_t t = (n0 + wc * NI + n) * 32 + i / 4 * 8 + 4 * (lane / 32) + i % 4;
                    if (t >= T) continue;
                    float *at = &out[(size_t)t * rows + r];
                    if (decltype(past)::value)
                        __builtin_nontemporal_store(acc[m][n][i], at);
                    else
                        *at = acc[m][n][i];
                }
            }
    };
    if (lines) return store(std::true_type{});
    // (the smallest tiles' products have fewer)
    if (L::kRows * L::kVecs <= 8 || (size_t)T * rows <= kStageSums) return store(std::false_type{});
    // Rows that begin inside a line, and more sums than the L2s put together: the sums
    // of 8 WC vectors at a time pass through LDS, where a vector's lie as its 16-byte
    // pieces of out do, and a wave stores all of them in a row; past the caches but
    // for the lines at both ends.  With 4-bit X, straight from the registers | this:
    // 4095 x 7001 x 2816 67.8 | 62.0 us, 1100 x 30001 x 512 53.7 | 39.3; but 2000 x
    // 5001 x 1024 (40 MB) 17.1 | 17.5, 500 x 4865 x 896 7.0 | 8.8.
    constexpr uint32_t kR = 32 * L::kRows, kPitch = kR + 4;
    static_assert(8 * WC * kPitch * 4 <= sizeof lds, "the sums take the stages' place");
    float *const sums = reinterpret_cast<float *>(lds);
    const int count = (int)min(kR, rows - m0 * 32);
    const uint32_t base = (uint32_t)((uintptr_t)out / 4) + m0 * 32;  // (out is on 16 bytes)
#pragma unroll
    for (int n = 0; n < NI; n++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            if (n || g) arrive<63>();  // (not for the stores)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t v = wc * 8 + 4 * (lane / 32) + j, t = (n0 + wc * NI + n) * 32 + g * 8 + 4 * (lane / 32) + j;
                float *to = sums + v * kPitch + (base + t * rows) % 4 + wr * MI * 32 + lane % 32;
#pragma unroll
                for (int m = 0; m < MI; m++) to[m * 32] = acc[m][n][g * 4 + j];
            }
            arrive<63>();
            for (int v = wave; v < 8 * WC; v += L::kWaves) {
                const uint32_t t = (n0 + v / 8 * NI + n) * 32 + g * 8 + v % 8;
                if (t >= T) continue;
                float *const to = out + (size_t)t * rows + m0 * 32;
                const int q = (int)((base + t * rows) % 4);
                const float *from = sums + v * kPitch;
                for (int i = 4 * (int)lane; i + 4 <= count + q; i += 256) {
                    if (i < q) continue;
                    const mx_acc16 y = *reinterpret_cast<const mx_acc16 *>(from + i);
                    mx_acc16 *at = reinterpret_cast<mx_acc16 *>(to - q + i);
                    const int line = i - q - (int)((uintptr_t)at / 4 % 32);  // where its line begins
                    if (line >= 0 && line + 32 <= count)
                        __builtin_nontemporal_store(y, at);
                    else
                        *at = y;
                }
                // up to 3 at both ends
                const int e = lane < 3 ? (int)lane : (count + q) / 4 * 4 - q + (int)lane - 3;
                if (lane < 6 && e >= 0 && e < count && (lane >= 3 || e < (4 - q) % 4)) to[e] = from[q + e];
            }
        }
}

// Few vectors, or few rows: a workgroup computes 16 RT rows by 16 NT vectors, its
// waves split the columns and their sums meet in LDS.  Nothing is shared between
// the waves, so both operands go from memory to registers, the next group of 4
// blocks while one is computed: no barrier, and every CU has work where the
// tiles above would be too few.
constexpr int kThinWaves = 8;
template <int NL, int RT, int NT>
__global__ __launch_bounds__(64 * kThinWaves, 2) void k_mx_thin(MxSide w, MxSide x, uint32_t kg, uint32_t kq, uint32_t rows,
                                                                uint32_t T, float *out) {
    __shared__ float part[kThinWaves][RT][NT][16][17];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m0 = blockIdx.x * RT, n0 = blockIdx.y * NT;  // in tiles of 16
    const uint32_t each = (kg + kThinWaves - 1) / kThinWaves, g0 = wave * each, g1 = min(g0 + each, kg);
    struct Group {
        mx_op w[RT], x[NL][NT];
        uint32_t sw[RT], sx[NT];
    };
    auto fetch = [&](Group &r, uint32_t g) {
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const size_t tile = min(m0 + i, 2 * w.last + 1);
            r.w[i] = mx_op4(*reinterpret_cast<const mx_u32x4 *>(w.data + (tile * kg + g) * 1024 + lane * 16));
            r.sw[i] = *reinterpret_cast<const uint32_t *>(w.scales + (tile * kq + g / 4) * 256 + lane * 4);
        }
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const size_t tile = min(n0 + i, 2 * x.last + 1);
            r.sx[i] = *reinterpret_cast<const uint32_t *>(x.scales + (tile * kq + g / 4) * 256 + lane * 4);
            if constexpr (NL == 1) {
                r.x[0][i] = mx_op4(*reinterpret_cast<const mx_u32x4 *>(x.data + (tile * kg + g) * 1024 + lane * 16));
            } else {
                const uint8_t *u = x.data + (tile / 4 * 2 * kg + 2 * g + lane / 32) * kPairBytes;
                const uint32_t at = tile % 4 / 2 * kMxLimbs * 64 + lane % 32 / 16 * 32 + tile % 2 * 16 + lane % 16;
#pragma unroll
                for (int j = 0; j < NL; j++)
                    r.x[j][i] = mx_op6(reinterpret_cast<const mx_u32x4 *>(u)[at + j * 64],
                                       reinterpret_cast<const mx_u32x2 *>(u + kPairLo)[at + j * 64]);
            }
        }
    };
    mx_acc16 acc[RT][NT] = {};
    auto use = [&](const Group &r, uint32_t g) {
        const uint32_t shift = g % 4 * 8;
#pragma unroll
        for (int j = 0; j < NL; j++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int m = 0; m < RT; m++)
                    acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        r.x[j][n], r.w[m], acc[m][n], NL == 1 ? kMxCbszFp4 : kMxCbszFp6, kMxCbszFp4, 0,
                        (int)(r.sx[n] >> shift & 255u) - (NL == 1 ? 0 : (int)kMxLimbShift[j]), 0, (int)(r.sw[m] >> shift));
    };
    if (g0 < g1) {  // (past the last group: that one again, not used)
        Group r0, r1;
        fetch(r0, g0);
        for (uint32_t g = g0; g < g1; g += 2) {
            fetch(r1, min(g + 1, g1 - 1));
            use(r0, g);
            fetch(r0, min(g + 2, g1 - 1));
            if (g + 1 < g1) use(r1, g + 1);
        }
    }
#pragma unroll
    for (int m = 0; m < RT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) part[wave][m][n][4 * (lane / 16) + i][lane % 16] = acc[m][n][i];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < RT * NT * 256; o += 64 * kThinWaves) {
        const uint32_t c = o % 16, m = o / 16 % RT, v = o / (16 * RT);  // rows of W side by side
        const uint32_t row = (m0 + m) * 16 + c, t = n0 * 16 + v;
        if (row >= rows || t >= T) continue;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < kThinWaves; k++) s += part[k][m][v / 16][v % 16][c];
        out[(size_t)t * rows + row] = s;
    }
}

// Vectors whose limbs are in the workspace at once: 128 MiB of it, half of the
// last cache.
size_t batch_of(size_t T, size_t cols) {
    const size_t fit = (128u << 20) / (cols * kMxLimbs * 3 / 4) / 64 * 64;
    return T < fit ? T : fit;
}

template <int NL, int WR, int WC, int MI, int NI, int NST>
hipError_t launch_gemm(const DevTensor &W, const MxSide &x, uint32_t T, float *out, hipStream_t s) {
    using L = MxTile<NL, WR, WC, MI, NI, NST>;
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    const MxSide w{W.p0, W.p1, (uint32_t)((d.tiles - 1) / 2)};
    const uint32_t gm = (uint32_t)((W.rows + 32 * L::kRows - 1) / (32 * L::kRows)), gn = (T + 32 * L::kVecs - 1) / (32 * L::kVecs);
    const uint32_t grid = (gm * gn + 7) / 8 * 8;
    hipLaunchKernelGGL((k_mx_gemm<NL, WR, WC, MI, NI, NST>), dim3(grid), dim3(64 * WR * WC), 0, s, w, x, d.kg, d.kq,
                       (uint32_t)W.rows, T, gm, gn, out);
    return hipGetLastError();
}

template <int NL, int RT, int NT>
hipError_t launch_thin(const DevTensor &W, const MxSide &x, uint32_t T, float *out, hipStream_t s) {
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    const MxSide w{W.p0, W.p1, (uint32_t)((d.tiles - 1) / 2)};
    const dim3 grid((unsigned)((W.rows + 16 * RT - 1) / (16 * RT)), (T + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((k_mx_thin<NL, RT, NT>), grid, dim3(64 * kThinWaves), 0, s, w, x, d.kg, d.kq, (uint32_t)W.rows, T, out);
    return hipGetLastError();
}

constexpr size_t kCus = 256;
size_t tiles_of(const DevTensor &W, size_t T, size_t m, size_t n) { return ((W.rows + m - 1) / m) * ((T + n - 1) / n); }

// Up to 2^20 sums the thin kernel: 4096 x 4096 with T = 7 | 64 | 256 vectors 8.5 |
// 13.4 | 35.6 us (tiles through LDS 32.8 | 33.9 | 36.8), 4-bit X 2.8 | 4.5 | 9.8
// (11.2 | 11.3 | 12.3); twice as many sums would be 64 (37) and 17 (13).  16 rows
// a workgroup for up to 16 vectors (T = 7: 8.5 us, 64 rows 10.2), unless there are
// so many rows that reading the vectors for each 16 costs more.
bool is_thin(const DevTensor &W, size_t T) { return (T + 15) / 16 * 16 * W.rows <= 1u << 20; }

// A stage of a 512 x 128 tile takes 1.13 us (one workgroup a CU), one of two 256
// x 64 tiles on a CU 0.63 us: the fewer rounds' time.  4096 x 8192 x 4096: 316
// and 348 us; 4095 x 7001 x 2816: 216 and 226; 1024 x 4096 x 4096: 105 and 62;
// 509 x 4864 x 2816: 73 and 32.
hipError_t limbs_product(const DevTensor &W, const MxSide &x, uint32_t T, float *out, hipStream_t s) {
    const size_t large = (tiles_of(W, T, 512, 128) + kCus - 1) / kCus, mid = (tiles_of(W, T, 256, 64) + 2 * kCus - 1) / (2 * kCus);
    if (is_thin(W, T))
        return T <= 16 && W.rows <= 8192 ? launch_thin<kMxLimbs, 1, 1>(W, x, T, out, s)
                                         : launch_thin<kMxLimbs, 4, 1>(W, x, T, out, s);
    if (large * 9 <= mid * 5) return launch_gemm<kMxLimbs, 4, 2, 4, 2, 3>(W, x, T, out, s);
    return launch_gemm<kMxLimbs, 4, 2, 2, 1, 3>(W, x, T, out, s);
}

}  // namespace

size_t matmul_mx_workspace(const DevTensor &W, size_t T) {
    if (matvecs_mx_fit(W, T)) return 0;
    const size_t cols = W.cols, n = batch_of(T, cols);
    return limb_bytes(mx_dims(n, cols / 32), n);
}

hipError_t launch_matmul_mx(const DevTensor &W, const float *X, size_t T, void *ws, float *out, hipStream_t s) {
    if (matvecs_mx_fit(W, T)) return launch_matvecs_mx(W, X, T, out, s);
    const size_t step = batch_of(T, W.cols);
    for (size_t t0 = 0; t0 < T; t0 += step) {
        const size_t n = T - t0 < step ? T - t0 : step;
        const MxDims d = mx_dims(limb_tiles(n) * 64, W.blocks_per_row);
        const MxLimbs p{(uint8_t *)ws, (uint8_t *)ws + limb_scales_at(d, n)};
        hipLaunchKernelGGL(k_mx_limbs, dim3((unsigned)(limb_tiles(n) * 2 * d.kg * 128 / kLimbThreads)), dim3(kLimbThreads), 0, s,
                           X + t0 * W.cols, (uint32_t)n, d, p);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const MxSide x{p.data, p.scales, (uint32_t)((d.tiles - 1) / 2)};
        e = limbs_product(W, x, (uint32_t)n, out + t0 * W.rows, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_matmul_mx_mx(const DevTensor &W, const DevTensor &X, size_t T, float *out, hipStream_t s) {
    const MxDims d = mx_dims(X.rows, X.blocks_per_row);
    const MxSide x{X.p0, X.p1, (uint32_t)((d.tiles - 1) / 2)};
    // 256 x 128 tiles once they fill the CUs: 4095 x 7001 x 2816 61 us (128 x 64: 72),
    // 1024 x 4096 x 4096 (128 of them) 22.8 us (17.2)
    if (is_thin(W, T))
        return T <= 16 && W.rows <= 8192 ? launch_thin<1, 1, 1>(W, x, (uint32_t)T, out, s)
                                         : launch_thin<1, 2, 2>(W, x, (uint32_t)T, out, s);
    if (tiles_of(W, T, 256, 128) >= kCus) return launch_gemm<1, 4, 2, 2, 2, 3>(W, x, (uint32_t)T, out, s);
    return launch_gemm<1, 2, 2, 2, 1, 4>(W, x, (uint32_t)T, out, s);
}

}  // namespace lt
