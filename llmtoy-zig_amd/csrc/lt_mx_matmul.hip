// lt_mx_matmul.hip -- products of an MXFP4 matrix with many vectors:
// out[t][r] = sum_c W[r][c] X[t][c].
//
// X in fp32: a first launch turns its blocks into limbs (lt_mx.h) laid out as
// matrix operands, [tile of 16 vectors][group of 4 blocks][limb][64 lanes],
// and the product runs one matrix instruction a limb into the same sums.  X as
// an MXFP4 tensor: its codes and scales are an operand already.
#include "llmtoy_hip.h"
#include "lt_internal.h"
#include "lt_mx.h"

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
size_t limb_bytes(const MxDims &d, size_t T) { return limb_data_bytes(d, T) + limb_tiles(T) * 4 * d.kq * 256; }

// A thread a block; vectors from T on and blocks from nb on are zeros.
__global__ __launch_bounds__(256) void k_mx_limbs(const float *__restrict__ X, uint32_t T, MxDims d, MxLimbs p) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
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

// The scale bytes of a lane's blocks in 16 groups' words: word h for the
// blocks 2 h + lane / 32 of a group, byte g for group g.
struct MxScales {
    uint32_t w[2];
};
__device__ __forceinline__ MxScales scales_at(const MxSide &p, uint32_t kq, uint32_t tile32, uint32_t q, uint32_t off) {
    const uint8_t *w = p.scales + ((size_t)2 * min(tile32, p.last) * kq + q) * 256;  // (uniform)
    return {{*reinterpret_cast<const uint32_t *>(w + off), *reinterpret_cast<const uint32_t *>(w + off + 128)}};
}

// out[t][r]: a workgroup of WR x WC waves computes 32 WR MI rows of W by 32 WC NI
// vectors, a wave MI x NI tiles of 32 x 32, KS pairs of blocks (64 columns) a
// stage.
//
// The vectors are the instruction's rows and W's rows its columns: a store of
// the sums is then 32 neighbouring rows of out for each of two vectors.
template <int NL, int WR, int WC, int MI, int NI, int KS>
struct MxTile {
    static constexpr int kRows = WR * MI, kVecs = WC * NI;  // tiles of 32
    static constexpr int kWBytes = kRows * KS * 1024;
    static constexpr int kXBytes = NL == 1 ? kVecs * KS * 1024 : kVecs / 2 * KS * (int)kPairBytes;
    static constexpr int kChunks = (kWBytes + kXBytes) / 1024, kWaves = WR * WC;
    static constexpr int kBytes = kWBytes + kXBytes;
};

template <int NL, int WR, int WC, int MI, int NI, int KS>
__global__ __launch_bounds__(64 * WR * WC, 2) void k_mx_gemm(MxSide w, MxSide x, uint32_t kg, uint32_t kq, uint32_t rows,
                                                             uint32_t T, uint32_t grid_m, uint32_t grid_n, float *out) {
    using L = MxTile<NL, WR, WC, MI, NI, KS>;
    __shared__ __attribute__((aligned(16))) uint8_t buf0[L::kBytes];
    __shared__ __attribute__((aligned(16))) uint8_t buf1[L::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wc = wave / WR;
    // blocks of one XCD (equal index % 8) take neighbouring tiles
    const uint32_t per = (grid_m * grid_n + 7) / 8;
    const uint32_t id = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (id >= grid_m * grid_n) return;
    const uint32_t m0 = id % grid_m * L::kRows, n0 = id / grid_m * L::kVecs;  // in tiles of 32
    const uint32_t steps = 2 * kg / KS;
    // a lane's place in a tile of 32's codes of a pair, and in its scale words
    const uint32_t code_off = (uint32_t)(lane & 31) / 16 * kg * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
    const uint32_t scale_off = (uint32_t)(lane & 31) / 16 * kq * 256 + (lane >> 5) * 64 + (lane & 15) * 4;

    auto fetch = [&](uint32_t step, uint8_t *dst) {
#pragma unroll
        for (int c0 = 0; c0 < L::kChunks; c0 += L::kWaves) {
            const int c = c0 + wave;
            if (L::kChunks % L::kWaves && c >= L::kChunks) break;
            const uint8_t *src;
            if (c < L::kRows * KS || NL == 1) {  // codes: chunk = tile of 32 and pair of blocks
                const bool isw = c < L::kRows * KS;
                const MxSide &p = isw ? w : x;
                const int i = isw ? c : c - L::kRows * KS;
                const uint32_t t32 = min((isw ? m0 : n0) + i / KS, p.last), pair = step * KS + i % KS;
                src = p.data + ((size_t)2 * t32 * kg + pair / 2) * 1024 + (pair % 2) * 512 + code_off;
            } else {  // limbs: 15 chunks a tile of 64 and pair
                const int i = c - L::kRows * KS;
                const uint32_t t64 = min(n0 / 2 + i / (15 * KS), (uint32_t)limb_tiles(T) - 1), pair = step * KS + i / 15 % KS;
                src = x.data + ((size_t)t64 * 2 * kg + pair) * kPairBytes + (i % 15) * 1024 + lane * 16;
            }
            to_lds(src, dst + c * 1024);
        }
    };

    mx_acc32 acc[MI][NI] = {};
    MxScales sw[MI], sx[NI];
    auto scales = [&](uint32_t q) {
#pragma unroll
        for (int i = 0; i < MI; i++) sw[i] = scales_at(w, kq, m0 + wr * MI + i, q, scale_off);
#pragma unroll
        for (int i = 0; i < NI; i++) sx[i] = scales_at(x, kq, n0 + wc * NI + i, q, scale_off);
    };
    auto compute = [&](uint32_t step, const uint8_t *src) {
#pragma unroll
        for (int h = 0; h < KS; h++) {
            const uint32_t pair = step * KS + h, shift = pair / 2 % 4 * 8;
            const bool odd = KS == 2 ? h : pair % 2;
            mx_op b[MI];
            int sb[MI], sa[NI];
#pragma unroll
            for (int i = 0; i < MI; i++) {
                b[i] = mx_op4(*reinterpret_cast<const mx_u32x4 *>(src + ((wr * MI + i) * KS + h) * 1024 + lane * 16));
                sb[i] = (int)((odd ? sw[i].w[1] : sw[i].w[0]) >> shift);
            }
#pragma unroll
            for (int i = 0; i < NI; i++) sa[i] = (int)((odd ? sx[i].w[1] : sx[i].w[0]) >> shift & 255u);
#pragma unroll
            for (int j = 0; j < NL; j++) {
                mx_op a[NI];
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int v = wc * NI + i;
                    if (NL == 1) {
                        a[i] = mx_op4(*reinterpret_cast<const mx_u32x4 *>(src + L::kWBytes + (v * KS + h) * 1024 + lane * 16));
                    } else {
                        const uint8_t *u = src + L::kWBytes + (v / 2 * KS + h) * (int)kPairBytes;
                        const int at = (v % 2 * kMxLimbs + j) * 64 + lane;
                        a[i] = mx_op6(reinterpret_cast<const mx_u32x4 *>(u)[at],
                                      reinterpret_cast<const mx_u32x2 *>(u + kPairLo)[at]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NI; n++)
#pragma unroll
                    for (int m = 0; m < MI; m++)
                        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                            a[n], b[m], acc[m][n], NL == 1 ? kMxCbszFp4 : kMxCbszFp6, kMxCbszFp4, 0,
                            sa[n] - (NL == 1 ? 0 : (int)kMxLimbShift[j]), 0, sb[m]);
            }
        }
    };

    fetch(0, buf0);
    for (uint32_t s = 0; s < steps; s += 2) {  // (an even number of steps)
        if (s * KS % 8 == 0) scales(s * KS / 8);
        __syncthreads();
        fetch(s + 1, buf1);
        compute(s, buf0);
        __syncthreads();
        if (s + 2 < steps) fetch(s + 2, buf0);
        compute(s + 1, buf1);
    }

#pragma unroll
    for (int n = 0; n < NI; n++)
#pragma unroll
        for (int m = 0; m < MI; m++) {
            const uint32_t r = (m0 + wr * MI + m) * 32 + (lane & 31);
            if (r >= rows) continue;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t t = (n0 + wc * NI + n) * 32 + i / 4 * 8 + 4 * (lane >> 5) + i % 4;
                if (t < T) out[(size_t)t * rows + r] = acc[m][n][i];
            }
        }
}

// Vectors whose limbs are in the workspace at once: 128 MiB of it, half of the
// last cache.
size_t batch_of(size_t T, size_t cols) {
    const size_t fit = (128u << 20) / (cols * kMxLimbs * 3 / 4) / 64 * 64;
    return T < fit ? T : fit;
}

template <int NL, int WR, int WC, int MI, int NI, int KS>
hipError_t launch_gemm(const DevTensor &W, const MxSide &x, uint32_t T, float *out, hipStream_t s) {
    using L = MxTile<NL, WR, WC, MI, NI, KS>;
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    const MxSide w{W.p0, W.p1, (uint32_t)((d.tiles - 1) / 2)};
    const uint32_t gm = (uint32_t)((W.rows + 32 * L::kRows - 1) / (32 * L::kRows)), gn = (T + 32 * L::kVecs - 1) / (32 * L::kVecs);
    const uint32_t grid = (gm * gn + 7) / 8 * 8;
    hipLaunchKernelGGL((k_mx_gemm<NL, WR, WC, MI, NI, KS>), dim3(grid), dim3(64 * WR * WC), 0, s, w, x, d.kg, d.kq,
                       (uint32_t)W.rows, T, gm, gn, out);
    return hipGetLastError();
}

}  // namespace

size_t matmul_mx_workspace(size_t T, size_t cols) {
    const size_t n = batch_of(T, cols);
    return limb_bytes(mx_dims(n, cols / 32), n);
}

hipError_t launch_matmul_mx(const DevTensor &W, const float *X, size_t T, void *ws, float *out, hipStream_t s) {
    const size_t step = batch_of(T, W.cols);
    for (size_t t0 = 0; t0 < T; t0 += step) {
        const size_t n = T - t0 < step ? T - t0 : step;
        const MxDims d = mx_dims(limb_tiles(n) * 64, W.blocks_per_row);
        const MxLimbs p{(uint8_t *)ws, (uint8_t *)ws + limb_data_bytes(d, n)};
        hipLaunchKernelGGL(k_mx_limbs, dim3((unsigned)((limb_tiles(n) * 2 * d.kg * 128 + 255) / 256)), dim3(256), 0, s,
                           X + t0 * W.cols, (uint32_t)n, d, p);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const MxSide x{p.data, p.scales, (uint32_t)((d.tiles - 1) / 2)};
        e = launch_gemm<kMxLimbs, 4, 1, 4, 2, 1>(W, x, (uint32_t)n, out + t0 * W.rows, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_matmul_mx_mx(const DevTensor &W, const DevTensor &X, size_t T, float *out, hipStream_t s) {
    const MxDims d = mx_dims(X.rows, X.blocks_per_row);
    const MxSide x{X.p0, X.p1, (uint32_t)((d.tiles - 1) / 2)};
    return launch_gemm<1, 2, 2, 4, 2, 1>(W, x, (uint32_t)T, out, s);
}

}  // namespace lt
