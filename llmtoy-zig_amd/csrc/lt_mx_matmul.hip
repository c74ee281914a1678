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

// The workspace of T vectors: operand words in two planes, and scale words as
// a tensor's.
struct MxLimbPlanes {
    mx_u32x4 *hi;  // [tile][kg][5][64]
    mx_u32x2 *lo;  // [tile][kg][5][64]
    uint8_t *sc;   // [tile][kq][64][4]
};
size_t limb_bytes(const MxDims &d) { return d.tiles * ((size_t)d.kg * kMxLimbs * 64 * 24 + (size_t)d.kq * 256); }
MxLimbPlanes limb_planes(void *ws, const MxDims &d) {
    uint8_t *p = (uint8_t *)ws;
    const size_t n = d.tiles * d.kg * kMxLimbs * 64;
    return {(mx_u32x4 *)p, (mx_u32x2 *)(p + n * 16), p + n * 24};
}

// A thread a block; vectors from T on and blocks from nb on are zeros.
__global__ __launch_bounds__(256) void k_mx_limbs(const float *__restrict__ X, uint32_t T, MxDims d, MxLimbPlanes p) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t grp = id / 64;
    if (grp >= d.tiles * d.kg) return;
    const uint32_t lane = (uint32_t)(id % 64), g = (uint32_t)(grp % d.kg), b = 4 * g + lane / 16;
    const size_t tile = grp / d.kg, t = tile * 16 + lane % 16;
    mx_f32x16 lo = {}, hi = {};
    if (t < T && b < d.nb) mx_load_block(X + (t * d.nb + b) * 32, lo, hi);
    const uint32_t s = mx_limb_scale(mx_top(lo, hi));
    p.sc[((tile * d.kq + g / 4) * 64 + lane) * 4 + g % 4] = (uint8_t)s;
    const size_t at = grp * kMxLimbs * 64 + lane;
    mx_limbs(lo, hi, s, [&](int j, const mx_u32x6 &q) {
        p.hi[at + j * 64] = mx_u32x4{q[0], q[1], q[2], q[3]};
        p.lo[at + j * 64] = mx_u32x2{q[4], q[5]};
    });
}

// A wave computes 16 rows by 16 vectors.
template <bool LIMBS>
__global__ __launch_bounds__(256) void k_mx_gemm(const uint8_t *wc, const uint8_t *ws, MxDims d, uint32_t rows,
                                                 MxLimbPlanes p, const uint8_t *xc, const uint8_t *xs, uint32_t T, float *out) {
    const int lane = threadIdx.x & 63;
    const size_t rt = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rt >= d.tiles) return;
    const size_t tt = blockIdx.y;
    mx_acc16 acc = {};
    for (uint32_t g = 0; g < d.kg; g++) {
        const mx_op a = mx_op4(*reinterpret_cast<const mx_u32x4 *>(wc + ((rt * d.kg + g) * 64 + lane) * 16));
        const int sa = ws[((rt * d.kq + g / 4) * 64 + lane) * 4 + g % 4];
        if (LIMBS) {
            const int sb = p.sc[((tt * d.kq + g / 4) * 64 + lane) * 4 + g % 4];
#pragma unroll
            for (int j = 0; j < kMxLimbs; j++) {
                const size_t at = ((tt * d.kg + g) * kMxLimbs + j) * 64 + lane;
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, mx_op6(p.hi[at], p.lo[at]), acc, kMxCbszFp4,
                                                                       kMxCbszFp6, 0, sa, 0, sb - (int)kMxLimbShift[j]);
            }
        } else {
            const mx_op b = mx_op4(*reinterpret_cast<const mx_u32x4 *>(xc + ((tt * d.kg + g) * 64 + lane) * 16));
            const int sb = xs[((tt * d.kq + g / 4) * 64 + lane) * 4 + g % 4];
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kMxCbszFp4, kMxCbszFp4, 0, sa, 0, sb);
        }
    }
    const size_t t = tt * 16 + (lane & 15);
    if (t < T)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const size_t r = rt * 16 + 4 * (lane >> 4) + i;
            if (r < rows) out[t * rows + r] = acc[i];
        }
}

// Vectors whose limbs are in the workspace at once: 128 MiB of it, half of the
// last cache, at least 16.
size_t batch_of(size_t T, size_t cols) {
    const size_t fit = (128u << 20) / (cols * kMxLimbs * 3 / 4) / 16 * 16;
    return T < fit ? T : fit;
}

}  // namespace

size_t matmul_mx_workspace(size_t T, size_t cols) { return limb_bytes(mx_dims(batch_of(T, cols), cols / 32)); }

hipError_t launch_matmul_mx(const DevTensor &W, const float *X, size_t T, void *ws, float *out, hipStream_t s) {
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    const size_t step = batch_of(T, W.cols);
    for (size_t t0 = 0; t0 < T; t0 += step) {
        const size_t n = T - t0 < step ? T - t0 : step;
        const MxDims dx = mx_dims(n, W.blocks_per_row);
        const MxLimbPlanes p = limb_planes(ws, dx);
        hipLaunchKernelGGL(k_mx_limbs, dim3((unsigned)((dx.tiles * dx.kg * 64 + 255) / 256)), dim3(256), 0, s,
                           X + t0 * W.cols, (uint32_t)n, dx, p);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(k_mx_gemm<true>, dim3((unsigned)((d.tiles + 3) / 4), (unsigned)dx.tiles), dim3(256), 0, s, W.p0,
                           W.p1, d, (uint32_t)W.rows, p, nullptr, nullptr, (uint32_t)n, out + t0 * W.rows);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_matmul_mx_mx(const DevTensor &W, const DevTensor &X, size_t T, float *out, hipStream_t s) {
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    hipLaunchKernelGGL(k_mx_gemm<false>, dim3((unsigned)((d.tiles + 3) / 4), (unsigned)((T + 15) / 16)), dim3(256), 0, s,
                       W.p0, W.p1, d, (uint32_t)W.rows, MxLimbPlanes{}, X.p0, X.p1, (uint32_t)T, out);
    return hipGetLastError();
}

}  // namespace lt
