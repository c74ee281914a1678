// lt_mx_quant.hip -- MXFP4 blocks: GGUF bytes to and from the device layout
// (lt_mx.h), fp32 rows into blocks and back.
//
// Quantisation of a block, a = max |x|:
//   e    = clamp(floor(log2 a) - 2, -127, 127), the scale byte e + 127; a = 0: byte 0;
//          a NaN or an infinity in the block: byte 255 and codes 0 (all NaN)
//   code = sign and the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 to |x| / 2^e, a
//          tie to the even code, 6 for what lies beyond
// so the largest element lands in [4, 8).  Scaling by a power of two is exact
// and the conversion instruction rounds once.
#include "llmtoy_hip.h"
#include "lt_internal.h"
#include "lt_mx.h"

namespace lt {

namespace {

// One thread a block: raw bytes (any alignment, staged through LDS as dwords)
// against the tensor's planes.  PCIe carries the bytes; this is not the bound.
constexpr int kMxStage = 256;
template <bool IN>
__global__ __launch_bounds__(kMxStage) void k_mx_blocks(uint8_t *raw, size_t nblk, size_t blk0, size_t rows, MxDims d,
                                                        uint8_t *codes, uint8_t *scales) {
    __shared__ uint32_t lds[kMxStage * kMxBlockBytes / 4];
    const size_t b0 = (size_t)blockIdx.x * kMxStage;
    const uint32_t n = nblk - b0 < (size_t)kMxStage ? (uint32_t)(nblk - b0) : (uint32_t)kMxStage;
    const uint32_t nw = (n * kMxBlockBytes + 3) / 4;
    uint32_t *words = reinterpret_cast<uint32_t *>(raw + b0 * kMxBlockBytes);
    uint8_t *mine = reinterpret_cast<uint8_t *>(lds) + threadIdx.x * kMxBlockBytes;
    if (IN) {
        for (uint32_t w = threadIdx.x; w < nw; w += kMxStage) lds[w] = words[w];
        __syncthreads();
    }
    if (threadIdx.x < n) {
        const size_t at = blk0 + b0 + threadIdx.x, row = at / d.nb;
        const uint32_t b = (uint32_t)(at % d.nb);
        const size_t expert = row / rows, r = row % rows, tile = expert * d.tiles + r / 16;
        uint32_t *code = reinterpret_cast<uint32_t *>(codes + mx_code_at(d, tile, (uint32_t)(r % 16), b));
        uint8_t *scale = scales + mx_scale_at(d, tile, (uint32_t)(r % 16), b);
        if (IN) {
            *scale = mine[0];
#pragma unroll
            for (int i = 0; i < 4; i++)
                code[i] = (uint32_t)mine[4 * i + 1] | (uint32_t)mine[4 * i + 2] << 8 | (uint32_t)mine[4 * i + 3] << 16 |
                          (uint32_t)mine[4 * i + 4] << 24;
        } else {
            mine[0] = *scale;
#pragma unroll
            for (int i = 0; i < 16; i++) mine[1 + i] = (uint8_t)(code[i / 4] >> (8 * (i % 4)));
        }
    }
    if (!IN) {
        __syncthreads();
        for (uint32_t w = threadIdx.x; w < nw; w += kMxStage) words[w] = lds[w];
    }
}

// 8 lanes a block, a float4 each; lanes 0-3 hold the low halves of the code
// bytes, lanes 4-7 the high ones.
__global__ __launch_bounds__(256) void k_mx_quantize(const float *__restrict__ x, size_t row0, uint32_t rows,
                                                     size_t expert_rows, MxDims d, uint8_t *codes, uint8_t *scales) {
    const size_t unit = ((size_t)blockIdx.x * 256 + threadIdx.x) / 8;
    const uint32_t j = threadIdx.x % 8;
    if (unit >= (size_t)rows * d.nb) return;  // (whole groups of 8 lanes)
    const uint32_t row = (uint32_t)(unit / d.nb), b = (uint32_t)(unit % d.nb);
    const float4 v = ldg16f(x + unit * 32 + 4 * j);
    uint32_t top = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                       max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
    for (int off = 4; off; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 8));
    const bool bad = top >= 0x7f800000u;
    const int e = max((int)(top >> 23) - 2, 0);  // the scale byte
    uint32_t q = 0;
    if (!bad) {
        const int up = 127 - e;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, ldexpf(v.x, up), ldexpf(v.y, up), 1.0f, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, ldexpf(v.z, up), ldexpf(v.w, up), 1.0f, 1);
        q = (q & 0xfu) | (q & 0xf0u) << 4 | (q & 0xf00u) << 8 | (q & 0xf000u) << 12;  // a nibble a byte
    }
    const uint32_t hi = (uint32_t)__shfl_down((int)q, 4, 8);
    const size_t all = row0 + row, r = all % expert_rows, tile = all / expert_rows * d.tiles + r / 16;
    if (j < 4) reinterpret_cast<uint32_t *>(codes + mx_code_at(d, tile, (uint32_t)(r % 16), b))[j] = q | hi << 4;
    if (j == 0) scales[mx_scale_at(d, tile, (uint32_t)(r % 16), b)] = bad ? (uint8_t)255 : (uint8_t)e;
}

__global__ __launch_bounds__(256) void k_mx_dequantize(float *__restrict__ out, size_t row0, uint32_t rows,
                                                       size_t expert_rows, MxDims d, const uint8_t *codes,
                                                       const uint8_t *scales) {
    const size_t unit = ((size_t)blockIdx.x * 256 + threadIdx.x) / 8;
    const uint32_t j = threadIdx.x % 8;
    if (unit >= (size_t)rows * d.nb) return;
    const uint32_t row = (uint32_t)(unit / d.nb), b = (uint32_t)(unit % d.nb);
    const size_t all = row0 + row, r = all % expert_rows, tile = all / expert_rows * d.tiles + r / 16;
    const uint32_t w = reinterpret_cast<const uint32_t *>(codes + mx_code_at(d, tile, (uint32_t)(r % 16), b))[j % 4];
    const uint32_t e = scales[mx_scale_at(d, tile, (uint32_t)(r % 16), b)];
    const uint32_t n = (j < 4 ? w : w >> 4) & 0x0f0f0f0fu;
    const uint32_t q = (n & 0xfu) | (n >> 4 & 0xf0u) | (n >> 8 & 0xf00u) | (n >> 12 & 0xf000u);
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    const int up = (int)e - 127;
    float4 v = make_float4(ldexpf(lo[0], up), ldexpf(lo[1], up), ldexpf(hi[0], up), ldexpf(hi[1], up));
    if (e == 255u) v = make_float4(NAN, NAN, NAN, NAN);
    *reinterpret_cast<float4 *>(out + unit * 32 + 4 * j) = v;
}

unsigned grid_of(size_t units) { return (unsigned)((units * 8 + 255) / 256); }

}  // namespace

hipError_t launch_mx_blocks(const DevTensor &t, uint8_t *raw, size_t nblk, size_t blk0, bool in, hipStream_t s) {
    const MxDims d = mx_dims(t.rows, t.blocks_per_row);
    const dim3 grid((unsigned)((nblk + kMxStage - 1) / kMxStage));
    uint8_t *codes = const_cast<uint8_t *>(t.p0), *scales = const_cast<uint8_t *>(t.p1);
    if (in)
        hipLaunchKernelGGL(k_mx_blocks<true>, grid, dim3(kMxStage), 0, s, raw, nblk, blk0, t.rows, d, codes, scales);
    else
        hipLaunchKernelGGL(k_mx_blocks<false>, grid, dim3(kMxStage), 0, s, raw, nblk, blk0, t.rows, d, codes, scales);
    return hipGetLastError();
}

hipError_t launch_mx_quantize(const DevTensor &t, const float *x, size_t row0, size_t rows, hipStream_t s) {
    const MxDims d = mx_dims(t.rows, t.blocks_per_row);
    hipLaunchKernelGGL(k_mx_quantize, dim3(grid_of(rows * d.nb)), dim3(256), 0, s, x, row0, (uint32_t)rows,
                       t.rows, d, const_cast<uint8_t *>(t.p0), const_cast<uint8_t *>(t.p1));
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const DevTensor &t, float *out, size_t row0, size_t rows, hipStream_t s) {
    const MxDims d = mx_dims(t.rows, t.blocks_per_row);
    hipLaunchKernelGGL(k_mx_dequantize, dim3(grid_of(rows * d.nb)), dim3(256), 0, s, out, row0, (uint32_t)rows,
                       t.rows, d, t.p0, t.p1);
    return hipGetLastError();
}

}  // namespace lt
