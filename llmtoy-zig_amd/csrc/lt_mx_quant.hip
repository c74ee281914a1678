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
#include "lt_topk.h"

namespace lt {

namespace {

// One thread a block: raw bytes (any alignment, staged through LDS as dwords)
// against the tensor's planes.  PCIe carries the bytes; this is not the bound.
constexpr int kMxStage = 256;
template <bool IN>
__global__ __launch_bounds__(kMxStage) void k_mx_blocks(uint8_t *raw, size_t nblk, size_t blk0, size_t rows, MxDims d,
                                                        uint8_t *codes, uint8_t *scales, uint32_t *beyond) {
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
            if (mine[0] == 253 || mine[0] == 254) *beyond = 1;
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

// A workgroup a tile of 16 rows and a group of 16 blocks (512 columns): 32 KiB of
// fp32 against 4 KiB of codes, which stand in a row, and a KiB's quarter of
// scale words.  16 threads a row, 8 lanes a block with a float4 each; codes and
// scales pass through LDS between a row's order and the tile's.  Bound by HBM:
// 9728 x 4096 (181 MB) quantised in 30.8 us, 5.9 TB/s, with loads past the caches
// (41.5 without; a block of 8 lanes on its own, with divisions, 43); read back in
// 27.8.  What fits the L2s may be there still: 1024 x 4096 7.6 us past the caches,
// 6.5 through them.
constexpr size_t kMxNtBytes = 32 << 20;
struct MxSpan {
    size_t row0, rows;  // of the tensor, over all experts
    size_t expert_rows;
    uint32_t tile0;     // the first row's tile
    MxDims d;
};
struct MxTileAt {
    size_t tile;        // in the planes
    size_t first;       // its row 0's place in the span's array, as row0 stands at 0 (may be before it)
    __device__ __forceinline__ bool has(const MxSpan &p, uint32_t r, uint32_t in_expert) const {
        const size_t at = first + r;  // (wraps below 0)
        return in_expert + r < p.expert_rows && at < p.rows;
    }
};

template <bool NT>
__global__ __launch_bounds__(256) void k_mx_quantize(const float *__restrict__ x, MxSpan p, uint8_t *codes, uint8_t *scales) {
    __shared__ uint32_t lc[16][16][5];  // [block][row][word], a word of padding
    __shared__ uint8_t ls[16][4][4];    // [row][lane group][group of 4 blocks]
    const uint32_t r = threadIdx.x / 16, l = threadIdx.x % 16, q = blockIdx.x;
    const size_t tile = p.tile0 + blockIdx.y, expert = tile / p.d.tiles;
    const uint32_t in = (uint32_t)(tile % p.d.tiles) * 16;
    const MxTileAt t{tile, expert * p.expert_rows + in - p.row0};
    if (t.has(p, r, in)) {
        const float *row = x + (t.first + r) * p.d.nb * 32;
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (16 * q + 2 * i + l / 8 < p.d.nb) v[i] = NT ? ldg16f_nt(row + 512 * q + 64 * i + 4 * l) : ldg16f(row + 512 * q + 64 * i + 4 * l);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t b = 2 * i + l / 8, j = l % 8;
            uint32_t word = 0, e = 0;
            if (16 * q + b < p.d.nb) {  // (8 lanes together)
                float most = __builtin_elementwise_maximum(
                    __builtin_elementwise_maximum(__builtin_fabsf(v[i].x), __builtin_fabsf(v[i].y)),
                    __builtin_elementwise_maximum(__builtin_fabsf(v[i].z), __builtin_fabsf(v[i].w)));  // (NaN where one is)
                most = __builtin_elementwise_maximum(most, dpp<0xB1>(most));   // lane ^ 1
                most = __builtin_elementwise_maximum(most, dpp<0x4E>(most));   // lane ^ 2
                most = __builtin_elementwise_maximum(most, dpp<0x141>(most));  // the other four
                const uint32_t top = __float_as_uint(most) & 0x7fffffffu;
                e = (uint32_t)max((int)(top >> 23) - 2, 0);
                if (top >= 0x7f800000u) {
                    e = 255;
                } else {
                    const float scale = __uint_as_float(e << 23);  // (its exponent is what counts: 0 is 2^-127)
                    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[i].x, v[i].y, scale, 0);
                    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[i].z, v[i].w, scale, 1);
                    word = (word & 0xfu) | (word & 0xf0u) << 4 | (word & 0xf00u) << 8 | (word & 0xf000u) << 12;  // a nibble a byte
                }
            }
            const uint32_t hi = dpp_u<0x104>(word);  // from lane + 4; lanes 4-7: elements 16 on, the high halves
            if (j < 4) lc[b][r][j] = word | hi << 4;
            if (j == 0) ls[r][b % 4][b / 4] = (uint8_t)e;
        }
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, row = lane % 16, g = 4 * q + wave;
    if (!t.has(p, row, in)) return;
    if (g < p.d.kg) {
        const uint32_t *w = lc[4 * wave + lane / 16][row];
        reinterpret_cast<uint4 *>(codes)[(tile * p.d.kg + g) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (wave == 0)
        reinterpret_cast<uint32_t *>(scales)[(tile * p.d.kq + q) * 64 + lane] =
            *reinterpret_cast<const uint32_t *>(ls[row][lane / 16]);
}

__global__ __launch_bounds__(256) void k_mx_dequantize(float *__restrict__ out, MxSpan p, const uint8_t *codes,
                                                       const uint8_t *scales) {
    __shared__ uint32_t lc[16][16][5];
    __shared__ uint32_t ls[16][4];
    const uint32_t r = threadIdx.x / 16, l = threadIdx.x % 16, q = blockIdx.x;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, g = 4 * q + wave;
    const size_t tile = p.tile0 + blockIdx.y, expert = tile / p.d.tiles;
    const uint32_t in = (uint32_t)(tile % p.d.tiles) * 16;
    const MxTileAt t{tile, expert * p.expert_rows + in - p.row0};
    if (g < p.d.kg) {
        const uint4 w = reinterpret_cast<const uint4 *>(codes)[(tile * p.d.kg + g) * 64 + lane];
        uint32_t *to = lc[4 * wave + lane / 16][lane % 16];
        to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
    }
    if (wave == 0) ls[lane % 16][lane / 16] = reinterpret_cast<const uint32_t *>(scales)[(tile * p.d.kq + q) * 64 + lane];
    __syncthreads();
    if (!t.has(p, r, in)) return;
    float *row = out + (t.first + r) * p.d.nb * 32;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t b = 2 * i + l / 8, j = l % 8;
        if (16 * q + b >= p.d.nb) continue;
        const uint32_t w = lc[b][r][j % 4], n = (j < 4 ? w : w >> 4) & 0x0f0f0f0fu;
        const uint32_t four = (n & 0xfu) | (n >> 4 & 0xf0u) | (n >> 8 & 0xf00u) | (n >> 12 & 0xf000u);
        const uint32_t e = ls[r][b % 4] >> (b / 4 * 8) & 255u;
        const float scale = __uint_as_float(e << 23);  // (255: every value NaN)
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, scale, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, scale, 1);
        *reinterpret_cast<float4 *>(row + 512 * q + 64 * i + 4 * l) = make_float4(lo[0], lo[1], hi[0], hi[1]);
    }
}

// One launch for each 65535 tiles (a grid's limit) of the rows.
template <typename Launch>
hipError_t over_tiles(const DevTensor &t, size_t row0, size_t rows, Launch launch) {
    MxSpan p{row0, rows, t.rows, 0, mx_dims(t.rows, t.blocks_per_row)};
    auto tile_of = [&](size_t row) { return row / t.rows * p.d.tiles + row % t.rows / 16; };
    const size_t last = tile_of(row0 + rows - 1);
    for (size_t first = tile_of(row0); first <= last; first += 65535) {
        p.tile0 = (uint32_t)first;
        launch(p, dim3(p.d.kq, (unsigned)(last - first + 1 < 65535 ? last - first + 1 : 65535)));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_mx_blocks(const DevTensor &t, uint8_t *raw, size_t nblk, size_t blk0, bool in, hipStream_t s) {
    const MxDims d = mx_dims(t.rows, t.blocks_per_row);
    const dim3 grid((unsigned)((nblk + kMxStage - 1) / kMxStage));
    uint8_t *codes = const_cast<uint8_t *>(t.p0), *scales = const_cast<uint8_t *>(t.p1);
    if (in)
        hipLaunchKernelGGL(k_mx_blocks<true>, grid, dim3(kMxStage), 0, s, raw, nblk, blk0, t.rows, d, codes, scales,
                           mx_beyond_flag(t));
    else
        hipLaunchKernelGGL(k_mx_blocks<false>, grid, dim3(kMxStage), 0, s, raw, nblk, blk0, t.rows, d, codes, scales, nullptr);
    return hipGetLastError();
}

hipError_t launch_mx_quantize(const DevTensor &t, const float *x, size_t row0, size_t rows, hipStream_t s) {
    const auto kernel = rows * t.cols * 4 > kMxNtBytes ? k_mx_quantize<true> : k_mx_quantize<false>;
    return over_tiles(t, row0, rows, [&](const MxSpan &p, dim3 grid) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, x, p, const_cast<uint8_t *>(t.p0), const_cast<uint8_t *>(t.p1));
    });
}

hipError_t launch_mx_dequantize(const DevTensor &t, float *out, size_t row0, size_t rows, hipStream_t s) {
    return over_tiles(t, row0, rows, [&](const MxSpan &p, dim3 grid) {
        hipLaunchKernelGGL(k_mx_dequantize, grid, dim3(256), 0, s, out, p, t.p0, t.p1);
    });
}

}  // namespace lt
