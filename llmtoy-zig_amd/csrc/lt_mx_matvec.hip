// lt_mx_matvec.hip -- products of MXFP4 matrices with one vector: matvec, the
// experts' gate/up and down by id.
//
//   y[r] = sum_b 2^(e_rb - 127) sum_i w_rbi x_bi,   x_bi = sum_j q_jbi s_b 2^(-shift_j)   (lt_mx.h)
//
// One v_mfma_scale_f32_16x16x128 takes 16 rows of 4 weight blocks, codes and
// scales as they stand in memory, against a 128 x 16 operand whose columns 0..4
// are the five limbs of those 128 activations (the other columns are zero): the
// row's sum over the columns is the product with the fp32 activations.  No
// weight is ever converted; a KiB of weights costs one matrix instruction (about
// 18 cycles) and two LDS reads.
//
// A workgroup converts the vector once, while its first weights are on their
// way, and its waves split a tile's row over groups of 16 blocks (one scale
// word); what they summed meets in LDS in the waves' order.
#include "llmtoy_hip.h"
#include "lt_internal.h"
#include "lt_mx.h"

namespace lt {

namespace {

constexpr int kMvWaves = 8;
constexpr int kMvThreads = 64 * kMvWaves;

// LDS of a vector's limbs: per block and limb 16 + 8 bytes of operand words,
// per group of 16 blocks and lane group a word of four scale bytes.
struct MxVec {
    mx_u32x4 *hi;  // [4 kg][5]
    mx_u32x2 *lo;  // [4 kg][5]
    uint8_t *sc;   // [kq][4 lane groups][4]
};
__host__ __device__ inline size_t mx_vec_bytes(uint32_t kg) {
    const size_t nb = 4 * (size_t)kg, kq = (kg + 3) / 4;
    return nb * kMxLimbs * 24 + kq * 16;
}
__device__ __forceinline__ MxVec mx_vec_at(uint8_t *lds, uint32_t kg) {
    MxVec v;
    v.hi = reinterpret_cast<mx_u32x4 *>(lds);
    v.lo = reinterpret_cast<mx_u32x2 *>(lds + (size_t)4 * kg * kMxLimbs * 16);
    v.sc = lds + (size_t)4 * kg * kMxLimbs * 24;
    return v;
}

// Blocks [0, 4 kg) of x's limbs into v by the workgroup (blocks from nb on:
// zeros).  Followed by a barrier.
__device__ __forceinline__ void mx_vec_fill(const MxVec &v, const float *x, uint32_t nb, uint32_t kg) {
    for (uint32_t b = threadIdx.x; b < 4 * kg; b += blockDim.x) {
        mx_f32x16 lo = {}, hi = {};
        if (b < nb) mx_load_block(x + (size_t)b * 32, lo, hi);
        const uint32_t s = mx_limb_scale(mx_top(lo, hi));
        v.sc[(b / 16) * 16 + (b % 4) * 4 + (b / 4) % 4] = (uint8_t)s;
        mx_limbs(lo, hi, s, [&](int j, const mx_u32x6 &q) {
            v.hi[b * kMxLimbs + j] = mx_u32x4{q[0], q[1], q[2], q[3]};
            v.lo[b * kMxLimbs + j] = mx_u32x2{q[4], q[5]};
        });
    }
}

// One lane's way through 16 rows: its row's codes and scales.
struct MxRow {
    const uint8_t *codes;      // + 1024 per group of 4 blocks
    const uint8_t *scales;     // + 256 per group of 16 blocks
};
__device__ __forceinline__ MxRow mx_row_at(const uint8_t *codes, const uint8_t *scales, const MxDims &d, size_t expert,
                                           uint32_t row, int lane) {
    const size_t tile = expert * d.tiles + row / 16;
    const uint32_t l = (uint32_t)(lane & 48) + row % 16;
    return {codes + (tile * d.kg * 64 + l) * 16, scales + (tile * d.kq * 64 + l) * 4};
}

struct MxWords {
    mx_u32x4 c[4];
    uint32_t s;
};
__device__ __forceinline__ void mx_fetch(MxWords &w, const MxRow &r, uint32_t q, uint32_t kg) {
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
        if (4 * q + j < kg) w.c[j] = *reinterpret_cast<const mx_u32x4 *>(r.codes + (size_t)(4 * q + j) * 1024);
    w.s = *reinterpret_cast<const uint32_t *>(r.scales + (size_t)q * 256);
}

// acc += the groups 4 q .. of the rows in w times the vector's.
template <int J>
__device__ __forceinline__ mx_acc16 mx_step(const MxWords &w, const MxVec &v, uint32_t q, uint32_t sv, bool live, int limb,
                                            int lane, mx_acc16 acc) {
    mx_op x = {};
    const uint32_t b = (4 * q + J) * 4 + (uint32_t)(lane >> 4);
    if (live) x = mx_op6(v.hi[b * kMxLimbs + limb], v.lo[b * kMxLimbs + limb]);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_op4(w.c[J]), x, acc, kMxCbszFp4, kMxCbszFp6, J, (int)w.s, J,
                                                            (int)sv);
}
__device__ __forceinline__ mx_acc16 mx_dot(const MxWords &w, const MxVec &v, uint32_t q, uint32_t kg, int lane,
                                           mx_acc16 acc) {
    const int col = lane & 15;
    const bool live = col < kMxLimbs;
    const int limb = live ? col : 0;
    constexpr uint64_t shifts = 0ull | 4ull << 8 | 9ull << 16 | 14ull << 24 | 19ull << 32;
    const uint32_t shift = (uint32_t)(shifts >> (8 * limb)) & 255u;
    // the limb's scale bytes: every byte of the word is at least kMxLeastScale
    const uint32_t sv = reinterpret_cast<const uint32_t *>(v.sc)[q * 4 + (lane >> 4)] - shift * 0x01010101u;
    acc = mx_step<0>(w, v, q, sv, live, limb, lane, acc);
    if (4 * q + 1 < kg) acc = mx_step<1>(w, v, q, sv, live, limb, lane, acc);
    if (4 * q + 2 < kg) acc = mx_step<2>(w, v, q, sv, live, limb, lane, acc);
    if (4 * q + 3 < kg) acc = mx_step<3>(w, v, q, sv, live, limb, lane, acc);
    return acc;
}

// The sums over the columns: row 4 (lane / 16) + i in acc[i] of every lane of
// the 16, then row lane % 16 from lanes of column i = row % 4.
__device__ __forceinline__ float mx_rows(mx_acc16 acc, int lane, bool first) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = group_sum_dpp<16>(acc[i], first);
    const int i = lane & 3;
    return i == 0 ? acc[0] : i == 1 ? acc[1] : i == 2 ? acc[2] : acc[3];
}
// the lane that holds row r of mx_rows is 16 (r / 4) + r % 4: lanes with
// lane % 16 < 4 write row 4 (lane / 16) + lane % 4

__global__ __launch_bounds__(kMvThreads) void k_mx_matvec(const uint8_t *codes, const uint8_t *scales, MxDims d,
                                                          uint32_t rows, uint32_t expert_rows, const float *x, float *y) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kMvWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool first = p32_first(lane);
    const MxVec v = mx_vec_at(lds, d.kg);
    mx_vec_fill(v, x, d.nb, d.kg);
    __syncthreads();
    const size_t ntiles = (size_t)(rows / expert_rows) * d.tiles;
    for (size_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        const size_t expert = tile / d.tiles;
        const uint32_t row0 = (uint32_t)(tile % d.tiles) * 16;
        const MxRow r = mx_row_at(codes, scales, d, expert, row0 + (uint32_t)(lane & 15), lane);
        mx_acc16 acc = {};
        for (uint32_t q = wave; q < d.kq; q += kMvWaves) {
            MxWords w;
            mx_fetch(w, r, q, d.kg);
            acc = mx_dot(w, v, q, d.kg, lane, acc);
        }
        const float t = mx_rows(acc, lane, first);
        if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
        __syncthreads();
        if (threadIdx.x < 16 && row0 + threadIdx.x < expert_rows) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kMvWaves; i++) s += part[i][threadIdx.x];
            y[expert * expert_rows + row0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
}

// h[slot][j] = act(G x)[j] (U x)[j] of expert ids[slot], zeros from F to
// down_cols: waves 0-3 the 16 gate rows, 4-7 the up rows, which may begin
// inside a tile.  G and U are one tensor of 2 F rows an expert, or (ids null)
// two tensors.
struct MxPair {
    const uint8_t *codes[2], *scales[2];
    uint32_t row0[2], rows;  // first row of either half; rows of an expert in memory
    MxDims d;
};
__global__ __launch_bounds__(kMvThreads) void k_mx_gate_up(MxPair p, const float *x, const uint32_t *ids, uint32_t n_experts,
                                                           uint32_t F, uint32_t down_cols, uint32_t act, float *h) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kMvWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t j0 = blockIdx.x * 16, expert = ids ? ids[blockIdx.y] : 0u;
    float *out = h + (size_t)blockIdx.y * down_cols;
    if (j0 >= F || expert >= n_experts) {  // padding (or no such expert)
        if (threadIdx.x < 16 && j0 + threadIdx.x < down_cols) out[j0 + threadIdx.x] = 0.0f;
        return;
    }
    const bool first = p32_first(lane);
    const MxVec v = mx_vec_at(lds, p.d.kg);
    mx_vec_fill(v, x, p.d.nb, p.d.kg);
    __syncthreads();
    const int half = wave >> 2;
    const uint32_t j = min(j0 + (uint32_t)(lane & 15), F - 1);
    const MxRow r = mx_row_at(p.codes[half], p.scales[half], p.d, expert, p.row0[half] + j, lane);
    mx_acc16 acc = {};
    for (uint32_t q = wave & 3; q < p.d.kq; q += 4) {
        MxWords w;
        mx_fetch(w, r, q, p.d.kg);
        acc = mx_dot(w, v, q, p.d.kg, lane, acc);
    }
    const float t = mx_rows(acc, lane, first);
    if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
    __syncthreads();
    if (threadIdx.x < 16 && j0 + threadIdx.x < down_cols) {
        const uint32_t i = threadIdx.x;
        const float g = ((part[0][i] + part[1][i]) + part[2][i]) + part[3][i];
        const float u = ((part[4][i] + part[5][i]) + part[6][i]) + part[7][i];
        out[j0 + i] = j0 + i < F ? act_apply(act, g) * u : 0.0f;
    }
}

// out[i] = sum over slots of w (D_id h[slot])[i]: the waves take the (slot, 16
// blocks) pieces of a tile's rows in turn, `per` slots' limbs in LDS at once.
__global__ __launch_bounds__(kMvThreads) void k_mx_down(const uint8_t *codes, const uint8_t *scales, MxDims d, uint32_t rows,
                                                        uint32_t n_experts, const float *h, const uint32_t *ids,
                                                        const float *wts, uint32_t k, uint32_t per, const float *base,
                                                        int accumulate, const float *dscale, float *out) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kMvWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool first = p32_first(lane);
    const uint32_t row0 = blockIdx.x * 16;
    const size_t vec = mx_vec_bytes(d.kg);
    mx_acc16 sum = {};
    for (uint32_t s0 = 0; s0 < k; s0 += per) {
        const uint32_t n = min(per, k - s0);
        if (s0) __syncthreads();
        for (uint32_t i = 0; i < n; i++)
            mx_vec_fill(mx_vec_at(lds + i * vec, d.kg), h + (size_t)(s0 + i) * d.nb * 32, d.nb, d.kg);
        __syncthreads();
        for (uint32_t it = wave; it < n * d.kq; it += kMvWaves) {
            const uint32_t i = it / d.kq, q = it % d.kq, e = ids[s0 + i];
            if (e >= n_experts) continue;
            const MxRow r = mx_row_at(codes, scales, d, e, row0 + (uint32_t)(lane & 15), lane);
            MxWords w;
            mx_fetch(w, r, q, d.kg);
            const mx_acc16 t = mx_dot(w, mx_vec_at(lds + i * vec, d.kg), q, d.kg, lane, mx_acc16{});
            const float f = dscale ? wts[s0 + i] * dscale[e] : wts[s0 + i];
            sum += t * f;
        }
    }
    const float t = mx_rows(sum, lane, first);
    if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
    __syncthreads();
    const uint32_t row = row0 + threadIdx.x;
    if (threadIdx.x < 16 && row < rows) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kMvWaves; i++) s += part[i][threadIdx.x];
        if (accumulate) s = out[row] + s;
        out[row] = base ? base[row] + s : s;
    }
}

// Limbs of this many bytes at most in a down block's LDS (two blocks a CU).
constexpr size_t kDownLds = 72 << 10;

// Lets a kernel use the CU's LDS, once per kernel and device.
hipError_t allow_lds(const void *fn, bool *set) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    if (set[dev]) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
    if (e == hipSuccess) set[dev] = true;
    return e;
}

}  // namespace

hipError_t launch_matvec_mx(const DevTensor &W, const float *x, float *y, hipStream_t s) {
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    static bool set[64] = {};
    hipError_t e = allow_lds((const void *)k_mx_matvec, set);
    if (e != hipSuccess) return e;
    const size_t tiles = W.n_experts * d.tiles;
    const dim3 grid((unsigned)(tiles < 1024 ? tiles : 1024));
    hipLaunchKernelGGL(k_mx_matvec, grid, dim3(kMvThreads), mx_vec_bytes(d.kg), s, W.p0, W.p1, d, (uint32_t)W.total_rows,
                       (uint32_t)W.rows, x, y);
    return hipGetLastError();
}

static hipError_t launch_pair(const MxPair &p, const float *x, const uint32_t *ids, uint32_t n_experts, uint32_t k,
                              uint32_t F, uint32_t down_cols, uint32_t act, float *h, hipStream_t s) {
    static bool set[64] = {};
    hipError_t e = allow_lds((const void *)k_mx_gate_up, set);
    if (e != hipSuccess) return e;
    const dim3 grid((down_cols + 15) / 16, k);
    hipLaunchKernelGGL(k_mx_gate_up, grid, dim3(kMvThreads), mx_vec_bytes(p.d.kg), s, p, x, ids, n_experts, F, down_cols, act,
                       h);
    return hipGetLastError();
}

hipError_t launch_gate_up_mx(const DevTensor &G, const DevTensor &U, const float *x, uint32_t act, uint32_t down_cols,
                             float *h, hipStream_t s) {
    MxPair p{{G.p0, U.p0}, {G.p1, U.p1}, {0, 0}, (uint32_t)G.rows, mx_dims(G.rows, G.blocks_per_row)};
    return launch_pair(p, x, nullptr, 1, 1, (uint32_t)G.rows, down_cols, act, h, s);
}

hipError_t launch_expert_gate_up_mx(const DevTensor &GU, const float *x, const uint32_t *ids, uint32_t k, uint32_t d_expert,
                                    uint32_t down_cols, uint32_t act, float *h, hipStream_t s) {
    MxPair p{{GU.p0, GU.p0}, {GU.p1, GU.p1}, {0, d_expert}, (uint32_t)GU.rows, mx_dims(GU.rows, GU.blocks_per_row)};
    return launch_pair(p, x, ids, (uint32_t)GU.n_experts, k, d_expert, down_cols, act, h, s);
}

hipError_t launch_expert_down_mx(const DevTensor &D, const float *h, const uint32_t *ids, const float *w, uint32_t k,
                                 const float *base, int accumulate, const float *dscale, float *out, hipStream_t s) {
    const MxDims d = mx_dims(D.rows, D.blocks_per_row);
    static bool set[64] = {};
    hipError_t e = allow_lds((const void *)k_mx_down, set);
    if (e != hipSuccess) return e;
    const size_t vec = mx_vec_bytes(d.kg);
    uint32_t per = (uint32_t)(kDownLds / vec);
    per = per < 1 ? 1 : per > k ? k : per;
    hipLaunchKernelGGL(k_mx_down, dim3((unsigned)d.tiles), dim3(kMvThreads), per * vec, s, D.p0, D.p1, d, (uint32_t)D.rows,
                       (uint32_t)D.n_experts, h, ids, w, k, per, base, accumulate, dscale, out);
    return hipGetLastError();
}

}  // namespace lt
