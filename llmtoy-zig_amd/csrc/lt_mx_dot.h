// lt_mx_dot.h -- products of rows of MXFP4 with a vector or a few, as the matvec, the experts'
// kernels and the single-launch layer have them.
//
//   y[r] = sum_b 2^(e_rb - 127) sum_i w_rbi x_bi
//
// A weight times its block's scale is a bf16 number (2 bits times a power of
// two; scale bytes 253 and 254 have weights beyond them, see DevTensor::beyond), and v_cvt_scalef32_pk_bf16_fp4 makes two of them from a byte.  An
// activation is the sum of three bf16 numbers of 8 bits each, cut off from the
// top, exactly (from 2^-110 on; bits below 2^-133 are no bf16 number's).  So v_mfma_f32_16x16x32_bf16 with 16 rows of weights on one
// side and the three parts as columns on the other gives the products with the
// fp32 activations; the row's sum over the columns is y.  (The scaled
// instruction, which takes the codes as they are, needs activations in FP6:
// their conversion is 32 values wide and cost every workgroup 0.7 us before its
// first product, three parts cut off by masks 0.1.  FP8 operands converted in
// pairs are no way out: sums with them were 1e-4 off.)
#pragma once

#include "lt_internal.h"
#include "lt_mx.h"

namespace lt {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A vector's three parts in LDS: [block][quarter][part], 8 bf16 each, in the
// order of the codes (position 2 i: element i, 2 i + 1: element 16 + i).  (A wave's
// reads, 4 blocks by 3 parts, fall on different banks.)
constexpr int kParts = 3;
__host__ __device__ inline size_t mx_vec_bytes(uint32_t kg) { return (size_t)kg * 4 * 4 * kParts * 16; }

// Quarter u % 4 of block u / 4 (blocks from nb on: the last one again, against
// weights of zero).
struct MxQuarter {
    float4 a, h;  // elements 4 m .. + 3 and 16 + 4 m .. + 3
};
__device__ __forceinline__ MxQuarter mx_vec_load(const float *x, uint32_t u, uint32_t nb) {
    const float *p = x + (size_t)min(u / 4, nb - 1) * 32 + u % 4 * 4;
    return {ldg16f(p), ldg16f(p + 16)};
}
// NV vectors side by side: vector n's parts are 3 n .. of [block][quarter][3 NV].
template <int NV = 1>
__device__ __forceinline__ void mx_vec_put(mx_u32x4 *v, uint32_t u, const MxQuarter &x, int n = 0) {
    float a[4] = {x.a.x, x.a.y, x.a.z, x.a.w}, h[4] = {x.h.x, x.h.y, x.h.z, x.h.w};
#pragma unroll
    for (int c = 0; c < kParts; c++) {
        mx_u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t ua = __float_as_uint(a[i]), uh = __float_as_uint(h[i]);
            w[i] = __builtin_amdgcn_perm(uh, ua, 0x07060302u);  // the upper halves
            a[i] -= __uint_as_float(ua & 0xffff0000u);
            h[i] -= __uint_as_float(uh & 0xffff0000u);
        }
        v[u * (kParts * NV) + kParts * n + c] = w;
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
// NT: read past the caches, which then keep what is read again (experts are).
template <bool NT>
__device__ __forceinline__ void mx_fetch(MxWords &w, const MxRow &r, uint32_t q, uint32_t kg) {
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
        if (4 * q + j < kg) {
            const mx_u32x4 *p = reinterpret_cast<const mx_u32x4 *>(r.codes + (size_t)(4 * q + j) * 1024);
            w.c[j] = NT ? __builtin_nontemporal_load(p) : *p;
        }
    w.s = *reinterpret_cast<const uint32_t *>(r.scales + (size_t)q * 256);
}

// acc += the groups 4 q .. of the rows in w times the vector's.  Columns from 3
// on repeat the third: mx_rows leaves them out.
struct MxSum {
    mx_acc16 s[4];  // chains
    __device__ __forceinline__ mx_acc16 all() const { return (s[0] + s[1]) + (s[2] + s[3]); }
};
template <int J, int NV>
__device__ __forceinline__ void mx_step(const MxWords &w, const mx_u32x4 *v, MxSum &acc) {
    // a float whose exponent is the scale byte: 2^(e - 127), 255 makes NaN
    const float scale = __uint_as_float((J < 3 ? w.s << (23 - 8 * J) : w.s >> 1) & 0x7f800000u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        union {
            bf16x2 p[4];
            bf16x8 v;
        } m;
        m.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.c[J][i], scale, 0);
        m.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.c[J][i], scale, 1);
        m.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.c[J][i], scale, 2);
        m.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.c[J][i], scale, 3);
        const bf16x8 x = __builtin_bit_cast(bf16x8, v[(16 * J + i) * (kParts * NV)]);
        acc.s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m.v, x, acc.s[i], 0, 0, 0);
    }
}
template <int NV = 1>
__device__ __forceinline__ void mx_dot(const MxWords &w, const mx_u32x4 *v, uint32_t q, uint32_t kg, int lane, MxSum &acc) {
    v += ((16 * q + (uint32_t)(lane >> 4)) * 4) * (kParts * NV) + min(lane & 15, kParts * NV - 1);
    mx_step<0, NV>(w, v, acc);
    if (4 * q + 1 < kg) mx_step<1, NV>(w, v, acc);
    if (4 * q + 2 < kg) mx_step<2, NV>(w, v, acc);
    if (4 * q + 3 < kg) mx_step<3, NV>(w, v, acc);
}

// The sums over the columns: row 4 (lane / 16) + i in acc[i] of every lane of
// the 16, then row lane % 16 from lanes of column i = row % 4.
__device__ __forceinline__ float mx_rows(mx_acc16 acc, int lane, bool first) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = group_sum_dpp<16>((lane & 15) < kParts ? acc[i] : 0.0f, first);
    const int i = lane & 3;
    return i == 0 ? acc[0] : i == 1 ? acc[1] : i == 2 ? acc[2] : acc[3];
}
// the lane that holds row r of mx_rows is 16 (r / 4) + r % 4: lanes with
// lane % 16 < 4 write row 4 (lane / 16) + lane % 4

// Of several vectors: the sum over the three columns of vector n in lanes of column
// 3 n, row 4 (lane / 16) + i in [i].
__device__ __forceinline__ mx_acc16 mx_rows_of(mx_acc16 acc) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float one = dpp<0x101>(acc[i]), two = dpp<0x102>(acc[i]);  // lanes + 1, + 2
        acc[i] = (acc[i] + one) + two;
    }
    return acc;
}

// Loads stay behind this point, or before it.
__device__ __forceinline__ void mx_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Division of u by a number that the host knows, as a multiplication: exact for
// u d < 2^32.  (A division takes a chain of 30 instructions, and these stand
// before a kernel's first loads.)
struct MxDiv {
    uint32_t d, m;
    __device__ __forceinline__ uint32_t by(uint32_t u) const { return d == 1 ? u : __umulhi(u, m); }
};
inline MxDiv mx_div(uint32_t d) { return {d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }

struct MxRoute {
    const float *logits;
    uint32_t k, norm, *ids;
    float *w;
};
struct MxPair {
    const uint8_t *codes[2], *scales[2];
    uint32_t row0[2];  // first row of either half
    MxDims d;
};
constexpr uint32_t kPairWaves = 8, kPairThreads = 64 * kPairWaves;
// Rows j0 .. j0 + 15 of an expert's h, by a workgroup: vector() between the first
// loads and the products puts x into v; put(i, h) by thread i.
template <class Vector, class Put>
__device__ __forceinline__ void mx_gate_rows(const MxPair &p, uint32_t expert, uint32_t j0, uint32_t F, uint32_t down_cols,
                                             uint32_t act, const mx_u32x4 *v, float (*part)[16], Vector vector, Put put) {
    constexpr uint32_t S = kPairWaves / 2;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave / S, sp = wave % S;
    const MxDims &d = p.d;
    const bool first = p32_first(lane);
    const uint32_t j = min(j0 + (uint32_t)(lane & 15), F - 1);
    const MxRow r = mx_row_at(half ? p.codes[1] : p.codes[0], half ? p.scales[1] : p.scales[0], d, expert,
                              (half ? p.row0[1] : p.row0[0]) + j, lane);
    MxWords w0, w1;
    if (sp < d.kq) mx_fetch<false>(w0, r, sp, d.kg);
    if (sp + S < d.kq) mx_fetch<false>(w1, r, sp + S, d.kg);
    mx_order();
    vector();
    MxSum acc = {};
    for (uint32_t q = sp; q < d.kq; q += 2 * S) {
        mx_dot(w0, v, q, d.kg, lane, acc);
        if (q + 2 * S < d.kq) mx_fetch<false>(w0, r, q + 2 * S, d.kg);
        if (q + S < d.kq) mx_dot(w1, v, q + S, d.kg, lane, acc);
        if (q + 3 * S < d.kq) mx_fetch<false>(w1, r, q + 3 * S, d.kg);
    }
    const float t = mx_rows(acc.all(), lane, first);
    if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
    __syncthreads();
    if (threadIdx.x < 16 && j0 + threadIdx.x < down_cols) {
        const uint32_t i = threadIdx.x;
        float g = part[0][i], u = part[S][i];
        for (uint32_t k = 1; k < S; k++) {
            g += part[k][i];
            u += part[S + k][i];
        }
        put(i, j0 + i < F ? act_apply(act, g) * u : 0.0f);
    }
}

// Lets a kernel use the CU's LDS, once per kernel and device.
inline hipError_t allow_lds(const void *fn, bool *set) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    if (set[dev]) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
    if (e == hipSuccess) set[dev] = true;
    return e;
}

}  // namespace lt
