// lt_mx.h -- MXFP4 tensors on the device and the operands their products are
// made of.
//
// A block is 32 elements of a row: a scale byte e (2^(e - 127); 255: NaN) and
// 32 four-bit codes, a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6.  The matrix
// instructions with block scales (v_mfma_scale_f32_*_f8f6f4) take such blocks
// as they are: a lane holds one block of one row (16 bytes of codes, its scale
// byte in a register of its own).  So the device layout is the operand's:
//
//   codes   [tile of 16 rows][group of 4 blocks][64 lanes][16 B]
//   scales  [tile of 16 rows][4 groups][64 lanes][4 B]
//
// where lane 16 (b % 4) + row % 16 of group b / 4 holds block b of the row,
// and byte g of its scale word is the scale in group 4 q + g.  A wavefront's
// load of a group is 1 KiB in a row, and one word holds the scales of four.
// Rows are padded to 16 per expert, blocks to groups of 4 (scales: 16), with
// zeros: they add nothing.
//
// Inside a block the codes stand in GGUF's order: byte i holds element i (low
// half) and 16 + i (high half), so position 2 i is element i and 2 i + 1 is
// element 16 + i.  v_cvt_scalef32_2xpk16_fp6_f32 of (elements 0..15, elements
// 16..31) interleaves the same way, which makes the other operand's order.
//
// fp32 activations as matrix operands.  A block of 32 values becomes five FP6
// (E2M3) limbs over one power of two: with s such that the largest |x| / s is
// in (3.875, 7.75],
//   x / s = q0 + q1 / 2^4 + q2 / 2^9 + q3 / 2^14 + q4 / 2^19 + r
// E2M3 is exact to 1/16 up to 2, 1/8 up to 4 and 1/4 up to 7.75, so the first
// remainder is at most 1/4 (times 2^4: 4), each next at most 1/8 (times 2^5:
// 4), and |r| <= 2^-22: 2^-24 of the block's largest value, the error of fp32
// itself.  Products of E2M1 and E2M3 are exact and the sums are fp32, so the
// result is that of fp32 activations.  FP6 runs at the rate of FP4 (measured
// 8.7 PFLOP/s; FP4 with FP8 4.7): five limbs leave 1.7 PFLOP/s, where f16
// activations in two limbs of 11 bits would leave half of 2.5 and need the
// weights converted besides.
#pragma once

#include "lt_internal.h"

namespace lt {

constexpr int kMxLimbs = 5;
constexpr int kMxCbszFp6 = 2, kMxCbszFp4 = 4;  // operand formats of the instruction
// scale exponents of the limbs below the first one's
constexpr uint32_t kMxLimbShift[kMxLimbs] = {0, 4, 9, 14, 19};
// keeps the last limb's unit a normal number: of blocks below 2^-105, 2^-129 may be lost
// (more than 2^-24 of the largest)
constexpr uint32_t kMxLeastScale = 20;

typedef int mx_op __attribute__((ext_vector_type(8)));          // a matrix operand's registers
typedef float mx_acc16 __attribute__((ext_vector_type(4)));     // 16 x 16 sums
typedef float mx_acc32 __attribute__((ext_vector_type(16)));    // 32 x 32 sums
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
typedef float mx_f32x32 __attribute__((ext_vector_type(32)));
typedef unsigned int mx_u32x6 __attribute__((ext_vector_type(6)));
typedef unsigned int mx_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int mx_u32x2 __attribute__((ext_vector_type(2)));

// Sizes of a tensor's two planes.
struct MxDims {
    uint32_t nb;    // blocks of a row
    uint32_t kg;    // groups of 4 blocks
    uint32_t kq;    // groups of 16 blocks (scale words)
    size_t tiles;   // 16-row tiles of an expert
};
__host__ __device__ inline MxDims mx_dims(size_t rows, size_t nb) {
    MxDims d;
    d.nb = (uint32_t)nb;
    d.kg = (uint32_t)((nb + 3) / 4);
    d.kq = (d.kg + 3) / 4;
    d.tiles = (rows + 15) / 16;
    return d;
}
// Behind the planes a tile's codes and 4 KiB more are allocated: the batched
// product takes 32 rows at once, and its last loads run a few blocks past a
// row's end, so it may read (never use) what is there.
inline size_t mx_slack_bytes(const MxDims &d) { return (size_t)d.kg * 1024 + 4096; }
inline size_t mx_code_bytes(const MxDims &d, size_t n_experts) { return n_experts * d.tiles * d.kg * 1024; }
inline size_t mx_scale_bytes(const MxDims &d, size_t n_experts) { return n_experts * d.tiles * d.kq * 256; }

// Where block b of row `row` (of the tile's expert) stands.
__device__ __forceinline__ size_t mx_code_at(const MxDims &d, size_t tile, uint32_t row16, uint32_t b) {
    return ((tile * d.kg + b / 4) * 64 + (b % 4) * 16 + row16) * 16;
}
__device__ __forceinline__ size_t mx_scale_at(const MxDims &d, size_t tile, uint32_t row16, uint32_t b) {
    return ((tile * d.kq + b / 16) * 64 + (b % 4) * 16 + row16) * 4 + (b / 4) % 4;
}

__device__ __forceinline__ mx_op mx_op4(mx_u32x4 v) {
    return mx_op{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}
__device__ __forceinline__ mx_op mx_op6(mx_u32x4 v, mx_u32x2 w) {
    return mx_op{(int)v[0], (int)v[1], (int)v[2], (int)v[3], (int)w[0], (int)w[1], 0, 0};
}

// The largest |x| of a block; NaN where one is.
__device__ __forceinline__ float mx_top(const mx_f32x16 &a, const mx_f32x16 &b) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++)
        m = __builtin_elementwise_maximum(m, __builtin_elementwise_maximum(__builtin_fabsf(a[i]), __builtin_fabsf(b[i])));
    return m;
}

// The scale byte of a block of activations: 255 (NaN) where a value is NaN or
// infinite.
__device__ __forceinline__ uint32_t mx_limb_scale(float largest) {
    const uint32_t top = __float_as_uint(largest);
    if (top >= 0x7f800000u) return 255u;
    const uint32_t s = (top >> 23) + ((top & 0x7fffffu) > 0x780000u ? 1u : 0u);
    return s < kMxLeastScale + 2 ? kMxLeastScale : s - 2;
}

// The limbs of a block of 32 activations (a: elements 0..15, b: 16..31) of
// scale byte s; put(limb, operand words).
template <typename Put>
__device__ __forceinline__ void mx_limbs(mx_f32x16 a, mx_f32x16 b, uint32_t s, Put put) {
#pragma unroll
    for (int j = 0; j < kMxLimbs; j++) {
        // (s = 255: the words do not matter, every product with the block is NaN)
        const float unit = __uint_as_float((min(s, 253u) - kMxLimbShift[j]) << 23);
        const mx_u32x6 q = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, unit);
        put(j, q);
        if (j + 1 < kMxLimbs) {
            const mx_f32x32 back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q, unit);
#pragma unroll
            for (int i = 0; i < 16; i++) {  // exact: the remainder has fewer bits
                a[i] -= back[2 * i];
                b[i] -= back[2 * i + 1];
            }
        }
    }
}

__device__ __forceinline__ float4 ldg16f_nt(const float *p) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p));
    return make_float4(v.x, v.y, v.z, v.w);
}

// 32 floats at x (16-byte aligned)
__device__ __forceinline__ void mx_load_block(const float *x, mx_f32x16 &a, mx_f32x16 &b) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 u = ldg16f(x + 4 * i), v = ldg16f(x + 16 + 4 * i);
        a[4 * i] = u.x; a[4 * i + 1] = u.y; a[4 * i + 2] = u.z; a[4 * i + 3] = u.w;
        b[4 * i] = v.x; b[4 * i + 1] = v.y; b[4 * i + 2] = v.z; b[4 * i + 3] = v.w;
    }
}

}  // namespace lt
