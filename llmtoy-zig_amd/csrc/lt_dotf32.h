// lt_dotf32.h -- a router row's logit in dotf32's order (ops/math.zig:96-116), by
// two wavefronts: the router's kernel and the single-launch router with experts.
#pragma once

#include "lt_internal.h"

namespace lt {

// wr . x (+ *bias) for 32 nit elements (nit a multiple of 8), x and wr on 16 bytes.
// Of the two wavefronts h = 0, 1, h takes chains 16 h + [0, 16), so that a row is on
// its way in 16-byte loads (lane L of load q: stride 16 q + L / 4, chains 4 (L & 3)
// + [0, 4) of the wavefront's).  The products of a load pass through LDS (prod: two
// [16][16] buffers of the wavefront) to the chain lanes (chain c = lane & 15), which
// add them stride by stride; (acc0 + acc1) is formed in each wavefront, (acc2 +
// acc3) crosses to the first one (xch: 8 floats of the row), which finishes the
// ordered sum: dotf32's rounded operations in its order.  Loads go in batches of 4
// (2,048 elements), the next batch's before this one's products are added.  Called by
// whole workgroups; the sum is h = 0's.
__device__ __forceinline__ float dotf32_pair(const float *wr, const float *x, const float *bias, int nit, int h, int lane,
                                             float *prod, float *xch) {
#pragma clang fp contract(off)
    float4 wv[2][4], xv[2][4];
    auto load_batch = [&](int b, int qb) {  // unconditional: strides clamped
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int it = min(16 * (qb + q) + (lane >> 2), nit - 1);
            const int e = 32 * it + 16 * h + 4 * (lane & 3);
            wv[b][q] = ldg16f(wr + e);
            xv[b][q] = ldg16f(x + e);
        }
    };
    load_batch(0, 0);
    const float bv = bias ? *bias : 0.0f;
    float acc = 0.0f;
    auto add_batch = [&](int b, int qb) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (16 * (qb + q) < nit) {
                float4 pr;
                pr.x = wv[b][q].x * xv[b][q].x;
                pr.y = wv[b][q].y * xv[b][q].y;
                pr.z = wv[b][q].z * xv[b][q].z;
                pr.w = wv[b][q].w * xv[b][q].w;
                float *buf = prod + (q & 1) * 256;
                *reinterpret_cast<float4 *>(buf + 4 * lane) = pr;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                const int n = nit - 16 * (qb + q);  // 8 (the rest is not added) or 16 and more
                float v[16];
#pragma unroll
                for (int u = 0; u < 16; u++) v[u] = buf[u * 16 + (lane & 15)];
#pragma unroll
                for (int u0 = 0; u0 < 16; u0 += 8)
                    if (u0 < n)
#pragma unroll
                        for (int u = 0; u < 8; u++) acc = acc + v[u0 + u];
            }
        }
    };
    for (int qb = 0; 16 * qb < nit; qb += 8) {
        if (16 * (qb + 4) < nit) load_batch(1, qb + 4);
        add_batch(0, qb);
        if (16 * (qb + 4) < nit) {
            if (16 * (qb + 8) < nit) load_batch(0, qb + 8);
            add_batch(1, qb + 4);
        }
    }
    const float s2 = acc + dpp<0x128>(acc);  // lanes l < 8: chains 16 h + l and 16 h + l + 8
    if (h == 1 && lane < 8) xch[lane] = s2;
    __syncthreads();
    if (h != 0) return 0.0f;
    const float a8 = s2 + xch[lane & 7];
    float sum = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a8), 0));
#pragma unroll
    for (int l = 1; l < 8; l++) sum = sum + __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a8), l));
    if (bias) sum = sum + bv;
    return sum;
}

// The same for any nit.  LEAN keeps 4 loads in registers instead of 8, the next one under
// way as soon as one's products are formed (where 80 registers are all there are).  (128
// rows of 2,048: 5.4 us with the top-k, 5.15 above.)
template <bool LEAN>
__device__ __forceinline__ float dotf32_pair_any(const float *wr, const float *x, const float *bias, int nit, int h, int lane,
                                                 float *prod, float *xch) {
#pragma clang fp contract(off)
    constexpr int kBatches = LEAN ? 1 : 2;
    float4 wv[kBatches][4], xv[kBatches][4];
    auto load = [&](int b, int j, int q) {  // unconditional: strides clamped
        const int it = min(16 * q + (lane >> 2), nit - 1);
        const int e = 32 * it + 16 * h + 4 * (lane & 3);
        wv[b][j] = ldg16f(wr + e);
        xv[b][j] = ldg16f(x + e);
    };
    auto load_batch = [&](int b, int qb) {
#pragma unroll
        for (int j = 0; j < 4; j++) load(b, j, qb + j);
    };
    load_batch(0, 0);
    const float bv = bias ? *bias : 0.0f;
    float acc = 0.0f;
    auto add_batch = [&](int b, int qb) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (16 * (qb + j) < nit) {
                float4 pr;
                pr.x = wv[b][j].x * xv[b][j].x;
                pr.y = wv[b][j].y * xv[b][j].y;
                pr.z = wv[b][j].z * xv[b][j].z;
                pr.w = wv[b][j].w * xv[b][j].w;
                float *buf = prod + (j & 1) * 256;
                *reinterpret_cast<float4 *>(buf + 4 * lane) = pr;
                if (LEAN && 16 * (qb + 4 + j) < nit) load(b, j, qb + 4 + j);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                const int n = nit - 16 * (qb + j);  // strides left: up to 16 of them are added
                float v[16];
#pragma unroll
                for (int u = 0; u < 16; u++) v[u] = buf[u * 16 + (lane & 15)];
                if (n >= 16) {
#pragma unroll
                    for (int u = 0; u < 16; u++) acc = acc + v[u];
                } else {
#pragma unroll
                    for (int u = 0; u < 15; u++)
                        if (u < n) acc = acc + v[u];
                }
            }
        }
    };
    if constexpr (LEAN) {
        for (int qb = 0; 16 * qb < nit; qb += 4) add_batch(0, qb);
    } else {
        for (int qb = 0; 16 * qb < nit; qb += 8) {
            if (16 * (qb + 4) < nit) load_batch(1, qb + 4);
            add_batch(0, qb);
            if (16 * (qb + 4) < nit) {
                if (16 * (qb + 8) < nit) load_batch(0, qb + 8);
                add_batch(1, qb + 4);
            }
        }
    }
    const float s2 = acc + dpp<0x128>(acc);  // lanes l < 8: chains 16 h + l and 16 h + l + 8
    if (h == 1 && lane < 8) xch[lane] = s2;
    __syncthreads();
    if (h != 0) return 0.0f;
    const float a8 = s2 + xch[lane & 7];
    float sum = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a8), 0));
#pragma unroll
    for (int l = 1; l < 8; l++) sum = sum + __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a8), l));
    if (bias) sum = sum + bv;
    return sum;
}

}  // namespace lt
