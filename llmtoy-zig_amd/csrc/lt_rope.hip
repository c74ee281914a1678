// lt_rope.hip -- RMS norms of queries and keys for each head and the position
// rotation, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w      (w null: without; (1 + w) with LT_NORM_ONE_PLUS_W)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t) for the pairs (a, b) of the
//   first n_rot elements: (i, i + n_rot / 2) or (2 i, 2 i + 1)
//
// The angle is counted in turns, position * turns[i], in 64 bits: at a position
// of a million fp32 would be 0.05 turns off.  What is left of the whole turns,
// within half a turn, is exact enough for fp32.
//
// Bound by the reads and writes of the heads.  A group of lanes takes a token's
// heads, HB at a time, and finds the token's angles once; the angles of
// one pair take about 60 instructions, 15 times those of turning it.
// 4,095 tokens of 16 + 8 heads of 256, half of each turned: 48 us, 4.2 TB/s; one token of 36
// heads of 128 3.3 us in a graph's row of 16.
#include "llmtoy_hip.h"
#include "lt_kv.h"

namespace lt {

namespace {

struct RopeArgs {
    const double *turns;
    const float *q, *k, *wq, *wk;
    float *q_out, *k_out;
    const uint32_t *pos;
    size_t q_stride, k_stride, q_out_stride, k_out_stride;
    uint32_t T, n_heads, n_all, per, parts, D, n_rot, neox, norm;  // per: heads a group; parts: groups a token
    float eps, bias;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
// (MANY: past the caches; 4,095 tokens of 24 heads of 256: 52 -> 48 us, of 36 of 128 36 -> 31)
template <bool MANY>
__device__ __forceinline__ void put(float *to, const float *v) {
    const f32x4 x = {v[0], v[1], v[2], v[3]};
    if (MANY) __builtin_nontemporal_store(x, reinterpret_cast<f32x4 *>(to));
    else *reinterpret_cast<f32x4 *>(to) = x;
}

// V consecutive pairs a lane and step, W lanes a head, KP steps, HB heads at a time.
template <int V, int W, int KP, int HB>
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs a) {
    const uint32_t lane = threadIdx.x % W;
    const size_t group = (size_t)blockIdx.x * (256 / W) + threadIdx.x / W;
    if (group >= (size_t)a.T * a.parts) return;  // (whole groups of lanes: the shuffles stay among them)
    const uint32_t t = (uint32_t)(group / a.parts), h0 = (uint32_t)(group % a.parts) * a.per;
    const uint32_t h1 = h0 + a.per < a.n_all ? h0 + a.per : a.n_all;
    const uint32_t half = a.n_rot / 2, pairs = a.D / 2;
    // the lane's 2 V elements: V in a row from at, V from to
    uint32_t at[KP], to[KP];
#pragma unroll
    for (int i = 0; i < KP; i++) {
        const uint32_t p = (lane + i * W) * V;
        const bool turned = p < half;  // (half is a whole number of V)
        if (a.neox) {
            at[i] = turned ? p : a.n_rot + (p - half) * 2;
            to[i] = turned ? p + half : at[i] + V;
        } else {
            at[i] = 2 * p;
            to[i] = 2 * p + V;
        }
    }
    const auto get = [&](const float *x, int i, float (&u)[2 * V]) {
        if ((lane + i * W) * V >= pairs) {
#pragma unroll
            for (int j = 0; j < 2 * V; j++) u[j] = 0.0f;
        } else if constexpr (V == 4) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(x + at[i]), hi = *reinterpret_cast<const f32x4 *>(x + to[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = lo[j], u[4 + j] = hi[j];
        } else {
            u[0] = x[at[i]], u[1] = x[to[i]];
        }
    };
    const auto head_of = [&](uint32_t h) {
        return h < a.n_heads ? a.q + (size_t)t * a.q_stride + (size_t)h * a.D
                             : a.k + (size_t)t * a.k_stride + (size_t)(h - a.n_heads) * a.D;
    };
    // everything that is read first, side by side: the heads, the position and rates, the weights
    float u[HB][KP][2 * V], g[2][KP][2 * V];
    const auto fetch = [&](uint32_t h) {
#pragma unroll
        for (int b = 0; b < HB; b++)
#pragma unroll
            for (int i = 0; i < KP; i++) get(head_of(h + b < h1 ? h + b : h1 - 1), i, u[b][i]);
    };
    fetch(h0);
    const uint32_t pos = a.pos[t];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float *w = k ? a.wk : a.wq;
#pragma unroll
        for (int i = 0; i < KP; i++) {
            if (a.norm && w) get(w, i, g[k][i]);
#pragma unroll
            for (int j = 0; j < 2 * V; j++) g[k][i][j] = a.norm && w ? a.bias + g[k][i][j] : 1.0f;
        }
    }
    float cs[KP][V], sn[KP][V];
#pragma unroll
    for (int i = 0; i < KP; i++) {
        const uint32_t p = (lane + i * W) * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
            cs[i][j] = 1.0f, sn[i][j] = 0.0f;
            if (p < half) {
                const double turn = (double)pos * a.turns[p + j];
                sincospif(2.0f * (float)(turn - rint(turn)), &sn[i][j], &cs[i][j]);
            }
        }
    }
    for (uint32_t h = h0; h < h1; h += HB) {
        if (h != h0) fetch(h);
#pragma unroll
        for (int b = 0; b < HB; b++) {
            if (h + b >= h1) break;
            const bool is_q = h + b < a.n_heads;
            float *y = is_q ? a.q_out + (size_t)t * a.q_out_stride + (size_t)(h + b) * a.D
                            : a.k_out + (size_t)t * a.k_out_stride + (size_t)(h + b - a.n_heads) * a.D;
            float r = 1.0f;
            if (a.norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < KP; i++)
#pragma unroll
                    for (int j = 0; j < 2 * V; j++) ss += u[b][i][j] * u[b][i][j];
#pragma unroll
                for (int off = W / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, W);
                r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
            }
#pragma unroll
            for (int i = 0; i < KP; i++) {
                if ((lane + i * W) * V >= pairs) continue;
                float v[2 * V], o[2 * V];
#pragma unroll
                for (int j = 0; j < 2 * V; j++) v[j] = u[b][i][j] * (r * (is_q ? g[0][i][j] : g[1][i][j]));
                if (a.neox) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        o[j] = v[j] * cs[i][j] - v[j + V] * sn[i][j];
                        o[j + V] = v[j] * sn[i][j] + v[j + V] * cs[i][j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        o[2 * j] = v[2 * j] * cs[i][j] - v[2 * j + 1] * sn[i][j];
                        o[2 * j + 1] = v[2 * j] * sn[i][j] + v[2 * j + 1] * cs[i][j];
                    }
                }
                if constexpr (V == 4) {
                    put<(HB > 1)>(y + at[i], o);
                    put<(HB > 1)>(y + to[i], o + 4);
                } else {
                    y[at[i]] = o[0];
                    y[to[i]] = o[1];
                }
            }
        }
    }
}

template <int V, int W, int KP>
void go(RopeArgs &a, hipStream_t s) {
    // heads a group: enough groups to fill the chip before angles are shared
    constexpr uint32_t kEnough = 256 * 16 * (kWave / W);
    a.per = 1;
    while (a.per < a.n_all && (uint64_t)a.T * ((a.n_all + 2 * a.per - 1) / (2 * a.per)) >= kEnough) a.per *= 2;
    a.parts = (a.n_all + a.per - 1) / a.per;
    const size_t groups = (size_t)a.T * a.parts;
    const dim3 grid((unsigned)((groups + 256 / W - 1) / (256 / W)));
    if (a.per == 1) hipLaunchKernelGGL((k_qk_norm_rope<V, W, KP, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_qk_norm_rope<V, W, KP, (V == 4 ? 4 : 2)>), grid, dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeDev &rope, float *q_out, float *k_out, const float *q, const float *k,
                               const float *wq, const float *wk, const uint32_t *pos, uint32_t T, uint32_t n_heads,
                               uint32_t n_kv, const size_t stride[4], float eps, bool norm, bool one_plus,
                               hipStream_t s) {
    RopeArgs a{};
    a.turns = rope.turns;
    a.q = q, a.k = k, a.wq = wq, a.wk = wk, a.q_out = q_out, a.k_out = k_out, a.pos = pos;
    a.q_stride = stride[0], a.k_stride = stride[1], a.q_out_stride = stride[2], a.k_out_stride = stride[3];
    a.T = T, a.n_heads = n_heads, a.n_all = n_heads + n_kv, a.D = rope.D, a.n_rot = rope.n_rot;
    a.neox = rope.style == LT_ROPE_NEOX;
    a.norm = norm, a.eps = eps, a.bias = one_plus ? 1.0f : 0.0f;
    if (rope.D == 0 || rope.D % 2 || rope.D > 512 || T == 0 || a.n_all == 0) return hipErrorInvalidValue;
    // 16-byte accesses where every piece of four lies on 16 bytes
    const void *ptr[] = {q, k, wq, wk, q_out, k_out};
    bool wide = rope.D % 8 == 0 && rope.n_rot % 8 == 0;
    for (const void *p : ptr) wide &= (uintptr_t)p % 16 == 0;
    for (int i = 0; i < 4; i++) wide &= stride[i] % 4 == 0;
    if (wide) {
        const uint32_t lanes = rope.D / 8;
        if (lanes <= 8) go<4, 8, 1>(a, s);
        else if (lanes <= 16) go<4, 16, 1>(a, s);
        else if (lanes <= 32) go<4, 32, 1>(a, s);
        else go<4, 64, 1>(a, s);
    } else if (rope.D <= 128) {
        go<1, 64, 1>(a, s);
    } else {
        go<1, 64, 4>(a, s);
    }
    return hipGetLastError();
}

}  // namespace lt
