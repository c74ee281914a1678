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
// heads one after the other and finds the token's angles once; the angles of
// one pair take about 60 instructions, 15 times those of turning it.
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

// V consecutive pairs a lane and step, W lanes a head, KP steps.
template <int V, int W, int KP>
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs a) {
    const uint32_t lane = threadIdx.x % W;
    const size_t group = (size_t)blockIdx.x * (256 / W) + threadIdx.x / W;
    if (group >= (size_t)a.T * a.parts) return;  // (whole groups of lanes: the shuffles stay among them)
    const uint32_t t = (uint32_t)(group / a.parts), h0 = (uint32_t)(group % a.parts) * a.per;
    const uint32_t h1 = h0 + a.per < a.n_all ? h0 + a.per : a.n_all;
    const uint32_t half = a.n_rot / 2, pairs = a.D / 2;
    // the lane's 2 V elements: V in a row from at, V from to
    uint32_t at[KP], to[KP];
    float cs[KP][V], sn[KP][V];
    const uint32_t pos = a.pos[t];
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
#pragma unroll
        for (int j = 0; j < V; j++) {
            cs[i][j] = 1.0f, sn[i][j] = 0.0f;
            if (turned) {
                const double turn = (double)pos * a.turns[p + j];
                sincospif(2.0f * (float)(turn - rint(turn)), &sn[i][j], &cs[i][j]);
            }
        }
    }
    for (uint32_t h = h0; h < h1; h++) {
        const bool is_q = h < a.n_heads;
        const uint32_t hh = is_q ? h : h - a.n_heads;
        const float *x = is_q ? a.q + (size_t)t * a.q_stride : a.k + (size_t)t * a.k_stride;
        float *y = is_q ? a.q_out + (size_t)t * a.q_out_stride : a.k_out + (size_t)t * a.k_out_stride;
        const float *w = is_q ? a.wq : a.wk;
        x += (size_t)hh * a.D;
        y += (size_t)hh * a.D;
        float u[KP][2 * V];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const bool in = (lane + i * W) * V < pairs;
            if (V == 4) {
                const float4 z = make_float4(0, 0, 0, 0);
                const float4 lo = in ? *reinterpret_cast<const float4 *>(x + at[i]) : z;
                const float4 hi = in ? *reinterpret_cast<const float4 *>(x + to[i]) : z;
                u[i][0] = lo.x, u[i][1 % (2 * V)] = lo.y, u[i][2 % (2 * V)] = lo.z, u[i][3 % (2 * V)] = lo.w;
                u[i][4 % (2 * V)] = hi.x, u[i][5 % (2 * V)] = hi.y, u[i][6 % (2 * V)] = hi.z, u[i][7 % (2 * V)] = hi.w;
            } else {
                u[i][0] = in ? x[at[i]] : 0.0f;
                u[i][1] = in ? x[to[i]] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 2 * V; j++) ss += u[i][j] * u[i][j];
        }
        float r = 1.0f;
        if (a.norm) {
#pragma unroll
            for (int off = W / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, W);
            r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
        }
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const bool in = (lane + i * W) * V < pairs;
            if (!in) continue;
            float g[2 * V];
#pragma unroll
            for (int j = 0; j < 2 * V; j++) g[j] = r;
            if (a.norm && w) {
                if (V == 4) {
                    const float4 lo = *reinterpret_cast<const float4 *>(w + at[i]);
                    const float4 hi = *reinterpret_cast<const float4 *>(w + to[i]);
                    const float ww[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int j = 0; j < 2 * V; j++) g[j] *= a.bias + ww[j];
                } else {
                    g[0] *= a.bias + w[at[i]];
                    g[1] *= a.bias + w[to[i]];
                }
            }
#pragma unroll
            for (int j = 0; j < 2 * V; j++) u[i][j] *= g[j];
            float o[2 * V];
            if (a.neox) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    o[j] = u[i][j] * cs[i][j] - u[i][j + V] * sn[i][j];
                    o[j + V] = u[i][j] * sn[i][j] + u[i][j + V] * cs[i][j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    o[2 * j] = u[i][2 * j] * cs[i][j] - u[i][2 * j + 1] * sn[i][j];
                    o[2 * j + 1] = u[i][2 * j] * sn[i][j] + u[i][2 * j + 1] * cs[i][j];
                }
            }
            if (V == 4) {
                *reinterpret_cast<float4 *>(y + at[i]) = make_float4(o[0], o[1 % (2 * V)], o[2 % (2 * V)], o[3 % (2 * V)]);
                *reinterpret_cast<float4 *>(y + to[i]) =
                    make_float4(o[4 % (2 * V)], o[5 % (2 * V)], o[6 % (2 * V)], o[7 % (2 * V)]);
            } else {
                y[at[i]] = o[0];
                y[to[i]] = o[1];
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
    hipLaunchKernelGGL((k_qk_norm_rope<V, W, KP>), dim3((unsigned)((groups + 256 / W - 1) / (256 / W))), dim3(256), 0, s, a);
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
