// lt_mx_matvec.hip -- products of MXFP4 matrices with one vector: matvec, the
// experts' gate/up and down by id (lt_mx_dot.h).
//
// Bound by the weights' bytes (262144 x 2816, 392 MB: 65 us, 6.0 TB/s), and where
// there are few of those by the chain launch - vector - product - sum over the
// waves: 4096 x 4096 4.9 to 5.2 us a graph's node (cards differ), of which an empty
// one has 1.8 and, at 4.9, the loads alone 4.4; 4865 x 896 3.6 to 4.0.  A workgroup converts the vector once, while its
// first weights are on their way.  A tile's rows are split over S waves, 16 blocks
// (a scale word) at a time; what they summed meets in LDS in the waves' order.
#include "llmtoy_hip.h"
#include "lt_internal.h"
#include "lt_mx_dot.h"
#include "lt_topk.h"

namespace lt {

namespace {

constexpr int kMvWaves = 16;  // of a workgroup at most

// Workgroups of S waves a tile (threadIdx.x; and TP tiles side by side, threadIdx.y)
// walk the tiles.  Two items (16 rows by 16 blocks) of a wave are on their way, over the
// tiles' ends, before the vector is converted and from then on.
//
// NV vectors at once, [NV][cols] to [NV][rows] of a matrix: their parts are columns of
// the same instructions, of which there are 16.  1 | 2 | 5 vectors of 4096 x 4096 5.2 |
// 5.4 | 6.6 us a graph's node (limbs and the thin product 9.3), of 262144 x 2816 64 |
// 64 | 69 (limbs and tiles 113), of 11008 x 4096 8.4 | 9.1 | 9.2 (12.8).
template <bool NT, int NV>
__global__ __launch_bounds__(64 * kMvWaves) void k_mx_matvec(const uint8_t *codes, const uint8_t *scales, MxDims d,
                                                             uint32_t ntiles, uint32_t expert_rows, uint32_t S, uint32_t TP,
                                                             const float *x, float *y) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[2][kMvWaves][NV][16];
    const int lane = threadIdx.x & 63;
    const uint32_t sp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tp = __builtin_amdgcn_readfirstlane(threadIdx.y);
    const uint32_t wave = tp * S + sp, threads = 64 * S * TP, tid = 64 * wave + lane, stride = gridDim.x * TP, t0 = blockIdx.x * TP;
    const bool first = p32_first(lane);
    mx_u32x4 *const v = reinterpret_cast<mx_u32x4 *>(lds);
    const uint32_t units = 16 * d.kg;
    MxQuarter xb[NV];
    const size_t cols = (size_t)d.nb * 32;
#pragma unroll
    for (int n = 0; n < NV; n++)
        if (tid < units) xb[n] = mx_vec_load(x + n * cols, tid, d.nb);
    mx_order();

    // every wave of the workgroup goes through the same number of tiles (past
    // the last one: that one again, not written)
    const uint32_t rounds = (ntiles - t0 + stride - 1) / stride, n = rounds * ((d.kq - sp + S - 1) / S);
    uint32_t ft = t0 + tp, fq = sp;  // the next item to fetch
    auto fetch = [&](MxWords &w) {
        const uint32_t tile = min(ft, ntiles - 1);
        const MxRow r{codes + ((size_t)tile * d.kg * 64 + lane) * 16, scales + ((size_t)tile * d.kq * 64 + lane) * 4};
        mx_fetch<NT>(w, r, fq, d.kg);
        if ((fq += S) >= d.kq) fq = sp, ft += stride;
    };
    MxWords w0, w1;
    fetch(w0);
    if (n > 1) fetch(w1);
    mx_order();
#pragma unroll
    for (int n = 0; n < NV; n++) {
        if (tid < units) mx_vec_put<NV>(v, tid, xb[n], n);
        for (uint32_t u = tid + threads; u < units; u += threads) mx_vec_put<NV>(v, u, mx_vec_load(x + n * cols, u, d.nb), n);
    }
    __syncthreads();

    MxSum acc = {};
    uint32_t tile = t0 + tp, q = sp, turn = 0;
    auto use = [&](const MxWords &w) {
        mx_dot<NV>(w, v, q, d.kg, lane, acc);
        if ((q += S) < d.kq) return;
        const uint32_t row0 = tile % d.tiles * 16;
        float *out = y + (size_t)(tile / d.tiles) * expert_rows + row0;
        if constexpr (NV == 1) {
            const float t = mx_rows(acc.all(), lane, first);
            const uint32_t r = 4 * (lane >> 4) + (lane & 3);
            if (S == 1) {
                if ((lane & 15) < 4 && tile < ntiles && row0 + r < expert_rows) out[r] = t;
            } else if ((lane & 15) < 4) {
                part[turn][wave][0][r] = t;
            }
        } else {
            const mx_acc16 t = mx_rows_of(acc.all());
            const uint32_t n = (uint32_t)(lane & 15) / 3, r = 4 * (lane >> 4);
            if ((lane & 15) % 3 == 0 && n < NV) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (S > 1)
                        part[turn][wave][n][r + i] = t[i];
                    else if (tile < ntiles && row0 + r + i < expert_rows)
                        out[(size_t)n * expert_rows + r + i] = t[i];
                }
            }
        }
        if (S > 1) {
            __syncthreads();
            if (sp == 0 && tile < ntiles)
                for (uint32_t e = lane; e < 16 * NV; e += 64) {
                    const uint32_t n = e / 16, r = e % 16;
                    float s = part[turn][wave][n][r];
                    for (uint32_t i = 1; i < S; i++) s += part[turn][wave + i][n][r];
                    if (row0 + r < expert_rows) out[(size_t)n * expert_rows + r] = s;
                }
            turn ^= 1;
        }
        acc = MxSum{};
        q = sp;
        tile += stride;
    };
    for (uint32_t i = 0; i < n; i += 2) {
        use(w0);
        if (i + 2 < n) fetch(w0);
        if (i + 1 < n) {
            use(w1);
            if (i + 3 < n) fetch(w1);
        }
    }
}

// h[slot][j] = act(G x)[j] (U x)[j] of expert ids[slot], zeros from F to
// down_cols: S waves the 16 gate rows, S more the up rows, which may begin
// inside a tile.  G and U are one tensor of 2 F rows an expert, or (ids null)
// two tensors.
//
// ROUTE = PER > 0: the selection is not there yet.  Every wave finds its slot's
// expert in the router's logits (up to 64 PER) itself, and a workgroup of its own
// writes the selection and its weights for the down kernel.  Against the top-k
// in the router's last workgroup, 128 experts of 768 by 2048, top 8: 18.4 -> 16.0
// us a layer.  (One wave that selects for all eight: 6.45 us against 5.75, as the
// others' weights then wait for it.)
//
// 13.4 MB of weights there: 5.4 us with the ids at hand, of which the launch has
// 1.8, the weights at the rate of a copy 2.6.
template <int ROUTE>
__global__ __launch_bounds__(64 * kPairWaves) void k_mx_gate_up(MxPair p, const float *x, const uint32_t *ids, MxRoute route,
                                                                uint32_t n_experts, uint32_t F, uint32_t down_cols,
                                                                uint32_t act, float *h) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kPairWaves][16];
    const int lane = threadIdx.x & 63;
    [[maybe_unused]] const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t j0 = blockIdx.x * 16;
    const MxDims &d = p.d;
    const uint32_t units = 16 * d.kg;
    float logit[ROUTE ? ROUTE : 1];
    if constexpr (ROUTE > 0) {
        if (j0 >= down_cols) {  // the workgroups past the rows: slot 0's writes the selection
            if (blockIdx.y == 0 && wave == 0)
                topk_softmax_wave<ROUTE>(route.logits, (int)n_experts, (int)route.k, (int)route.norm, route.ids, route.w,
                                         nullptr, lane);
            return;
        }
#pragma unroll
        for (int i = 0; i < ROUTE; i++) logit[i] = route.logits[min((uint32_t)lane + 64u * i, n_experts - 1)];
    }
    MxQuarter xb;
    if (threadIdx.x < units) xb = mx_vec_load(x, threadIdx.x, d.nb);
    mx_order();
    uint32_t expert = 0;
    if constexpr (ROUTE > 0)
        expert = (uint32_t)__builtin_amdgcn_readfirstlane(topk_index_at<ROUTE>(logit, (int)n_experts, (int)blockIdx.y, lane));
    else if (ids)
        expert = ids[blockIdx.y];
    float *out = h + (size_t)blockIdx.y * down_cols;
    if (j0 >= F || expert >= n_experts) {  // padding (or no such expert)
        if (threadIdx.x < 16 && j0 + threadIdx.x < down_cols) out[j0 + threadIdx.x] = 0.0f;
        return;
    }
    mx_u32x4 *const v = reinterpret_cast<mx_u32x4 *>(lds);
    mx_gate_rows(
        p, expert, j0, F, down_cols, act, v, part,
        [&] {
            if (threadIdx.x < units) mx_vec_put(v, threadIdx.x, xb);
            for (uint32_t u = threadIdx.x + kPairThreads; u < units; u += kPairThreads)
                mx_vec_put(v, u, mx_vec_load(x, u, d.nb));
            __syncthreads();
        },
        [&](uint32_t i, float y) { out[j0 + i] = y; });
}

// out[i] = sum over slots of w (D_id h[slot])[i]: the waves take the (slot, 16
// blocks) items of a tile's rows in turn, `per` slots' vectors in LDS at once.
// 8 x 2048 x 768 (6.7 MB): 5.7 us, a chain of launch (1.8), ids, weights, sums.  8
// rows a workgroup, twice as many of them: 5.7, and 6.3 -> 10.4 on 4 x 2816 x 2112.
constexpr int kDownWaves = 16;
__global__ __launch_bounds__(64 * kDownWaves) void k_mx_down(const uint8_t *codes, const uint8_t *scales, MxDims d,
                                                             uint32_t rows, uint32_t n_experts, const float *h,
                                                             const uint32_t *ids, const float *wts, uint32_t k,
                                                             uint32_t per, uint32_t NW, MxDiv by_kq, MxDiv by_of,
                                                             const float *base, int accumulate, const float *dscale,
                                                             float *out) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kDownWaves][16];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), threads = 64 * NW;
    const bool first = p32_first(lane);
    const uint32_t row0 = blockIdx.x * 16, vec = (uint32_t)mx_vec_bytes(d.kg), of = 16 * d.kg;
    mx_acc16 sum = {};
    for (uint32_t s0 = 0; s0 < k; s0 += per) {
        const uint32_t n = min(per, k - s0), items = n * d.kq, units = n * of;
        if (s0) __syncthreads();
        auto vec_of = [&](uint32_t i) { return reinterpret_cast<mx_u32x4 *>(lds + i * vec); };
        auto load = [&](uint32_t u) {
            const uint32_t i = by_of.by(u);
            return mx_vec_load(h + (size_t)(s0 + i) * d.nb * 32, u - i * of, d.nb);
        };
        auto put = [&](uint32_t u, const MxQuarter &x) { mx_vec_put(vec_of(0), u, x); };  // (the vectors lie in a row)
        MxQuarter xb;
        if (threadIdx.x < units) xb = load(threadIdx.x);
        mx_order();
        auto fetch = [&](MxWords &w, uint32_t it) {
            const uint32_t i = by_kq.by(it), e = min(ids[s0 + i], n_experts - 1);
            mx_fetch<false>(w, mx_row_at(codes, scales, d, e, row0 + (uint32_t)(lane & 15), lane), it - i * d.kq, d.kg);
        };
        auto use = [&](const MxWords &w, uint32_t it) {
            const uint32_t i = by_kq.by(it), e = ids[s0 + i];
            MxSum t = {};
            mx_dot(w, vec_of(i), it - i * d.kq, d.kg, lane, t);
            if (e < n_experts) sum += t.all() * (dscale ? wts[s0 + i] * dscale[e] : wts[s0 + i]);
        };
        MxWords w0, w1;
        if (wave < items) fetch(w0, wave);
        if (wave + NW < items) fetch(w1, wave + NW);
        mx_order();
        if (threadIdx.x < units) put(threadIdx.x, xb);
        for (uint32_t u = threadIdx.x + threads; u < units; u += threads) put(u, load(u));
        __syncthreads();
        for (uint32_t it = wave; it < items; it += 2 * NW) {
            use(w0, it);
            if (it + 2 * NW < items) fetch(w0, it + 2 * NW);
            if (it + NW < items) use(w1, it + NW);
            if (it + 3 * NW < items) fetch(w1, it + 3 * NW);
        }
    }
    const float t = mx_rows(sum, lane, first);
    if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
    __syncthreads();
    const uint32_t row = row0 + threadIdx.x;
    if (threadIdx.x < 16 && row < rows) {
        float s = part[0][threadIdx.x];
        for (uint32_t i = 1; i < NW; i++) s += part[i][threadIdx.x];
        if (accumulate) s = out[row] + s;
        out[row] = base ? base[row] + s : s;
    }
}

// Parts of this many bytes at most in a down block's LDS (two blocks a CU).
constexpr size_t kDownLds = 72 << 10;

// Waves a tile: as many as it takes to have 4,096 (4 a SIMD), each with the same
// number of items where they can; with few tiles a workgroup each, with many
// 8 waves of several tiles, which walk on.
constexpr size_t kMvTarget = 4096, kMvGroups = 1024;
// Matrices from 8 MiB on are read past the caches: a model of them does not fit
// the 256 MiB there are (262144 x 2816 73 -> 65 us, 4096 x 4096 5.1 -> 4.9).
constexpr size_t kNtBytes = 8u << 20;

}  // namespace

template <int NV>
static hipError_t launch_matvec(const DevTensor &W, const float *x, float *y, hipStream_t s) {
    const MxDims d = mx_dims(W.rows, W.blocks_per_row);
    static bool set[2][64] = {};
    const bool nt = W.bytes >= kNtBytes;
    const auto kernel = nt ? k_mx_matvec<true, NV> : k_mx_matvec<false, NV>;
    hipError_t e = allow_lds((const void *)kernel, set[nt]);
    if (e != hipSuccess) return e;
    const size_t tiles = W.n_experts * d.tiles;
    uint32_t S = (uint32_t)((kMvTarget + tiles - 1) / tiles);
    S = S > (uint32_t)kMvWaves ? (uint32_t)kMvWaves : S;
    S = S > d.kq ? d.kq : S;
    const uint32_t each = (d.kq + S - 1) / S;
    S = (d.kq + each - 1) / each;
    uint32_t TP = tiles * S <= kMvTarget || S > 4 ? 1 : 8 / S;
    size_t most = kMvGroups;
    const size_t lds = NV * mx_vec_bytes(d.kg), fit = (150 << 10) / (lds + sizeof(float) * 2 * kMvWaves * NV * 16);
    // few workgroups a CU: of 16 waves between them, if there are tiles for that (11008
    // x 4096 with 4 vectors 17.5 -> 8.7 us)
    if (NV > 1 && fit < 4) {
        most = 256 * fit;
        const size_t each_gets = (tiles + most - 1) / most;
        TP = (uint32_t)kMvWaves / (uint32_t)fit / S;
        TP = TP < 1 ? 1 : TP > each_gets ? (uint32_t)each_gets : TP;
    }
    const size_t groups = (tiles + TP - 1) / TP;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(groups < most ? groups : most)), dim3(64 * S, TP), lds, s, W.p0, W.p1, d,
                       (uint32_t)tiles, (uint32_t)W.rows, S, TP, x, y);
    return hipGetLastError();
}

hipError_t launch_matvec_mx(const DevTensor &W, const float *x, float *y, hipStream_t s) { return launch_matvec<1>(W, x, y, s); }

// Vectors whose parts fit the LDS together (768 B a vector for 128 columns).  At the edge, 4096
// rows, this | limbs and the thin product for 32 columns more: 2 of 10880 10.2 | 16.3 us, 3 of
// 7168 8.5 | 13.3, 4 of 5376 8.0 | 11.6, 5 of 4352 7.8 | 10.5.
bool matvecs_mx_fit(const DevTensor &W, size_t T) {
    return T <= kMxFew && !W.beyond && T * mx_vec_bytes(mx_dims(W.rows, W.blocks_per_row).kg) <= (128 << 10);
}

hipError_t launch_matvecs_mx(const DevTensor &W, const float *X, size_t T, float *out, hipStream_t s) {
    if (W.n_experts != 1 || !matvecs_mx_fit(W, T)) return hipErrorInvalidValue;
    switch (T) {
    case 1: return launch_matvec<1>(W, X, out, s);
    case 2: return launch_matvec<2>(W, X, out, s);
    case 3: return launch_matvec<3>(W, X, out, s);
    case 4: return launch_matvec<4>(W, X, out, s);
    case 5: return launch_matvec<5>(W, X, out, s);
    default: return hipErrorInvalidValue;
    }
}

template <int ROUTE>
static hipError_t launch_pair(const MxPair &p, const float *x, const uint32_t *ids, const MxRoute &route, uint32_t n_experts,
                              uint32_t k, uint32_t F, uint32_t down_cols, uint32_t act, float *h, hipStream_t s) {
    static bool set[64] = {};
    hipError_t e = allow_lds((const void *)k_mx_gate_up<ROUTE>, set);
    if (e != hipSuccess) return e;
    const dim3 grid((down_cols + 15) / 16 + (ROUTE ? 1 : 0), k);
    hipLaunchKernelGGL(k_mx_gate_up<ROUTE>, grid, dim3(kPairThreads), mx_vec_bytes(p.d.kg), s, p, x, ids, route, n_experts, F,
                       down_cols, act, h);
    return hipGetLastError();
}

hipError_t launch_gate_up_mx(const DevTensor &G, const DevTensor &U, const float *x, uint32_t act, uint32_t down_cols,
                             float *h, hipStream_t s) {
    MxPair p{{G.p0, U.p0}, {G.p1, U.p1}, {0, 0}, mx_dims(G.rows, G.blocks_per_row)};
    return launch_pair<0>(p, x, nullptr, MxRoute{}, 1, 1, (uint32_t)G.rows, down_cols, act, h, s);
}

hipError_t launch_expert_gate_up_mx(const DevTensor &GU, const float *x, const uint32_t *ids, uint32_t k, uint32_t d_expert,
                                    uint32_t down_cols, uint32_t act, float *h, hipStream_t s) {
    MxPair p{{GU.p0, GU.p0}, {GU.p1, GU.p1}, {0, d_expert}, mx_dims(GU.rows, GU.blocks_per_row)};
    return launch_pair<0>(p, x, ids, MxRoute{}, (uint32_t)GU.n_experts, k, d_expert, down_cols, act, h, s);
}

hipError_t launch_expert_gate_up_mx_routed(const DevTensor &GU, const float *x, const float *logits, uint32_t k, uint32_t norm,
                                           uint32_t d_expert, uint32_t down_cols, uint32_t act, float *h, uint32_t *ids_out,
                                           float *w_out, hipStream_t s) {
    MxPair p{{GU.p0, GU.p0}, {GU.p1, GU.p1}, {0, d_expert}, mx_dims(GU.rows, GU.blocks_per_row)};
    const MxRoute route{logits, k, norm, ids_out, w_out};
    const uint32_t n = (uint32_t)GU.n_experts;
    if (n > 256) return hipErrorInvalidValue;
    return n <= 128 ? launch_pair<2>(p, x, nullptr, route, n, k, d_expert, down_cols, act, h, s)
                    : launch_pair<4>(p, x, nullptr, route, n, k, d_expert, down_cols, act, h, s);
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
    const uint32_t items = per * d.kq, NW = items < (uint32_t)kDownWaves ? items : (uint32_t)kDownWaves;
    hipLaunchKernelGGL(k_mx_down, dim3((unsigned)d.tiles), dim3(64 * NW), per * vec, s, D.p0, D.p1, d, (uint32_t)D.rows,
                       (uint32_t)D.n_experts, h, ids, w, k, per, NW, mx_div(d.kq), mx_div(16 * d.kg), base, accumulate, dscale,
                       out);
    return hipGetLastError();
}

}  // namespace lt
