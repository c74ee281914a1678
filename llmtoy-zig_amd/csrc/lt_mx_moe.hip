// lt_mx_moe.hip -- one decode MoE layer with MXFP4 experts (batch 1) in a single
// launch: the router's logits and selection (ops/moe.zig:44-52), the selected
// experts' gate/up (55-66) and down with the weighted sum (67-76).
//
// Workgroup b runs on XCD b % 8 (its "group"; probed by the context), and slot s of
// the selected experts is group s % 8's alone, so that h goes through one L2.  By the
// index i = b / 8 inside the group:
//
//   i < NR          4 logits in dotf32's order, published in 8 copies
//   next SPG J      16 rows of h of slot x + 8 u: waits for the logits
//   next SPG ND     64 output rows of the slot: waits for the logits, has its first
//                   weights on the way, waits for h; publishes the weighted rows.  The
//                   last slot's adds those of all slots, in their order, to out.
//
// What is handed over are words of a value and the launch's epoch (lt_internal.h):
// h with stores that stay in the group's L2 where the probe found it (0.2 us, past it
// 0.6 and more), all else past the L2s.  A workgroup waits only for ones of lower
// index, and workgroups start in that order, so every wait ends; a limit on the clock
// ends it too (NaN, and the error word).  The epoch is each workgroup's own count of
// its launches: the memory belongs to one shape, whose grid is always the same.
// (Two such launches at once, from two contexts, could each fill an XCD that the
// other's first workgroups need, and end at the limit with the error: one context a
// device at a time.)
//
// Bound by a chain of latencies.  128 experts of 768 by 2048, top 8, us from the
// start: logits made 2.0 and seen 3.2, experts known 3.5-4.5 (a round of the selection
// 0.13), h made 7, read 8, rows published 9, summed 10.5.  us a token in a graph, this |
// three launches: 13.0 | 14.5, top 6 12.5 | 13.7, top 16 18.4 | 20.6; 128 of 704 by 2816,
// top 8, 15.4 | 16.5; 32 of 2112 by 2816, top 8, 25.0 | 28.1; 64 of 512 by 1024, top 8,
// 10.9 | 12.9; 60 of 1408 by 2048, top 8, 16.9 | 17.4.
//
// A slot has one XCD's share of the memory's rate, so slots that leave XCDs without
// one cost: top 4 of 32 of 2112 by 2816 22.9 | 19.0, top 10 of 128 of 768 by 2048 16.6 |
// 15.5; and with more workgroups than are there at once fewer idle ones do: top 6 of 8
// of 1024 by 2400 17.1 | 15.4, top 8 18.3 | 17.5 (8 of 2048 by 1024 16.7 | 19.5).  So it
// is taken where no XCD of a turn is idle, or at most two and all are there at once, or
// the slots are small: 64 of 512 by 1024 (0.8 MB a slot) top 1 8.3 | 10.2, top 4 10.0 |
// 10.9, top 9 11.1 | 13.4; 60 of 320 by 2048 (1.04 MB) top 4 10.7 | 11.4, but top 9 13.4 |
// 12.8.  h past the L2s instead, as it is without the placement: 12.9 -> 14.4 us.  Three
// workgroups a CU: 13.2 us, two 15.0.
#include "llmtoy_hip.h"
#include "lt_dotf32.h"
#include "lt_internal.h"
#include "lt_mx_dot.h"
#include "lt_topk.h"

#include <math.h>

namespace lt {

namespace {

constexpr uint32_t kMxMaxLogits = 256, kMxDownRows = 64;
constexpr uint32_t kMxAtOnce = 96;  // workgroups of a group on its 32 CUs
struct MxLayer {
    const float *router, *bias, *x, *base;
    MxPair gu;
    const uint8_t *codes, *scales;  // down
    MxDims d;
    MxRoute route;
    uint32_t n_experts, F, down_cols, rows, act;
    uint32_t NR, J, ND, SPG;
    MxDiv by_j, by_nd;
    int accumulate, local;
    uint32_t wait;  // the waits' limit, up to kMxWaitTicks
    float *out;
    uint32_t *counters, *err;
    uint64_t *lg;  // [8][kMxMaxLogits]
    uint64_t *hl;  // [slot][element of a lane's eight][quarter of a block]
    uint64_t *pl;  // [slot][row]
};

// Waits until every lane's words (up to N, `have` of them from its pointer p on,
// stride apart) carry the epoch; the others are 0.  False after the limit.
template <int N>
__device__ __forceinline__ bool mx_await(const uint64_t *p, uint32_t stride, uint32_t have, uint32_t ep, uint64_t t0, float (&v)[N]) {
    while (true) {
        uint64_t w[N];
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = (uint32_t)i < have ? hand_get(p + i * stride) : (uint64_t)ep << 32;
        bool good = true;
#pragma unroll
        for (int i = 0; i < N; i++) good = good && tag_is(w[i], ep);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = good ? __uint_as_float((uint32_t)w[i]) : NAN;
        if (__all(good)) return true;
        if (wall_clock64() - t0 > kMxWaitTicks) return false;
    }
}
// What a wait that ran out was for, in the error word (each bit's meaning stands in its text).
enum : uint32_t { kMxGateLogits = 1, kMxDownLogits = 2, kMxH = 4, kMxRows = 8 };
// (Which word was late, and its tag, are not recorded: every form of that cost 0.2 to 0.3
// us a layer where nothing is late.)
__device__ __forceinline__ void mx_late(const MxLayer &a, uint32_t what, uint32_t ep, int lane) {
    if (lane) return;
    report_timeout(a.err, what);
    report_detail(a.err, (int)blockIdx.x, what, kErrNotRecorded, kErrNotRecorded, ep);
}

// One wave: logit lane + 64 i in v[i], from the group's copy.  Late ones make all of them
// NaN (those that came in time might select another expert), and so the weights.
template <int PER>
__device__ __forceinline__ bool mx_logits(const MxLayer &a, uint32_t what, uint32_t ep, uint64_t t0, float (&v)[PER], int lane) {
    const uint64_t *w = a.lg + (blockIdx.x & 7) * kMxMaxLogits;
    float one[1];
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = 0.0f;
    const bool good = mx_await<1>(w + (blockIdx.x >> 3) % a.n_experts, 0, lane == 0, ep, t0, one) &&  // then all of them
                      mx_await<PER>(w + lane, 64, (a.n_experts + 63u - lane) / 64, ep, t0, v);
    if (__builtin_expect(!good, 0)) {
        mx_late(a, what, ep, lane);
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = NAN;
    }
    return good;
}

template <int ROUTE>
__global__ __launch_bounds__(kPairThreads, 6) void k_mx_moe(MxLayer a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float part[kPairWaves][16];
    __shared__ uint32_t s_ids[16], s_good;
    __shared__ float s_w[16];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.x, group = b % 8;
    mx_u32x4 *const v = reinterpret_cast<mx_u32x4 *>(lds);
    const uint32_t ep = a.counters[b] + 1u;
    const uint64_t t0 = wall_clock64() - (kMxWaitTicks - a.wait);  // (where kMxWaitTicks before the limit is)
    uint32_t i = b / 8;
    // (behind a barrier: every wave has read the count)
    auto done = [&] {
        if (threadIdx.x == 0) a.counters[b] = ep;
    };
    if (i < a.NR) {
        const uint32_t row = 4 * b + wave / 2, at = min(row, a.n_experts - 1);
        const float y = dotf32_pair_any<true>(a.router + (size_t)at * a.gu.d.nb * 32, a.x, a.bias ? a.bias + at : nullptr, (int)a.gu.d.nb,
                                    (int)(wave & 1), lane, reinterpret_cast<float *>(lds) + wave * 512, part[wave / 2]);
        if ((wave & 1) == 0 && lane < 8 && row < a.n_experts)
            hand_put(a.lg + lane * kMxMaxLogits + row, __float_as_uint(y), ep);
        return done();
    }
    i -= a.NR;
    if (i < a.SPG * a.J) {
        const uint32_t u = a.by_j.by(i), slot = group + 8 * u, j0 = (i - u * a.J) * 16, at = j0 / 32;
        // elements j0 + r of the slot's h: quarter 4 at + r / 4 of them, j0 % 32 / 8 + r % 4 of its eight
        uint64_t *const to = a.hl + ((size_t)slot * 8 + j0 % 32 / 4) * (4 * a.d.nb) + 4 * at;
        auto put = [&](uint32_t r, float y) {
            hand_put_group(to + r % 4 * (4 * a.d.nb) + r / 4, __float_as_uint(y), ep, a.local);
        };
        if (slot >= a.route.k || j0 >= a.F) {
            if (slot < a.route.k && threadIdx.x < 16) put(threadIdx.x, 0.0f);
            __syncthreads();
            return done();
        }
        const uint32_t units = 16 * a.gu.d.kg;
        for (uint32_t q = threadIdx.x; q < units; q += kPairThreads) mx_vec_put(v, q, mx_vec_load(a.x, q, a.gu.d.nb));
        if (wave == 0) {
            float logit[ROUTE];
            const bool good = mx_logits<ROUTE>(a, kMxGateLogits, ep, t0, logit, lane);
            const int e = topk_index_at<ROUTE>(logit, (int)a.n_experts, (int)slot, lane);
            if (lane == 0) s_ids[0] = (uint32_t)e, s_good = good;
        }
        __syncthreads();
        mx_gate_rows(
            a.gu, (uint32_t)__builtin_amdgcn_readfirstlane(s_ids[0]), j0, a.F, a.down_cols, a.act, v, part, [] {},
            [&](uint32_t r, float y) { put(r, s_good ? y : NAN); });
        return done();
    }
    i -= a.SPG * a.J;
    const uint32_t u = a.by_nd.by(i), slot = group + 8 * u, row0 = (i - u * a.ND) * kMxDownRows;
    if (slot >= a.route.k) {
        __syncthreads();
        return done();
    }
    if (wave == 0) {
        float logit[ROUTE];
        const bool good = mx_logits<ROUTE>(a, kMxDownLogits, ep, t0, logit, lane);
        uint32_t key[ROUTE];
        int e;
        float w;
        topk_softmax_regs<ROUTE>(logit, (int)a.n_experts, (int)a.route.k, (int)a.route.norm, s_ids, s_w, key, e, w, lane);
        if (lane == 0) s_good = good;
    }
    __syncthreads();
    const bool last = slot == a.route.k - 1;
    if (last && row0 == 0 && threadIdx.x < a.route.k) {
        a.route.ids[threadIdx.x] = s_good ? s_ids[threadIdx.x] : 0u;
        a.route.w[threadIdx.x] = s_good ? s_w[threadIdx.x] : NAN;
    }
    // a tile of 16 rows to two waves, 512 columns in turn
    const uint32_t tile = min(row0 / 16 + wave / 2, (uint32_t)a.d.tiles - 1), half = wave & 1;
    const MxRow rw = mx_row_at(a.codes, a.scales, a.d, (uint32_t)__builtin_amdgcn_readfirstlane(s_ids[slot]), 16 * tile + (lane & 15),
                               lane);
    MxWords w0;
    if (half < a.d.kq) mx_fetch<false>(w0, rw, half, a.d.kg);
    mx_order();
    uint32_t late = 0;
    for (uint32_t q = threadIdx.x; __any(q < 16 * a.d.kg); q += kPairThreads) {
        float y[8];
        const bool on = q < 4 * a.d.nb;
        if (!mx_await<8>(a.hl + (size_t)slot * 8 * (4 * a.d.nb) + q, 4 * a.d.nb, on ? 8 : 0, ep, t0, y)) late |= kMxH;
        if (q < 16 * a.d.kg)
            mx_vec_put(v, q, {make_float4(y[0], y[1], y[2], y[3]), make_float4(y[4], y[5], y[6], y[7])});
    }
    __syncthreads();
    MxSum acc = {};
    for (uint32_t q = half; q < a.d.kq; q += 2) {
        mx_dot(w0, v, q, a.d.kg, lane, acc);
        if (q + 2 < a.d.kq) mx_fetch<false>(w0, rw, q + 2, a.d.kg);
    }
    const float t = mx_rows(acc.all(), lane, p32_first(lane));
    if ((lane & 15) < 4) part[wave][4 * (lane >> 4) + (lane & 3)] = t;
    __syncthreads();
    float *const sums = reinterpret_cast<float *>(lds);  // [slot][row]
    if (threadIdx.x < kMxDownRows) {
        const uint32_t r = threadIdx.x, row = row0 + r;
        const float y = (part[r / 16 * 2][r % 16] + part[r / 16 * 2 + 1][r % 16]) * s_w[slot];
        if (last)
            sums[slot * kMxDownRows + r] = y;
        else if (row < a.rows)
            hand_put(a.pl + (size_t)slot * a.rows + row, __float_as_uint(y), ep);
    }
    if (last) {
        for (uint32_t q = threadIdx.x; __any(q < slot * kMxDownRows); q += kPairThreads) {
            const uint32_t row = row0 + q % kMxDownRows;
            const bool mine = q < slot * kMxDownRows, on = mine && row < a.rows;
            float y[1];
            if (!mx_await<1>(a.pl + (size_t)(q / kMxDownRows) * a.rows + row, 0, on, ep, t0, y)) late |= kMxRows;
            if (mine) sums[q] = y[0];
        }
        __syncthreads();
        const uint32_t row = row0 + threadIdx.x;
        if (threadIdx.x < kMxDownRows && row < a.rows) {
            float y = sums[threadIdx.x];
            for (uint32_t q = 1; q <= slot; q++) y += sums[q * kMxDownRows + threadIdx.x];
            if (a.accumulate) y = a.out[row] + y;
            a.out[row] = a.base ? a.base[row] + y : y;
        }
    }
    if (__builtin_expect(late != 0, 0)) mx_late(a, late, ep, lane);
    done();
}

constexpr size_t kMxLgBytes = 8 * kMxMaxLogits * 8;
// Workgroups of a group.
uint32_t layer_groups(uint32_t n_experts, uint32_t k, size_t d_model, size_t down_cols, uint32_t &NR, uint32_t &J, uint32_t &ND,
                             uint32_t &SPG) {
    NR = ((n_experts + 3) / 4 + 7) / 8, J = (uint32_t)(down_cols / 16), ND = (uint32_t)((d_model + kMxDownRows - 1) / kMxDownRows);
    SPG = (k + 7) / 8;
    return NR + SPG * (J + ND);
}

}  // namespace

bool moe_mx_fits(const DevTensor &R, const DevTensor &GU, const DevTensor &D, uint32_t k) {
    uint32_t NR, J, ND, SPG;
    const uint32_t n = (uint32_t)GU.n_experts, idle = (k + 7) / 8 * 8 - k;
    return GU.type == LT_TYPE_MXFP4 && D.type == LT_TYPE_MXFP4 && R.type == LT_TYPE_F32 &&
           GU.n_experts <= kMxMaxLogits && k >= 1 && k <= 16 &&
           (idle == 0 || (idle <= 2 && layer_groups(n, k, D.rows, D.cols, NR, J, ND, SPG) <= kMxAtOnce) ||
            (GU.bytes + D.bytes) / n <= (k <= 8 ? 1u << 20 : 7u << 17));
}

size_t moe_mx_bytes(uint32_t n_experts, uint32_t k, size_t d_model, size_t down_cols) {
    uint32_t NR, J, ND, SPG;
    const size_t blocks = 8 * (size_t)layer_groups(n_experts, k, d_model, down_cols, NR, J, ND, SPG);
    return kMxLgBytes + k * (down_cols + d_model) * 8 + blocks * 4;
}

hipError_t launch_moe_mx(const DevTensor &R, const float *bias, const DevTensor &GU, const DevTensor &D, const float *x, uint32_t k,
                         uint32_t norm, uint32_t d_expert, uint32_t act, const float *base, int accumulate, float *out,
                         uint32_t *ids, float *w, uint8_t *hand, int xcd_local, uint32_t wait, uint32_t *err, hipStream_t s) {
    MxLayer a{};
    const uint32_t n = (uint32_t)GU.n_experts;
    if (!moe_mx_fits(R, GU, D, k) || R.total_rows != n) return hipErrorInvalidValue;
    a.router = (const float *)R.p0, a.bias = bias, a.x = x, a.base = base;
    a.gu = MxPair{{GU.p0, GU.p0}, {GU.p1, GU.p1}, {0, d_expert}, mx_dims(GU.rows, GU.blocks_per_row)};
    a.codes = D.p0, a.scales = D.p1, a.d = mx_dims(D.rows, D.blocks_per_row);
    a.route = MxRoute{nullptr, k, norm, ids, w};
    a.n_experts = n, a.F = d_expert, a.down_cols = (uint32_t)D.cols, a.rows = (uint32_t)D.rows, a.act = act;
    const unsigned grid = 8 * layer_groups(n, k, D.rows, D.cols, a.NR, a.J, a.ND, a.SPG);
    a.by_j = mx_div(a.J), a.by_nd = mx_div(a.ND);
    a.accumulate = accumulate, a.local = xcd_local, a.wait = wait, a.out = out, a.err = err;
    a.lg = reinterpret_cast<uint64_t *>(hand);
    a.hl = reinterpret_cast<uint64_t *>(hand + kMxLgBytes);
    a.pl = a.hl + (size_t)k * D.cols;
    a.counters = reinterpret_cast<uint32_t *>(a.pl + (size_t)k * D.rows);
    static bool set[2][64] = {};
    const bool wide = n > 128;
    const auto kernel = wide ? k_mx_moe<4> : k_mx_moe<2>;
    hipError_t e = allow_lds((const void *)kernel, set[wide]);
    if (e != hipSuccess) return e;
    size_t need = kPairWaves * 512 * 4;  // the router's products, and the slots' rows
    if (mx_vec_bytes(a.gu.d.kg) > need) need = mx_vec_bytes(a.gu.d.kg);
    if (mx_vec_bytes(a.d.kg) > need) need = mx_vec_bytes(a.d.kg);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kPairThreads), need, s, a);
    return hipGetLastError();
}

}  // namespace lt
