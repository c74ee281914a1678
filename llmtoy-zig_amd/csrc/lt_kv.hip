// lt_kv.hip -- block tables and slot maps from request lengths, and tokens into
// and out of the 8-bit cache (layout: lt_kv.h).
#include "llmtoy_hip.h"
#include "lt_kv.h"

namespace lt {

namespace {

// ------------------------------------------------------------------- the plan
// With total = len + n_new of a row, it needs blocks for the indices
// ceil(len / 32) .. ceil(total / 32) - 1; the rows take them from the free list in
// order, and their tokens lie in the batch in order.  A row whose table has no room for them
// takes none.  Both are prefix sums over
// the rows, which one workgroup takes (kPlanRows a thread); new blocks and
// tokens then look their row up in the sums.  Bound by its chain of latencies:
// the lengths, the sums, the table's entry, the slot (8 rows 5.1 us; 2,000 rows 6.1, and the
// maps of 65,536 tokens 6.5 behind it).
constexpr uint32_t kPlanThreads = 1024, kPlanRows = kKvMaxSeqs / kPlanThreads;
// Tokens of a batch that the one workgroup maps; more go to a grid of their own
// behind it (k_kv_slots).
constexpr uint32_t kPlanTokens = 2048;

// Blocks that a row takes from the list: none where its table has no room; where even the
// length passes 32 bits, more than any list has, so that none is handed out behind it.
constexpr uint64_t kBeyondAny = 1ull << 40;
__device__ __forceinline__ uint64_t plan_need(uint32_t len, uint32_t add, uint32_t max_blocks) {
    const uint64_t total = (uint64_t)len + add;
    if (total >> 32) return kBeyondAny;
    const uint64_t b0 = ((uint64_t)len + kKvBlock - 1) / kKvBlock, b1 = (total + kKvBlock - 1) / kKvBlock;
    return b1 <= max_blocks ? b1 - b0 : 0;
}

__device__ __forceinline__ uint32_t sat32(uint64_t v) { return v < kKvNone ? (uint32_t)v : kKvNone; }

// The last row whose sum in first[0 .. n - 1] is <= u (first[0] = 0).
__device__ __forceinline__ uint32_t plan_row(const uint32_t *first, uint32_t n, uint32_t u) {
    uint32_t lo = 0, hi = n;  // first[lo] <= u < first[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ uint32_t plan_slot(const KvPlanArgs &a, uint32_t row, uint32_t pos) {
    const uint32_t j = pos / kKvBlock;
    const uint32_t b = j < a.max_blocks ? a.table[(size_t)row * a.max_blocks + j] : kKvNone;
    return b < kKvNone / kKvBlock ? b * kKvBlock + pos % kKvBlock : kKvNone;
}

__global__ __launch_bounds__(kPlanThreads) void k_kv_plan(KvPlanArgs a) {
    __shared__ uint32_t s_first[kKvMaxSeqs], s_need[kKvMaxSeqs], s_block[kKvMaxSeqs], s_pos[kKvMaxSeqs];
    __shared__ uint64_t s_wave[2][kPlanThreads / kWave];
    __shared__ uint32_t s_used;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const uint32_t used = a.used_in[0];
    uint32_t len[kPlanRows], add[kPlanRows];
    uint64_t take[kPlanRows], tok = 0, need = 0;
    for (uint32_t i = 0; i < kPlanRows; i++) {
        const uint32_t r = tid * kPlanRows + i;
        len[i] = r < a.n_seqs ? a.len_in[r] : 0;
        add[i] = r < a.n_seqs ? a.n_new[r] : 0;
        tok += add[i];
        take[i] = plan_need(len[i], add[i], a.max_blocks);
        need += take[i];
    }
    // sums before this thread's rows
    uint64_t itok = tok, ineed = need;
    for (int off = 1; off < kWave; off <<= 1) {
        const uint64_t p = __shfl_up(itok, off, kWave), q = __shfl_up(ineed, off, kWave);
        if ((int)lane >= off) itok += p, ineed += q;
    }
    if (lane == kWave - 1) s_wave[0][wave] = itok, s_wave[1][wave] = ineed;
    if (tid == 0) s_used = used;
    __syncthreads();  // (every length is read: len and len_in may be one array, so may used and used_in)
    // (the wavefronts' sums, a lane each: those before this one's, and all)
    static_assert(kPlanThreads / kWave == 16, "");
    uint64_t before[2], sum[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint64_t mine = s_wave[k][lane % 16];
        uint64_t up = lane % 16 < wave ? mine : 0, every = mine;
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) up += __shfl_xor(up, off, kWave), every += __shfl_xor(every, off, kWave);
        before[k] = up, sum[k] = every;
    }
    uint64_t btok = itok - tok + before[0], bneed = ineed - need + before[1];
    const uint64_t all = sum[0], fresh = sum[1];
    uint32_t most = used;
    for (uint32_t i = 0; i < kPlanRows; i++) {
        const uint32_t r = tid * kPlanRows + i;
        const uint64_t total = (uint64_t)len[i] + add[i];
        const uint64_t b0 = ((uint64_t)len[i] + kKvBlock - 1) / kKvBlock, b1 = (total + kKvBlock - 1) / kKvBlock;
        if (r < a.n_seqs) {
            a.start[r] = sat32(btok);
            a.len[r] = sat32(total);
            s_first[r] = sat32(btok);
            s_pos[r] = len[i];
            s_need[r] = sat32(bneed);
            const bool room = b1 <= a.max_blocks && !(total >> 32), served = room && used + bneed + (b1 - b0) <= a.n_free;
            s_block[r] = served ? (uint32_t)b0 : kKvNone;
            if (served) most = max(most, (uint32_t)(used + bneed + (b1 - b0)));
            else if (b1 > b0 || (!room && add[i])) kv_report(a.err, kKvErrPool, r);
            if (!served)  // (its new entries: nothing; the entries of a served row are written below)
                for (uint64_t j = b0; j < b1 && j < a.max_blocks; j++) a.table[(size_t)r * a.max_blocks + j] = kKvNone;
        }
        btok += add[i];
        bneed += take[i];
    }
    // (a wavefront's largest first: 1,024 atomics on one word took 3 us)
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) most = max(most, (uint32_t)__shfl_xor(most, off, kWave));
    if (lane == 0) atomicMax(&s_used, most);
    __syncthreads();
    if (tid == 0) {
        a.start[a.n_seqs] = sat32(all);
        a.used[0] = s_used;
        if (all > a.n_tokens) kv_report(a.err, kKvErrRoom, a.n_seqs - 1);
    }
    const uint64_t left = used < a.n_free ? a.n_free - used : 0;  // (blocks beyond the list are nobody's)
    const uint32_t blocks = (uint32_t)(fresh < left ? fresh : left);
    for (uint32_t k = tid; k < blocks; k += kPlanThreads) {
        const uint32_t r = plan_row(s_need, a.n_seqs, k), b0 = s_block[r];
        if (b0 != kKvNone) a.table[(size_t)r * a.max_blocks + b0 + (k - s_need[r])] = a.free_blocks[used + k];
    }
    if (a.n_tokens > kPlanTokens) return;
    // (a new block's number from the list, not from the table, which is being written)
    const uint32_t end = (uint32_t)(all < a.n_tokens ? all : a.n_tokens);
    for (uint32_t t = tid; t < a.n_tokens; t += kPlanThreads) {
        uint64_t pos = 0;
        uint32_t slot = kKvNone;
        if (t < end) {
            const uint32_t r = plan_row(s_first, a.n_seqs, t);
            pos = (uint64_t)s_pos[r] + (t - s_first[r]);
            const uint64_t j = pos / kKvBlock, first_new = ((uint64_t)s_pos[r] + kKvBlock - 1) / kKvBlock;
            uint32_t block = kKvNone;
            if (j >= first_new) {
                if (s_block[r] != kKvNone) block = a.free_blocks[used + s_need[r] + (uint32_t)(j - first_new)];
            } else if (j < a.max_blocks) {
                block = a.table[(size_t)r * a.max_blocks + j];
            }
            if (block < kKvNone / kKvBlock) slot = block * kKvBlock + (uint32_t)pos % kKvBlock;
        }
        a.pos[t] = (uint32_t)pos;
        a.slot[t] = slot;
    }
}

// The maps of a large batch.  A workgroup's tokens begin in the row that its
// first wavefront finds and mostly end there; each thread goes on from it.
__global__ __launch_bounds__(256) void k_kv_slots(KvPlanArgs a) {
    const uint32_t t0 = blockIdx.x * 256, t = t0 + threadIdx.x;
    uint32_t r = kv_row(a.n_seqs, t0, [&](uint32_t i) { return a.start[i]; });
    if (t >= a.n_tokens) return;
    uint32_t pos = 0, slot = kKvNone;
    const uint32_t all = a.start[a.n_seqs];
    if (t < all) {
        uint32_t next = a.start[r + 1];
        while (next <= t) next = a.start[++r + 1];  // (t < all: ends at the last row)
        pos = a.len[r] - (next - t);
        slot = plan_slot(a, r, pos);
    }
    a.pos[t] = pos;
    a.slot[t] = slot;
}

// ------------------------------------------------------------------- appending
// A (sequence, block) that the batch touches is one unit; unit u belongs to the
// last row with first / 32 + 2 r <= u, which leaves every row as many units as
// its tokens can touch blocks.
__host__ __device__ __forceinline__ uint32_t append_units(uint32_t n_tokens, uint32_t n_seqs) {
    return n_tokens / kKvBlock + 2 * n_seqs;
}

// The row that unit u belongs to, by a whole wavefront: up to 64 rows from one round of
// loads, more in three.  (row.falls: or behind)
__device__ __forceinline__ uint32_t append_row(const KvBatchDev &b, uint32_t u, KvRow &row) {
    const auto base = [&](uint32_t start, uint32_t i) { return (start < b.n_tokens ? start : b.n_tokens) / kKvBlock + 2 * i; };
    uint32_t r;
    if (b.n_seqs <= kWave) {
        const uint32_t lane = threadIdx.x % kWave, i = lane < b.n_seqs ? lane : b.n_seqs - 1;
        const KvRow k = kv_row_of(b, i);
        const uint64_t below = __ballot(lane < b.n_seqs && base(b.start[i], i) <= u);
        r = below ? 63 - __builtin_clzll(below) : 0;
        row.first = __builtin_amdgcn_readlane(k.first, r), row.n = __builtin_amdgcn_readlane(k.n, r);
        row.len = __builtin_amdgcn_readlane(k.len, r);
        row.bad = __builtin_amdgcn_readlane(k.bad, r), row.falls = __builtin_amdgcn_readlane(k.falls || k.behind, r);
    } else {
        r = __builtin_amdgcn_readfirstlane(kv_row(b.n_seqs, u, [&](uint32_t i) { return base(b.start[i], i); }));
        const KvRow k = kv_row_of(b, r);
        row.first = __builtin_amdgcn_readfirstlane(k.first), row.n = __builtin_amdgcn_readfirstlane(k.n);
        row.len = __builtin_amdgcn_readfirstlane(k.len);
        row.bad = __builtin_amdgcn_readfirstlane(k.bad), row.falls = __builtin_amdgcn_readfirstlane(k.falls || k.behind);
    }
    return r;  // (in scalar registers, as what follows from it)
}

// round(x / s), ties to even, |x| <= 127.5 s: the product with 1 / s is at most
// one code off, and what remains of x beside code * s is exact.
__device__ __forceinline__ float kv_code(float x, float s, float inv) {
    float q = rintf(x * inv);
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    const float r = fmaf(-q, s, x), h = 0.5f * s;
    const float odd = fabsf(q) - 2.0f * floorf(0.5f * fabsf(q));  // 1 or 0
    const float up = fabsf(r) > h ? 1.0f : fabsf(r) == h ? odd : 0.0f;
    q += r < 0.0f ? -up : up;
    return fminf(fmaxf(q, -127.0f), 127.0f);
}

// The codes + 128 of 16 values, s > 0 their block's scale (or 0: all 0).  Off a border between two
// codes the product with 1 / s, off by 2^-16 at most, rounds as the quotient does; where one of a
// wavefront's values is nearer to one (1 in 25,000 is), all are taken by kv_code.
__device__ __forceinline__ uint4 kv_codes16(const float (&x)[16], float s) {
    // (next to the subnormal numbers the remainders of kv_code would not be exact: scaled up by 2^100 they are)
    const float up = s < 0x1p-100f ? 0x1p100f : 1.0f;
    const float su = s * up, inv = s > 0.0f ? 1.0f / su : 0.0f;
    float q[16], near = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float y = x[e] * up * inv;
        q[e] = rintf(y);
        near = fmaxf(near, fabsf(y - q[e]));
    }
    if (__any(near > 0.49998f) || up != 1.0f) {  // (a subnormal scale may be too small by a half: kv_code's bounds)
#pragma unroll
        for (int e = 0; e < 16; e++) q[e] = s > 0.0f ? kv_code(x[e] * up, su, inv) : 0.0f;
    }
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = 0;
#pragma unroll
        for (int f = 0; f < 4; f++) w[e] = __builtin_amdgcn_cvt_pk_u8_f32(q[4 * e + f] + 128.0f, f, w[e]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ size_t open_at(const KvDev &kv, uint32_t seq, uint32_t h, uint32_t which, uint32_t block) {
    return ((((size_t)seq * kv.n_kv + h) * 2 + which) * 2 + (block & 1)) * kKvBlock * kv.D;
}

// Block `page` is begun anew by row r: the tags of the row that had it last (former; 0: none) forget it, but for
// those that this launch writes (parity `own` of row r; 2: none).  Where another workgroup of the launch writes
// such a tag, whichever comes first, its own value stays.
__device__ __forceinline__ void forget(const KvDev &kv, uint32_t page, uint32_t former, uint32_t r, uint32_t own, uint32_t threads) {
    if (threadIdx.x == 0 && former != r + 1) kv.owner[page] = r + 1;
    if (former == 0 || former > kv.n_seqs) return;
    uint2 *tags = kv.tags + (size_t)(former - 1) * kv.n_kv * 4;
    for (uint32_t i = threadIdx.x; i < kv.n_kv * 4; i += threads) {
        const uint2 t = tags[i];
        if (t.x != page || t.y == 0 || (former - 1 == r && i % 2 == own)) continue;
        unsigned long long was = t.x | (unsigned long long)t.y << 32;
        (void)__hip_atomic_compare_exchange_strong(reinterpret_cast<unsigned long long *>(tags + i), &was, (unsigned long long)page,
                                                   __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// Grid: units, heads, keys or values.  A workgroup takes the block's tokens into
// registers as the layout's pieces (16 elements a thread: two runs of
// eight channels for keys, two of eight tokens for values), finds the largest,
// and writes the codes.
// Bound by the reads of the new tokens; a single token by its chain of
// latencies: the lengths, then the table, the tag and the tokens, the largest, the codes.
// 4,103 tokens of 8 heads of 128 12.5 us (42 MB; at a copy's rate 8.1: the values' loads are of 4 bytes, 16 a thread),
// 512 5.5; one token each of 16 sequences 6 us.  (Keys
// and values by one workgroup: slower by a third.  A code for keys and one for values: 16.5 -> 13.1 us.)
template <int D, int which>
__device__ __forceinline__ void append_unit(const KvDev &kv, const KvBatchDev &b, const float *kv_src, size_t stride, uint32_t *err) {
    constexpr int kWaves = 2 * D / kWave;
    const uint32_t h = blockIdx.y, tid = threadIdx.x;
    const uint32_t lane = tid % kWave, c = tid / kWave, g = lane / 16, n = lane % 16;
    KvRow row;
    const uint32_t r = append_row(b, blockIdx.x, row);
    if (row.n == 0) {
        if (row.falls && tid == 0) kv_report(err, kKvErrRows, r);
        return;
    }
    if (row.bad || r >= kv.n_seqs) {
        if (tid == 0) kv_report(err, kKvErrRows, r);
        return;
    }
    const uint32_t begin = row.len - row.n, first = begin / kKvBlock, last = (row.len - 1) / kKvBlock;
    const uint32_t j = blockIdx.x - (row.first / kKvBlock + 2 * r) + first;
    if (j < first || j > last) return;  // (more units than blocks; start that falls)
    const uint32_t page = b.table[(size_t)r * b.max_blocks + j];  // (looked at behind the loads of the tokens)
    const uint32_t base = j * kKvBlock;                           // position of the block's first token
    const uint32_t from = begin > base ? begin - base : 0;        // its first token in the batch
    const uint32_t held = row.len - base < kKvBlock ? row.len - base : kKvBlock;
    uint2 *tag = kv.tags + (((size_t)r * kv.n_kv + h) * 2 + which) * 2;
    const uint2 held_tag = tag[j & 1];
    const float *src = kv_src + (size_t)row.first * stride + (size_t)h * D;  // token i of the row at i * stride
    const float *open = kv.open + open_at(kv, r, h, which, j);
    float x[16];
    // The thread's piece, token t + more from at(t, more); tokens that nobody has are cleared.
    const auto piece = [&](auto at, uint32_t n_held) {
        if (which == 0) {
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const float4 *row4 = reinterpret_cast<const float4 *>(at(n, 16 * hi) + 32 * c + 8 * g);
                const float4 u = row4[0], w = row4[1];
                const float e8[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int f = 0; f < 8; f++) x[8 * hi + f] = n + 16 * hi < n_held ? e8[f] : 0.0f;
            }
        } else {
#pragma unroll
            for (int f = 0; f < 8; f++) {
                const int more = f % 4 + 16 * (f / 4);
                const float *row1 = at(4 * g, more) + 32 * c + n;
                const float lo = row1[0], hi = row1[16];
                x[f] = 4 * g + more < n_held ? lo : 0.0f;
                x[8 + f] = 4 * g + more < n_held ? hi : 0.0f;
            }
        }
    };
    // (a block that the batch fills: one stride between its tokens, no look at any)
    if (from == 0 && held == kKvBlock) {
        const float *block = src + (size_t)(base - begin) * stride;
        piece([&](uint32_t t, int more) { return block + t * stride + more * stride; }, kKvBlock);
    } else {
        // the tokens from before lie in the open block, the batch's in src; none: the last of those
        piece([&](uint32_t t, int more) -> const float * {
            t += more;
            return t < from ? open + (size_t)t * D : src + (size_t)(base + (t < held ? t : held - 1) - begin) * stride;
        }, held);
    }
    const bool lost = page >= kv.n_blocks;
    if (lost && tid == 0) kv_report(err, kKvErrBlock, r);
    const bool stale = from && !lost && (held_tag.x != page || held_tag.y < from);
    if (stale && tid == 0) kv_report(err, kKvErrOpen, r);
    const bool begins = which == 0 && h == 0 && from == 0 && !lost;  // (once for all heads)
    const uint32_t former = begins ? kv.owner[page] : 0;
    float top = 0.0f, odd = 0.0f;  // odd: NaN with an infinity or a NaN among them
#pragma unroll
    for (int e = 0; e < 16; e++) {
        odd = fmaf(x[e], 0.0f, odd);
        top = fmaxf(top, fabsf(x[e]));
    }
    if (odd != odd || stale) top = __builtin_inff();  // (all of the block becomes NaN)
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    __shared__ float s_top[kWaves];
    if (lane == 0) s_top[c] = top;
    __syncthreads();  // (and every earlier token of the block is read)
#pragma unroll
    for (int i = 0; i < kWaves; i++) top = fmaxf(top, s_top[i]);
    if (!lost) {
        const float s = top == __builtin_inff() ? __builtin_nanf("") : top / 127.0f;
        reinterpret_cast<uint4 *>(kv.codes + (((size_t)page * kv.n_kv + h) * 2 + which) * kKvBlock * D)[tid] = kv_codes16(x, s);
        if (tid == 0) reinterpret_cast<float *>(kv.scales + (size_t)page * kv.n_kv + h)[which] = s;
    }
    // The fp32 tokens of the row's last two blocks: each by its own unit, unless that would
    // overwrite, in the place that both share, tokens from before that the first block's
    // unit reads; then by that one.
    for (uint32_t o = last > first ? last - 1 : last; o <= last; o++) {
        const bool shared = begin % kKvBlock && o > first && (o - first) % 2 == 0;
        if (j != (shared ? first : o)) continue;
        if (o == first && stale) continue;  // (its place holds another block's, or a beginning without a gap)
        const uint32_t of = shared ? b.table[(size_t)r * b.max_blocks + o] : page;
        if (of >= kv.n_blocks) continue;
        const uint32_t b0 = o * kKvBlock, f = begin > b0 ? begin - b0 : 0;
        const uint32_t e = row.len - b0 < kKvBlock ? row.len - b0 : kKvBlock;
        float *dst = kv.open + open_at(kv, r, h, which, o);
        if (shared) {
            for (uint32_t i = f * D + tid; i < e * D; i += 2 * D)
                dst[i] = src[(size_t)(b0 + i / D - begin) * stride + i % D];
        } else if (which == 0) {
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const uint32_t t = n + 16 * hi;
                float4 *to = reinterpret_cast<float4 *>(dst + (size_t)t * D + 32 * c + 8 * g);
                if (t >= f && t < e) {
                    to[0] = make_float4(x[8 * hi], x[8 * hi + 1], x[8 * hi + 2], x[8 * hi + 3]);
                    to[1] = make_float4(x[8 * hi + 4], x[8 * hi + 5], x[8 * hi + 6], x[8 * hi + 7]);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const uint32_t t = 4 * g + u % 4 + 16 * (u / 4);
                if (t >= f && t < e) {
                    dst[(size_t)t * D + 32 * c + n] = x[u];
                    dst[(size_t)t * D + 32 * c + n + 16] = x[8 + u];
                }
            }
        }
        if (tid == 0) tag[o & 1] = make_uint2(of, e);
    }
    if (begins) forget(kv, page, former, r, j + 1 >= last ? j & 1 : 2, 2 * D);
}

template <int D>
__global__ __launch_bounds__(2 * D) void k_kv_append(KvDev kv, KvBatchDev b, const float *k, const float *v, size_t k_stride,
                                                     size_t v_stride, uint32_t *err) {
    if (blockIdx.z == 0) append_unit<D, 0>(kv, b, k, k_stride, err);
    else append_unit<D, 1>(kv, b, v, v_stride, err);
}

// ------------------------------------------------------------------- reading
// The values of single tokens: a thread four channels of a (slot, head).  A few tokens are a
// chain of latencies (one of 16 sequences 4 us); 4,103 tokens of 8 heads of 128 take 13.7 us for 42 MB, where a copy's
// rate would take 8.1: a value's four channels are four loads of a byte, 16 bytes apart.
constexpr int kReadThreads = 256;
template <int D, int U>
__global__ __launch_bounds__(kReadThreads) void k_kv_read(KvDev kv, const uint32_t *slots, uint32_t n, float *k, float *v) {
    constexpr uint32_t kQuads = D / 4, kPer = kReadThreads / kQuads;  // threads of a slot and head, those of a workgroup
    const uint32_t th0 = blockIdx.x * (kPer * U) + threadIdx.x / kQuads, d = threadIdx.x % kQuads * 4, all = n * kv.n_kv;
    if (threadIdx.x >= kPer * kQuads) return;
    uint32_t page[U], slot[U], kb[U], vb[U][4];
    float2 s[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t th = th0 + u * kPer < all ? th0 + u * kPer : all - 1;
        slot[u] = slots[th / kv.n_kv];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t th = th0 + u * kPer < all ? th0 + u * kPer : all - 1, h = th % kv.n_kv, t = slot[u] % kKvBlock, c = d / 32;
        page[u] = slot[u] / kKvBlock;
        const size_t at = (size_t)(page[u] < kv.n_blocks ? page[u] : 0) * kv.n_kv + h;
        s[u] = kv.scales[at];
        const uint8_t *kc = kv.codes + at * (2 * kKvBlock * D), *vc = kc + kKvBlock * D;
        // keys: four channels of one token in a row
        kb[u] = *reinterpret_cast<const uint32_t *>(kc + (c * kWave + (d % 32) / 8 * 16 + t % 16) * 16 + (t / 16) * 8 + d % 8);
        // values: token t is byte (t % 4) + 4 (t / 16) of lane group (t % 16) / 4
        const uint8_t *v0 = vc + (c * kWave + (t % 16) / 4 * 16 + d % 16) * 16 + (d % 32) / 16 * 8 + t % 4 + 4 * (t / 16);
#pragma unroll
        for (int e = 0; e < 4; e++) vb[u][e] = v0[16 * e];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t th = th0 + u * kPer;
        if (th >= all) return;
        if (page[u] >= kv.n_blocks) s[u] = make_float2(__builtin_nanf(""), __builtin_nanf(""));
        const auto val = [](uint32_t byte, float scale) { return (float)((int)byte - 128) * scale; };
        const size_t at = (size_t)th * D + d;
        *reinterpret_cast<float4 *>(k + at) = make_float4(val(kb[u] & 255, s[u].x), val(kb[u] >> 8 & 255, s[u].x),
                                                          val(kb[u] >> 16 & 255, s[u].x), val(kb[u] >> 24, s[u].x));
        *reinterpret_cast<float4 *>(v + at) = make_float4(val(vb[u][0], s[u].y), val(vb[u][1], s[u].y), val(vb[u][2], s[u].y),
                                                          val(vb[u][3], s[u].y));
    }
}

template <int D>
void go_append(const KvDev &kv, const KvBatchDev &b, const float *k, const float *v, size_t k_stride, size_t v_stride,
               uint32_t *err, hipStream_t s) {
    const uint32_t units = append_units(b.n_tokens, b.n_seqs);
    hipLaunchKernelGGL(k_kv_append<D>, dim3(units, kv.n_kv, 2), dim3(2 * D), 0, s, kv, b, k, v, k_stride, v_stride, err);
}

template <int D>
void go_read(const KvDev &kv, const uint32_t *slots, uint32_t n, float *k, float *v, hipStream_t s) {
    constexpr uint32_t kPer = kReadThreads / (D / 4);
    const uint32_t all = n * kv.n_kv;
    // (enough for every CU: four a thread, side by side)
    if (all / kPer >= 2048)
        hipLaunchKernelGGL((k_kv_read<D, 4>), dim3((all + 4 * kPer - 1) / (4 * kPer)), dim3(kReadThreads), 0, s, kv, slots, n, k, v);
    else
        hipLaunchKernelGGL((k_kv_read<D, 1>), dim3((all + kPer - 1) / kPer), dim3(kReadThreads), 0, s, kv, slots, n, k, v);
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanArgs &a, hipStream_t s) {
    if (a.n_seqs == 0 || a.n_seqs > kKvMaxSeqs) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(kPlanThreads), 0, s, a);
    if (a.n_tokens > kPlanTokens) hipLaunchKernelGGL(k_kv_slots, dim3((a.n_tokens + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvDev &kv, const KvBatchDev &b, const float *k, const float *v, size_t k_stride,
                            size_t v_stride, uint32_t *err, hipStream_t s) {
    switch (kv.D) {
    case 64: go_append<64>(kv, b, k, v, k_stride, v_stride, err, s); break;
    case 96: go_append<96>(kv, b, k, v, k_stride, v_stride, err, s); break;
    case 128: go_append<128>(kv, b, k, v, k_stride, v_stride, err, s); break;
    case 192: go_append<192>(kv, b, k, v, k_stride, v_stride, err, s); break;
    case 256: go_append<256>(kv, b, k, v, k_stride, v_stride, err, s); break;
    case 512: go_append<512>(kv, b, k, v, k_stride, v_stride, err, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvDev &kv, const uint32_t *slots, uint32_t n, float *k, float *v, hipStream_t s) {
    if ((uint64_t)n * kv.n_kv >= (1ull << 31)) return hipErrorInvalidValue;  // (slots and heads are counted in 32 bits)
    switch (kv.D) {
    case 64: go_read<64>(kv, slots, n, k, v, s); break;
    case 96: go_read<96>(kv, slots, n, k, v, s); break;
    case 128: go_read<128>(kv, slots, n, k, v, s); break;
    case 192: go_read<192>(kv, slots, n, k, v, s); break;
    case 256: go_read<256>(kv, slots, n, k, v, s); break;
    case 512: go_read<512>(kv, slots, n, k, v, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace lt
