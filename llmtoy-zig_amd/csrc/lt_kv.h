// lt_kv.h -- the 8-bit key/value cache: its layout, and how a batch's tokens
// and tiles are found on the device.
//
// A block holds kKvBlock = 32 tokens of one sequence.  For each block and head
// keys and values have one scale each, s = max |x| / 127, and a byte code + 128
// an element, code = round(x / s).  A (block, head)'s keys and values lie
// together, as operands of v_mfma_f32_16x16x32_f16, so that a wave's loads are
// whole KiB in order.  With lane = 16 g + n (g < 4, n < 16) and piece c of 32
// channels, the 16 bytes at (c * 64 + lane) * 16 are
//   keys    bytes 0-7: token n, channels 32 c + 8 g + 0..7; bytes 8-15: token 16 + n
//   values  bytes 0-7: channel 32 c + n, tokens 4 g + 0..3 and 16 + 4 g + 0..3;
//           bytes 8-15: channel 32 c + 16 + n
// The tokens' order in the values is the one in which the product of keys and
// queries leaves its results in a lane: the softmax's weights then are the next
// product's operand as they stand.
//
// The tokens of a sequence's last two blocks are also kept in fp32 (KvDev::open,
// by its row of the batch and the parity of the block's index), so that a block is coded from its tokens
// and never from codes, however they come.  A tag says whose they are: the block of the cache, and
// how many.  A block that is begun anew takes itself out of the tags of the row that had it
// (KvDev::owner), so that a tag never names a block that another sequence, or the same one anew, has written since.
#pragma once
#include "lt_cut.h"
#include "lt_internal.h"

namespace lt {

constexpr uint32_t kKvBlock = 32, kKvNone = 0xffffffffu;
constexpr uint32_t kKvMaxSeqs = 4096;  // (kv_row: two rounds of 64)
constexpr uint32_t kKvMaxTokens = 1u << 24;

// Words of the context's host-mapped error memory that the cache's kernels
// write (row + 1), one for each kind of fault.
enum KvErr : int { kKvErrPool = 9, kKvErrRoom, kKvErrBlock, kKvErrOpen, kKvErrRows, kKvErrEnd };

struct KvDev {
    uint8_t *codes;   // [n_blocks][n_kv][2][32 * D]
    float2 *scales;   // [n_blocks][n_kv]: keys', values'
    float *open;      // [n_seqs][n_kv][2 keys, values][2 parity][32][D]
    uint2 *tags;      // [n_seqs][n_kv][2][2]: block of the cache, tokens held (0: none)
    uint32_t *owner;  // [n_blocks]: row + 1 that began the block last (0: none)
    uint32_t n_blocks, n_kv, D, n_seqs;
};

struct KvBatchDev {
    uint32_t n_seqs, n_tokens, max_blocks, max_new;
    const uint32_t *start, *len, *table;
};

// One sequence's part of a batch: its tokens first .. first + n - 1, at the
// positions len - n .. len - 1.  bad: the arrays contradict themselves; falls: by a
// start that falls, so that n is 0; behind: by tokens that all lie behind n_tokens, so that n is 0 too.
struct KvRow {
    uint32_t first, n, len;
    bool bad, falls, behind;
};

#ifdef __HIPCC__

__device__ __forceinline__ void kv_report(uint32_t *err, int kind, uint32_t row) {
    __hip_atomic_store(err + kind, row + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

__device__ __forceinline__ KvRow kv_row_of(const KvBatchDev &b, uint32_t r) {
    KvRow k;
    const uint32_t s0 = b.start[r], s1 = b.start[r + 1], room = b.n_tokens;
    k.first = s0 < room ? s0 : room;
    const uint32_t end = s1 < room ? s1 : room;
    k.n = end > k.first ? end - k.first : 0;
    k.len = b.len[r];
    k.falls = s1 < s0;
    k.behind = s0 >= room && s1 > s0;
    k.bad = s1 > room || k.len < k.n || k.len > b.max_blocks * kKvBlock || (b.max_new && k.n > b.max_new);
    return k;
}

// The last row r < n_seqs with base(r) <= u, base not falling, base(0) = 0: by a
// whole wavefront, 64 rows at once, then the 64 behind the last of those.
template <typename F>
__device__ __forceinline__ uint32_t kv_row(uint32_t n_seqs, uint32_t u, F base) {
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t lo = 0;
    if (n_seqs > kWave) {
        const uint32_t r = lane * kWave;
        const uint64_t below = __ballot(r < n_seqs && base(r) <= u);
        lo = (below ? 63 - __builtin_clzll(below) : 0) * kWave;
    }
    const uint32_t r = lo + lane;
    const uint64_t below = __ballot(r < n_seqs && base(r) <= u);
    return lo + (below ? 63 - __builtin_clzll(below) : 0);
}

#endif  // __HIPCC__

// Device table of a rotation (lt_rope.hip): the turns a position that pair i's
// angle grows by.
struct RopeDev {
    const double *turns;  // [n_rot / 2]
    uint32_t D, n_rot, style;
};

hipError_t launch_qk_norm_rope(const RopeDev &rope, float *q_out, float *k_out, const float *q, const float *k,
                               const float *wq, const float *wk, const uint32_t *pos, uint32_t T, uint32_t n_heads,
                               uint32_t n_kv, const size_t stride[4], float eps, bool norm, bool one_plus,
                               hipStream_t s);
struct KvPlanArgs {
    uint32_t n_seqs, max_blocks, n_tokens, n_free;
    const uint32_t *len_in, *n_new, *free_blocks, *used_in;
    uint32_t *table, *len, *start, *used, *pos, *slot, *err;
};
hipError_t launch_kv_plan(const KvPlanArgs &a, hipStream_t s);
hipError_t launch_kv_append(const KvDev &kv, const KvBatchDev &b, const float *k, const float *v, size_t k_stride,
                            size_t v_stride, uint32_t *err, hipStream_t s);
hipError_t launch_kv_read(const KvDev &kv, const uint32_t *slots, uint32_t n, float *k, float *v, hipStream_t s);
struct AttnArgs {
    KvDev kv;
    KvBatchDev b;
    const float *q;
    float *out;
    size_t q_stride;
    uint32_t n_heads, group, window;
    float scale;
    void *work;
    uint32_t *tickets;  // kAttnTickets words, zero between launches
    uint32_t *err;
};
bool attention_head_dim(uint32_t D);
size_t attention_workspace(const AttnArgs &a);
hipError_t launch_attention(const AttnArgs &a, hipStream_t s);
size_t attention_wide_workspace(uint32_t D);
hipError_t launch_attention_wide(const AttnArgs &a, hipStream_t s);

}  // namespace lt
