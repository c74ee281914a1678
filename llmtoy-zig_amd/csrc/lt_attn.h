// lt_attn.h -- what the attention's two kernels share (lt_attention.hip: few rows,
// lt_attention_wide.hip: many).
#pragma once
#include "lt_kv.h"

#ifdef __HIPCC__

namespace lt {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The reference of the weights may lag behind the largest logit by this much
// (base 2), so that sums are rarely scaled down; weights go in times 2^kBits, and
// 2^(kBits + kSlack) is in f16's range.
constexpr float kSlack = 3.0f, kBits = 12.0f;

constexpr float kNegInf = -__builtin_huge_valf();

// log2 of a block's value scale.  A block of zeros has none: below every real one (2^-149 at least), so that its
// logits count in the softmax's sum and never set the reference that real values' weights are held against.
__device__ __forceinline__ float log2_scale(float s) { return s == 0.0f ? -200.0f : log2f(s); }

__device__ __forceinline__ uint32_t from_lane(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// A barrier behind which the workgroup's LDS accesses are done, and no more: __syncthreads
// also waits for the loads from memory that are under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A byte code + 128 is the f16 number 1024 + 128 + code with the byte 0x64 above it.
__device__ __forceinline__ half8 codes8(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        half2v h[4];
        half8 v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - off;
    return r.v;
}

// Two numbers as f16, and what is left of them.
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ half2v pair(float a, float b) { return __builtin_convertvector((f32x2{a, b}), half2v); }
// What is left of p beside h's first or second half, in one instruction.
__device__ __forceinline__ float rest0(half2v h, float p) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    return r;
}
__device__ __forceinline__ float rest1(half2v h, float p) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    return r;
}

// Partial results go past the L2s (sc1: agent scope), since another XCD reads them: 16 bytes a lane,
// at a float's index from the workspace's begin.
struct Shared {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ Shared(float *p, uint32_t floats) : r(__builtin_amdgcn_make_buffer_rsrc(p, 0, floats * 4, 0x00020000)) {}
    __device__ __forceinline__ void put(uint32_t at, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at * 4, 0, kPast);
    }
    __device__ __forceinline__ f32x4 get(uint32_t at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at * 4, 0, kPast));
    }
    static constexpr int kPast = 16;  // sc1
};

// What an output is of its sums: 2^(mo - m) / l, without the weights' 2^bits; no
// key seen: 0.
__device__ __forceinline__ float out_scale(float m, float l, float mo, float bits) {
    return l > 0.0f || l != l ? (mo == kNegInf ? 0.0f : exp2f(mo - m - bits)) / l : 0.0f;
}

}  // namespace lt

#endif  // __HIPCC__
