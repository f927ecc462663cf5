// What the attention kernels share whose queries are the accumulators' columns (attention_bf16.hip has the arrangement): the streamed tile's rows, exponentials, and the
// way of a 32x32 accumulator into the next product and out to memory.  How each keeps its tiles in LDS is its own.
#pragma once
#include "attention_common.h"

namespace ah {

constexpr int ST = 64;       // streamed rows per LDS tile
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4 lds_v4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float FIXED_MAX_CAP = 40.f;      // soft caps up to this use the constant-maximum softmax
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
// First statement of a block that only the tiles on the diagonal need (masking): with it the compiler keeps the block behind a
// branch the other tiles skip, where it would otherwise turn a cheap block into selects that every tile executes.
__device__ __forceinline__ void keep_branch() { asm volatile("; rare path" ::: "memory"); }

// accumulator registers 8m..8m+7 -> bf16 B operand of MFMA m
__device__ __forceinline__ bf16x8 acc_to_b(const f32x16 &s, int m) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = (__bf16)s[8 * m + i];
  return r;
}
// O^T-style accumulators (rows = features 32db + 8j + 4h + r, column = owned row) -> bf16 row-major store
template <int D, bool PAD = false>
__device__ __forceinline__ void store_rows(uint16_t *__restrict__ dst, const f32x16 (&acc)[D / 32], float mul, int lane, int hd = D) {
  int lk = lane >> 5;
#pragma unroll
  for (int db = 0; db < D / 32; db++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint2 w = make_uint2(pack_bf16x2(acc[db][4 * j] * mul, acc[db][4 * j + 1] * mul), pack_bf16x2(acc[db][4 * j + 2] * mul, acc[db][4 * j + 3] * mul));
      if (!PAD || 32 * db + 8 * j + 4 * lk < hd) *reinterpret_cast<uint2 *>(dst + 32 * db + 8 * j + 4 * lk) = w;
    }
}

}  // namespace ah
