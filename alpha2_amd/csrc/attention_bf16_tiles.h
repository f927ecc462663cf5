// Tiles of 64 streamed rows in LDS and what the 32x32x16 bf16 matrix instructions read of them: shared by the attention kernels whose queries are the
// accumulators' columns (attention_bf16.hip has the arrangement).
#pragma once
#include "attention_common.h"

namespace ah {

constexpr int ST = 64;       // streamed rows per LDS tile
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4 lds_v4;

template <int D> struct Geo {
  static constexpr int PITCH = D + 16;                 // bf16 elements; (D+16)*2 bytes = 32 mod 128 for D in {32,64,128}... see tile_frag_t
  static constexpr int ELEMS = ST * PITCH;
  static constexpr int CHUNKS = ST * D / 8 / 256;      // 16-byte chunks per thread per tile (D=32: 1, 64: 2, 128: 4)
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float FIXED_MAX_CAP = 40.f;      // soft caps up to this use the constant-maximum softmax
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
// First statement of a block that only the tiles on the diagonal need (masking): with it the compiler keeps the block behind a
// branch the other tiles skip, where it would otherwise turn a cheap block into selects that every tile executes.
__device__ __forceinline__ void keep_branch() { asm volatile("; rare path" ::: "memory"); }

template <int D>
__device__ __forceinline__ void tile_store(uint16_t *s, const u32x4 (&v)[Geo<D>::CHUNKS]) {
#pragma unroll
  for (int i = 0; i < Geo<D>::CHUNKS; i++) {
    int c = threadIdx.x + 256 * i, r = c / (D / 8), c8 = c % (D / 8);
    *reinterpret_cast<u32x4 *>(s + r * Geo<D>::PITCH + c8 * 8) = v[i];
  }
}
// A/B fragment with the tile ROW as the MFMA row/column (k = feature d): rows r0 + lane%32, d = 16*ks + 8*(lane/32)..
template <int D>
__device__ __forceinline__ bf16x8 tile_frag(const uint16_t *s, int r0, int ks, int lane) {
  return *reinterpret_cast<const bf16x8 *>(s + (r0 + (lane & 31)) * Geo<D>::PITCH + ks * 16 + (lane >> 5) * 8);
}
// A fragment with the feature d as the MFMA row (k = tile row, in the accumulator's slot order): features
// 32*db + lane%32, k-slot i of this half = tile row r0 + 16m + 8(i/4) + 4(lane/32) + i%4.
template <int D>
__device__ __forceinline__ bf16x8 tile_frag_t(const uint16_t *s, int r0, int m, int db, int lane) {
  int j = lane & 15, g = lane >> 4, lk = g >> 1;
  const uint16_t *p = s + (r0 + 16 * m + 4 * lk + (j >> 2)) * Geo<D>::PITCH + 32 * db + 16 * (g & 1) + 4 * (j & 3);
  bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)p);
  bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)(p + 8 * Geo<D>::PITCH));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
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
