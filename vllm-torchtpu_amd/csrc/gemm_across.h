// What the bf16 products with an operand across K share (vocabulary loss, gradients
// of a linear layer): K is the contiguous axis of an ordinary operand; of one
// that lies across K a stage is 64 K rows, copied to LDS as they lie and
// transposed on the way to registers.
#pragma once

#include "gemm_tile.h"

namespace {

__device__ __align__(16) const uint32_t kZeroChunk[4] = {0, 0, 0, 0};

// How an operand across K, rows of 256 or BM columns, passes through LDS.
// ds_read_b64_tr_b16: lane 4 r + c of 16 gives the address of row r's
// elements 4 c .. + 3, lane i receives column i of the 4 rows. An MFMA operand is
// two of them (k + 4) per lane; the 4 rows of an access lie in different 64-byte
// blocks, for which the 16-byte chunk c of row k is stored at c ^ tr_swz.
template <int RB>  // bytes of a row
__device__ __forceinline__ int tr_swz(int k) {
  return 4 * (RB == 128 ? (k >> 1) & 1 : k & 3);
}
// Byte of the lane's first 4 x 4 of k 0 .. 15 of columns 0 .. 31; those of columns
// 32 f .. are at this ^ 64 f
template <int RB>
__device__ __forceinline__ uint32_t tr_lane(int lane) {
  const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);
  return (uint32_t)(k * RB + ((32 * ((lane >> 4) & 1) + 8 * (lane & 3)) ^ (tr_swz<RB>(k) * 16)));
}
template <int RB>
__device__ __forceinline__ uint4 tr_read(const uint8_t* at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* Lds;
  union {
    s16x4 h[2];
    uint4 u;
  } r;
  r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(void*)at);
  r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(void*)(at + 4 * RB));
  return r.u;
}

__device__ __forceinline__ int vg_swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* q) {
  const uint64_t b = reinterpret_cast<uint64_t>(q);
  return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((int)b));
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  union {
    bf16x2 h;
    uint32_t u;
  } r;
  r.h = __builtin_convertvector(f32x2{a, b}, bf16x2);
  return r.u;
}

// opaque_*: a value the compiler takes for a new one, so that what depends on
// it (64 row scales, masks or addresses) is not kept for all MJ rounds at once.
__device__ __forceinline__ int opaque_s(int v) {
  asm volatile("" : "+s"(v));
  return v;
}
__device__ __forceinline__ int opaque_v(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ int vg_row_swz(int t) { return 4 * ((t ^ (t >> 3)) & 15); }

}  // namespace
