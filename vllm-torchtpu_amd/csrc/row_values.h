// Eight consecutive values of a row as float32, of the row types that the
// block's elementwise kernels take (bf16, f32, f16), and sums over wavefronts. A
// row's address is uniform and places in it are 32-bit offsets, so that accesses
// take a scalar base and one register.
#pragma once

#include "qmoe_common.h"

namespace qmoe_row {

enum { RT_BF16 = 0, RT_F32 = 1, RT_F16 = 2 };

QMOE_HD int rt_size(int t) { return t == RT_F32 ? 4 : 2; }

// Workgroups of a launch with one for every (few) rows: blockIdx.x, and above 2^16 of
// them blockIdx.z, since a launch takes less than 2^32 threads along an axis. The last
// of z may lie behind the end.
constexpr int64_t kRowGroups = 1 << 16;
inline dim3 row_groups(int64_t n, unsigned y = 1) {
  return dim3((unsigned)(n < kRowGroups ? n : kRowGroups), y, (unsigned)cdiv(n, kRowGroups));
}
__device__ __forceinline__ int64_t row_group() { return (int64_t)blockIdx.z * kRowGroups + blockIdx.x; }

// The values as they lie in memory, to be loaded long before they are used
template <int T>
struct Raw8 {
  uint4 q[T == RT_F32 ? 2 : 1];
};

template <int T>
__device__ __forceinline__ float one_value(const void* p, int64_t i) {
  if constexpr (T == RT_F32) return static_cast<const float*>(p)[i];
  else if constexpr (T == RT_BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return (float)static_cast<const _Float16*>(p)[i];
}

// Values i .. i + 7 of the row at p; AL: 16-byte aligned, and all there; else
// those from n on are zeros
template <int T, bool AL>
__device__ __forceinline__ Raw8<T> load_raw8(const void* p, uint32_t i, uint32_t n) {
  Raw8<T> r;
  if constexpr (AL) {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (T == RT_F32 ? 4u : 2u));
    r.q[0] = s[0];
    if constexpr (T == RT_F32) r.q[1] = s[1];
  } else if constexpr (T == RT_F32) {
    union {
      float f[8];
      uint4 q[2];
    } u;
#pragma unroll
    for (int k = 0; k < 8; ++k) u.f[k] = i + k < n ? static_cast<const float*>(p)[i + k] : 0.0f;
    r.q[0] = u.q[0];
    r.q[1] = u.q[1];
  } else {
    union {
      uint16_t h[8];
      uint4 q;
    } u;
#pragma unroll
    for (int k = 0; k < 8; ++k) u.h[k] = i + k < n ? static_cast<const uint16_t*>(p)[i + k] : (uint16_t)0;
    r.q[0] = u.q;
  }
  return r;
}

template <int T>
__device__ __forceinline__ void raw8_values(const Raw8<T>& r, float (&v)[8]) {
  union {
    uint4 q[2];
    uint32_t d[8];
    _Float16 e[16];
    float f[8];
  } u;
  u.q[0] = r.q[0];
  if constexpr (T == RT_F32) u.q[1] = r.q[1];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (T == RT_F32) v[k] = u.f[k];
    else if constexpr (T == RT_F16) v[k] = (float)u.e[k];
    else v[k] = bits_f32(k & 1 ? u.d[k / 2] & 0xffff0000u : u.d[k / 2] << 16);
  }
}

template <int T, bool AL>
__device__ __forceinline__ void load8(const void* p, uint32_t i, uint32_t n, float (&v)[8]) {
  raw8_values<T>(load_raw8<T, AL>(p, i, n), v);
}

// ... of a type known at run time (uniform)
template <bool AL>
__device__ __forceinline__ void load8_any(const void* p, int type, uint32_t i, uint32_t n, float (&v)[8]) {
  if (type == RT_BF16) load8<RT_BF16, AL>(p, i, n, v);
  else if (type == RT_F32) load8<RT_F32, AL>(p, i, n, v);
  else load8<RT_F16, AL>(p, i, n, v);
}
__device__ __forceinline__ float one_any(const void* p, int type, int64_t i) {
  return type == RT_BF16 ? one_value<RT_BF16>(p, i) : type == RT_F32 ? one_value<RT_F32>(p, i) : one_value<RT_F16>(p, i);
}

// One value as its type holds it (round to nearest, ties to even)
template <int T>
__device__ __forceinline__ float round_to(float f) {
  if constexpr (T == RT_BF16) return bf16_round(f);
  else if constexpr (T == RT_F16) return (float)(_Float16)f;
  else return f;
}

__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  union {
    bf16x2 h;
    uint32_t u;
  } r;
  r.h = __builtin_convertvector(f2{a, b}, bf16x2);
  return r.u;
}

template <int T, bool AL>
__device__ __forceinline__ void store8(void* p, uint32_t i, uint32_t n, const float (&v)[8]) {
  if constexpr (!AL) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) {
        if constexpr (T == RT_F32) static_cast<float*>(p)[i + k] = v[k];
        else if constexpr (T == RT_F16) static_cast<_Float16*>(p)[i + k] = (_Float16)v[k];
        else static_cast<uint16_t*>(p)[i + k] = f32_to_bf16(v[k]);
      }
  } else {
    uint4* d = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + i * (T == RT_F32 ? 4u : 2u));
    if constexpr (T == RT_F32) {
      d[0] = make_uint4(f32_bits(v[0]), f32_bits(v[1]), f32_bits(v[2]), f32_bits(v[3]));
      d[1] = make_uint4(f32_bits(v[4]), f32_bits(v[5]), f32_bits(v[6]), f32_bits(v[7]));
    } else if constexpr (T == RT_BF16) {
      d[0] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
    } else {
      union {
        _Float16 e[8];
        uint4 q;
      } u;
#pragma unroll
      for (int k = 0; k < 8; ++k) u.e[k] = (_Float16)v[k];
      d[0] = u.q;
    }
  }
}

// Sum over the wavefront, in every lane: DPP inside rows of 16 lanes, then the
// four rows' sums through scalars
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float wave_total(float v) {
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  v = dpp_add<0x140>(v);
  const int i = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

}  // namespace qmoe_row
