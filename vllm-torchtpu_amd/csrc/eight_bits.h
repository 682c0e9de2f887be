// 8 bits of a row: per 32 columns e4m3fn codes and one power of two, 2^(s - 127)
// with s the least byte for which the columns' finite absolute maximum is at
// most 448 2^(s - 127): nothing saturates, and dividing by the scale is exact,
// so a value is rounded once, to the code. Infinities and NaN become NaN codes
// and count for no scale.
#pragma once

#include "row_values.h"

namespace qmoe_row {

// The scale byte of 32 columns from the largest bits of their finite values.
// 448 = 1.75 2^8: the byte is the maximum's exponent - 8, or - 7 above 1.75
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int s = (int)(amax >> 23) - ((amax & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return (uint32_t)(s < 0 ? 0 : s);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return v > o ? v : o;
}

// 8 values of a lane -> codes, with the scale byte of the 32 columns that this
// lane and the other three of its group of four hold
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t a = f32_bits(v[k]) & 0x7fffffffu;
    m = a < 0x7f800000u && a > m ? a : m;
  }
  m = dpp_umax<0xB1>(m);
  m = dpp_umax<0x4E>(m);
  byte = scale_byte(m);
  const float inv = bits_f32((254u - byte) << 23);
  float q[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    q[k] = (f32_bits(v[k]) & 0x7fffffffu) < 0x7f800000u ? v[k] * inv : __builtin_nanf("");
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// 8 codes and their scale byte -> values, exactly
__device__ __forceinline__ void decode8(uint2 c, uint32_t byte, float (&v)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const float s = e8m0_to_f32(byte);
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
  const f2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
  v[0] = a[0] * s, v[1] = a[1] * s, v[2] = b[0] * s, v[3] = b[1] * s;
  v[4] = d[0] * s, v[5] = d[1] * s, v[6] = e[0] * s, v[7] = e[1] * s;
}

}  // namespace qmoe_row
