// Gated activation that keeps its operands in 8 bits for the backward pass, and
// the same 8 bits for the rows of a linear layer.
//
//   h = act(g, u);   dg = dh da/dg(g8, u8),  du = dh da/du(g8, u8),   g8, u8: the 8-bit values
//
// What bounds it: HBM, 2 bytes of each of g, u and h per column and 2 of codes
// forward, 2 of codes, 2 of dh and 4 of the gradients backward. A lane holds 8
// columns of g and of u: 16-byte accesses, and four neighbouring lanes make a
// block of 32 columns, whose maximum passes by two DPP steps. 8192 x 14336 silu:
// forward 192 us (948 MB, 4.9 TB/s), gradient 192 (954 MB, 5.0), where a large copy
// reaches 5.2.

#include <type_traits>

#include "../../include/qmoe.h"
#include "eight_bits.h"
#include "gemm_common.h"

namespace {

using namespace qmoe_row;

__device__ __forceinline__ float sigm(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
__device__ __forceinline__ float tanh_of(float x) {
  // odd; near zero 1 - 2 / (1 + e^2x) would cancel
  const float a = fabsf(x), e = __expf(-2.0f * a);
  const float big = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  const float x2 = x * x, small = a * (1.0f + x2 * (-1.0f / 3.0f + x2 * (2.0f / 15.0f - x2 * (17.0f / 315.0f))));
  return copysignf(a < 0.1f ? small : big, x);
}

// clamps that let a NaN through
__device__ __forceinline__ float below(float x, float top) { return x > top ? top : x; }
__device__ __forceinline__ float within(float x, float lim) { return x > lim ? lim : x < -lim ? -lim : x; }

// (value, derivative by g, derivative by u) of the fused activations; a clamp
// passes the gradient up to and at its limits
template <int ACT, bool GRAD>
__device__ __forceinline__ void gated(float g, float u, float p0, float p1, float& h, float& dg, float& du) {
  if constexpr (ACT == QA_SWIGLUOAI) {
    const float gc = below(g, p1), uc = within(u, p1), s = sigm(p0 * gc);
    if constexpr (GRAD) {
      // (far below, gc times the vanished product is zero before it meets p0)
      dg = g > p1 ? 0.0f : (uc + 1.0f) * (s + p0 * (gc * (s * (1.0f - s))));
      du = fabsf(u) > p1 ? 0.0f : gc * s;
    } else {
      h = (uc + 1.0f) * (gc * s);
    }
  } else if constexpr (ACT == QA_GELU_TANH) {
    // (1 + tanh a) / 2 = sigmoid(2 a)
    const float c2 = 2.0f * 0.7978845608028654f, a2 = c2 * (g + 0.044715f * g * g * g), s = sigm(a2);
    if constexpr (GRAD) {
      // (far out one of the sigmoids is zero, and the square may be infinite)
      const float slope = fabsf(g) > 1e3f ? 0.0f : g * s * sigm(-a2) * c2 * (1.0f + 3.0f * 0.044715f * g * g);
      dg = (s + slope) * u;
      du = g * s;
    } else {
      h = g * s * u;
    }
  } else if constexpr (ACT == QA_SITU) {
    const float s = sigm(g), t = tanh_of(g / p0);
    const float v = p1 > 0.0f ? tanh_of(u / p1) : 0.0f, uc = p1 > 0.0f ? p1 * v : u;
    if constexpr (GRAD) {
      dg = ((1.0f - t * t) * s + p0 * t * s * (1.0f - s)) * uc;
      du = p0 * t * s * (p1 > 0.0f ? 1.0f - v * v : 1.0f);
    } else {
      h = p0 * t * s * uc;
    }
  } else {  // QA_SILU, and QA_SILU_CLAMP
    const bool cl = ACT == QA_SILU_CLAMP;
    const float gc = cl ? below(g, p0) : g, uc = cl ? within(u, p0) : u, s = sigm(gc);
    if constexpr (GRAD) {
      dg = cl && g > p0 ? 0.0f : (s + gc * (s * (1.0f - s))) * uc;
      du = cl && fabsf(u) > p0 ? 0.0f : gc * s;
    } else {
      h = gc * s * uc;
    }
  }
}

struct ActParams {
  const uint8_t* x;  // forward: rows of g and u; backward: rows of dh
  int64_t ldx;       // bytes
  uint8_t* y;        // forward: h; backward: dg and du
  int64_t ldy;       // bytes
  uint8_t* codes;
  uint8_t* scales;
  int64_t T, I;
  int nb;  // blocks of 32 columns of g
  float p0, p1;
};

// codes / scale bytes of columns i .. i + 7 of row half r2 (2 t: g, 2 t + 1: u)
template <bool AL>
__device__ __forceinline__ void put_codes(const ActParams& p, int64_t r2, uint32_t i, const float (&v)[8]) {
  uint32_t byte;
  const uint2 c = encode8(v, byte);
  if (i >= p.I) return;
  uint8_t* at = p.codes + r2 * p.I + i;
  if constexpr (AL) {
    *reinterpret_cast<uint2*>(at) = c;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < p.I) at[k] = (uint8_t)((k < 4 ? c.x : c.y) >> (8 * (k & 3)));
  }
  if ((i & 31) == 0) p.scales[r2 * p.nb + i / 32] = (uint8_t)byte;
}
template <bool AL>
__device__ __forceinline__ void get_codes(const ActParams& p, int64_t r2, uint32_t i, uint2& c, uint32_t& byte) {
  const uint8_t* at = p.codes + r2 * p.I + i;
  if constexpr (AL) {
    c = *reinterpret_cast<const uint2*>(at);
  } else {
    c = make_uint2(0, 0);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < p.I) (k < 4 ? c.x : c.y) |= (uint32_t)at[k] << (8 * (k & 3));
  }
  byte = p.scales[r2 * p.nb + i / 32];
}

// Workgroup (t, y): row t (row_group), threads y * blockDim.x .. of 8 columns each
template <int T, int ACT, bool AL>
__global__ __launch_bounds__(512) void act_kernel(const ActParams p) {
  const int64_t t = row_group(), I = p.I;
  if (t >= p.T) return;
  const uint32_t i = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  const uint8_t* x = p.x + t * p.ldx;
  float g[8] = {}, u[8] = {}, h[8];
  if (i < I) {
    const auto gr = load_raw8<T, AL>(x, i, I);
    const auto ur = load_raw8<T, AL>(x + I * rt_size(T), i, I);
    raw8_values<T>(gr, g);
    raw8_values<T>(ur, u);
    float no;
#pragma unroll
    for (int k = 0; k < 8; ++k) gated<ACT, false>(g[k], u[k], p.p0, p.p1, h[k], no, no);
    store8<T, AL>(p.y + t * p.ldy, i, I, h);
  }
  if (!p.codes) return;
  put_codes<AL>(p, 2 * t, i, g);
  put_codes<AL>(p, 2 * t + 1, i, u);
}

template <int T, int ACT, bool AL>
__global__ __launch_bounds__(512) void act_grad_kernel(const ActParams p) {
  const int64_t t = row_group(), I = p.I;
  if (t >= p.T) return;
  const uint32_t i = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (i >= I) return;
  uint2 cg, cu;
  uint32_t bg, bu;
  get_codes<AL>(p, 2 * t, i, cg, bg);
  get_codes<AL>(p, 2 * t + 1, i, cu, bu);
  float g[8], u[8], d[8], no;
  load8<T, AL>(p.x + t * p.ldx, i, I, d);
  decode8(cg, bg, g);
  decode8(cu, bu, u);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float dg, du;
    gated<ACT, true>(g[k], u[k], p.p0, p.p1, no, dg, du);
    g[k] = d[k] * dg;
    u[k] = d[k] * du;
  }
  store8<T, AL>(p.y + t * p.ldy, i, I, g);
  store8<T, AL>(p.y + t * p.ldy + I * rt_size(T), i, I, u);
}

// Rows of bf16 -> 8 bits
__global__ __launch_bounds__(512) void pack_kernel(const ActParams p) {
  const int64_t t = row_group();
  if (t >= p.T) return;
  const uint32_t i = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  float v[8] = {};
  if (i < p.I) load8<RT_BF16, true>(p.x + t * p.ldx, i, p.I, v);
  put_codes<true>(p, t, i, v);
}

// threads of 8 columns, in whole groups of four: as few workgroups per row as
// take 512 at most, alike (8192 x 14336: 194 / 189 us, at most 256 192 / 186, at most 128
// 212 / 194; 777 x 2880 5.4 / 4.7 each)
dim3 row_grid(int64_t T, int64_t I, dim3* block) {
  const int64_t n = cdiv<int64_t>(I, 32) * 4;
  const int64_t parts = cdiv<int64_t>(n, 512);
  block->x = (unsigned)(cdiv<int64_t>(cdiv<int64_t>(n, parts), 64) * 64);
  return row_groups(T, (unsigned)cdiv<int64_t>(n, block->x));
}

template <typename F>
int with_act(int act, int type, bool al, F&& f) {
#define QMOE_ACT_CASE(A)                                                                                              \
  case A:                                                                                                             \
    if (type == RT_BF16 && al) f(std::integral_constant<int, RT_BF16>(), std::integral_constant<int, A>(), std::true_type()); \
    else if (type == RT_BF16) f(std::integral_constant<int, RT_BF16>(), std::integral_constant<int, A>(), std::false_type()); \
    else if (al) f(std::integral_constant<int, RT_F16>(), std::integral_constant<int, A>(), std::true_type());        \
    else f(std::integral_constant<int, RT_F16>(), std::integral_constant<int, A>(), std::false_type());               \
    return QMOE_OK
  switch (act) {
    QMOE_ACT_CASE(QA_SILU);
    QMOE_ACT_CASE(QA_SWIGLUOAI);
    QMOE_ACT_CASE(QA_GELU_TANH);
    QMOE_ACT_CASE(QA_SILU_CLAMP);
    QMOE_ACT_CASE(QA_SITU);
    default: return QMOE_ERR_ARG;
  }
#undef QMOE_ACT_CASE
}

bool al16(const void* p, int64_t ld_bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0; }

constexpr int64_t kMaxRows = 1 << 24, kMaxCols = 1 << 20;

}  // namespace

// See include/qmoe.h for the contract.
extern "C" int qmoe_act_checkpoint(const void* x, int64_t ldx, int type, int64_t T, int64_t I, int act, float act_p0,
                                   float act_p1, void* h, int64_t ldh, uint8_t* codes, uint8_t* scales,
                                   hipStream_t stream) {
  if (!x || !h || T < 1 || T > kMaxRows || I < 1 || I > kMaxCols || (type != RT_BF16 && type != RT_F16) ||
      ldx < 2 * I || ldh < I || (codes && !scales))
    return QMOE_ERR_ARG;
  const ActParams p{static_cast<const uint8_t*>(x), ldx * 2, static_cast<uint8_t*>(h), ldh * 2, codes, scales, T, I,
                    (int)cdiv<int64_t>(I, 32), act_p0, act_p1};
  const bool al = I % 8 == 0 && al16(x, ldx * 2) && al16(h, ldh * 2) && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
  dim3 block;
  const dim3 grid = row_grid(T, I, &block);
  const int st = with_act(act, type, al, [&](auto t, auto a, auto w) {
    hipLaunchKernelGGL((act_kernel<t(), a(), w()>), grid, block, 0, stream, p);
  });
  if (st != QMOE_OK) return st;
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_act_checkpoint_grad(const uint8_t* codes, const uint8_t* scales, int64_t T, int64_t I, int act,
                                        float act_p0, float act_p1, const void* dh, int64_t lddh, int type, void* dx,
                                        hipStream_t stream) {
  if (!codes || !scales || !dh || !dx || T < 1 || T > kMaxRows || I < 1 || I > kMaxCols ||
      (type != RT_BF16 && type != RT_F16) || lddh < I)
    return QMOE_ERR_ARG;
  const ActParams p{static_cast<const uint8_t*>(dh), lddh * 2, static_cast<uint8_t*>(dx), 4 * I,
                    const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales), T, I, (int)cdiv<int64_t>(I, 32), act_p0,
                    act_p1};
  const bool al = I % 8 == 0 && al16(dh, lddh * 2) && al16(dx, 4 * I) && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
  dim3 block;
  const dim3 grid = row_grid(T, I, &block);
  const int st = with_act(act, type, al, [&](auto t, auto a, auto w) {
    hipLaunchKernelGGL((act_grad_kernel<t(), a(), w()>), grid, block, 0, stream, p);
  });
  if (st != QMOE_OK) return st;
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_pack_8bit(const void* x, int64_t ldx, int64_t T, int64_t K, uint8_t* codes, uint8_t* scales,
                              hipStream_t stream) {
  if (!x || !codes || !scales || T < 1 || T > kMaxRows || K < 1 || K > kMaxCols || K % 8 || ldx < K ||
      !al16(x, ldx * 2) || reinterpret_cast<uintptr_t>(codes) % 8)
    return QMOE_ERR_ARG;
  const ActParams p{static_cast<const uint8_t*>(x), ldx * 2, nullptr, 0, codes, scales, T, K, (int)cdiv<int64_t>(K, 32),
                    0.0f, 0.0f};
  dim3 block;
  const dim3 grid = row_grid(T, K, &block);
  hipLaunchKernelGGL(pack_kernel, grid, block, 0, stream, p);
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
