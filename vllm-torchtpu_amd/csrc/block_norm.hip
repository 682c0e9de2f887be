// The norms before and after a block, fused with its gate and the residual:
//
//   n(a; w) = a r(a) (off + w),  r(a) = (mean a^2 + eps)^(-1/2)
//   b = n(y; wp) or y,   h = rs res + sc gate b (rounded as it is stored),   z = n(h; wn)
//
// (gate: one value per channel, per token or per element; every part but the
// residual may be left out, and without y h is the residual itself). With G the
// gradient of h, H the row length and means over a row:
//
//   H' = G + r(h) (gz - nh mean(gz nh)),  gz = dz (off + wn), nh = h r(h);   dwn = sum_t dz nh
//   dres = rs H',  db = sc gate H',  dgate = sc H' b (summed over what shares the gate)
//   dy = db, or r(y) (gp - ny mean(gp ny)),  gp = db (off + wp), ny = y r(y);   dwp = sum_t db ny
//
// What bounds it: HBM. A row is read once into registers: W wavefronts hold C
// pieces of 8 values per lane, and the row's two statistics (one after the other:
// the second norm needs the first's result) pass through LDS. R rows share a
// workgroup. The sums over tokens stay in registers over all rows of a workgroup
// and are added up by a second launch in a fixed order, without atomics.
//
// 8192 rows of 7168 bf16, both norms: forward 105 us (96 at best; 472 MB, 4.5 to 4.9 TB/s
// where a large copy reaches 5.2), gradients 174 (160; 720 MB, 4.1 to 4.5) and the sums
// over rows 5.5. 1024 rows of 4096 forward 11.0, one row 4.3. The next norm alone (no y),
// 8192 rows of 7168 bf16: forward 39 us (235 MB, 6.1 TB/s: the last level cache holds the
// rows), gradients 76 (352 MB, 4.6) and 4; one row 2.8 and 3.5 + 2.7.
//
// A row whose squares add up beyond float32's range has a row factor of zero: zeros
// behind the norm, and no gradient through it.

#include <type_traits>

#include "../../include/qmoe.h"
#include "row_values.h"

namespace {

using namespace qmoe_row;

constexpr int kMaxThreads = 1024;
constexpr int64_t kMaxLdsRow = 8192;  // two float32 vectors of a row in 64 KB of LDS
constexpr int64_t kMaxRow = kMaxThreads * 16, kMaxRows = 1 << 24;

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_TOKEN = 2, GATE_FULL = 3 };

// Sums of K values over the W wavefronts of a row (threadIdx.y: the row of the
// workgroup); `red` is this reduction's own LDS
template <int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*red)[16][K], int W) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_total(v[k]);
  if (W == 1) return;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[threadIdx.y][w][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.0f;
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += red[threadIdx.y][i][k];
}

// r of a row from its sum of squares, in float64: its error is one of every value of
// the row, and these few steps in float32 would double it (rms 5.1e-8 against 3.6e-8
// of a row of 7168)
__device__ __forceinline__ float row_factor(float sum, double inv, float eps) {
  return (float)rsqrt((double)sum * inv + (double)eps);
}

// Piece c of this thread starts at this column
__device__ __forceinline__ uint32_t piece(int c) { return (c * blockDim.x + threadIdx.x) * 8; }

// This wavefront's row of the workgroup
__device__ __forceinline__ int own_row() { return __builtin_amdgcn_readfirstlane(threadIdx.y); }

template <int YT, int RT, int C, int THREADS, bool AL>
__global__ __launch_bounds__(THREADS) void block_residual_kernel(const qmoe_block_desc p) {
  __shared__ float red[2][8][16][1];
  const int W = blockDim.x >> 6;
  const int64_t t = row_group() * blockDim.y + own_row();
  const uint32_t H = (uint32_t)p.H;
  const double inv = 1.0 / (double)H;
  const bool row = t < p.T;
  Raw8<YT> yr[C], gr[C];
  Raw8<RT> rr[C];
  const uint8_t* res = static_cast<const uint8_t*>(p.residual) + t * p.ldr * rt_size(RT);
  const uint8_t* y = static_cast<const uint8_t*>(p.y) + t * p.ldy * rt_size(YT);
  const uint8_t* full = static_cast<const uint8_t*>(p.gate) + t * p.ldg * rt_size(YT);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = piece(c);
    if (!row || i >= H) continue;
    if (p.y) yr[c] = load_raw8<YT, AL>(y, i, H);
    if (p.gate_kind == GATE_FULL) gr[c] = load_raw8<YT, AL>(full, i, H);
    rr[c] = load_raw8<RT, AL>(res, i, H);
  }
  float h[C][8];
  float ry = 1.0f;
  if (p.y && p.post_weight) {
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!row || piece(c) >= H) continue;
      float v[8];
      raw8_values<YT>(yr[c], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[0] += v[k] * v[k];
    }
    row_sums<1>(s, red[0], W);
    // (multiplied first: of a row of the type's lowest value it is zero, and so is the norm)
    ry = row_factor(s[0], inv, p.eps);
    if (row && p.rstd_y && threadIdx.x == 0) p.rstd_y[t] = ry;
  }
  const float gt = p.gate_kind == GATE_TOKEN && row ? one_any(p.gate, p.gate_type, t) : 1.0f;
  float s[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = piece(c);
    if (!row || i >= H) continue;
    raw8_values<RT>(rr[c], h[c]);
    if (p.y) {
      float v[8], m[8];
      raw8_values<YT>(yr[c], v);
      if (p.post_weight) {
        load8_any<AL>(p.post_weight, p.weight_type, i, H, m);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] * ry * (p.weight_offset + m[k]);
      }
      if (p.gate_kind == GATE_CHANNEL) load8_any<AL>(p.gate, p.gate_type, i, H, m);
      if (p.gate_kind == GATE_FULL) raw8_values<YT>(gr[c], m);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float g = p.gate_kind == GATE_CHANNEL || p.gate_kind == GATE_FULL ? m[k] : gt;
        h[c][k] = round_to<RT>(p.residual_scale * h[c][k] + p.scale * (g * v[k]));
      }
      store8<RT, AL>(static_cast<uint8_t*>(p.h) + t * p.ldh * rt_size(RT), i, H, h[c]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s[0] += !AL && i + k >= H ? 0.0f : h[c][k] * h[c][k];
  }
  if (!p.next_weight) return;
  row_sums<1>(s, red[1], W);
  const float rh = row_factor(s[0], inv, p.eps);
  if (row && p.rstd_h && threadIdx.x == 0) p.rstd_h[t] = rh;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = piece(c);
    if (!row || i >= H) continue;
    float m[8];
    load8_any<AL>(p.next_weight, p.weight_type, i, H, m);
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = h[c][k] * rh * (p.weight_offset + m[k]);
    store8<YT, AL>(static_cast<uint8_t*>(p.z) + t * p.ldz * rt_size(YT), i, H, m);
  }
}

// The gradients. What rows share are two vectors, c1 = off + wn and c2 = (off + wp)
// gate (a gate per channel; else without it), and what is summed over tokens are two
// as well: dz nh, and H' ny (times a gate per token or element), of which the
// gradients of wp and of a gate per channel are the multiples by sc gate and sc
// (off + wp). c1 and c2 lie in LDS (LDSC; rows of up to 8192), the sums in
// registers; they leave in parts [workgroups][2][H].
// PARTS: 1 both norms are there, 2 the second alone (no y), 0 asked at run time, at
// the cost of registers.
template <int YT, int RT, int C, int THREADS, bool AL, int PARTS, bool LDSC>
__global__ __launch_bounds__(THREADS, THREADS == 512 && AL ? 4 : 1) void block_residual_grad_kernel(
    const qmoe_block_desc p, const qmoe_block_grads d, float* parts) {
  __shared__ float red1[2][8][16][1], red2[2][8][16][2];
  extern __shared__ float dyn[];  // LDSC: c1 [H8], c2 [H8]; afterwards rows' sums
  const int W = blockDim.x >> 6, R = blockDim.y;
  const uint32_t H = (uint32_t)p.H, H8 = (H + 7) / 8 * 8;
  const float invH = 1.0f / (float)H;
  const bool has_y = PARTS ? PARTS == 1 : p.y != nullptr, post = PARTS ? PARTS == 1 : p.y && p.post_weight,
             next = PARTS || (p.next_weight && d.g_z);
  const int kind = p.gate_kind;
  auto make_c1 = [&](uint32_t i, float (&c)[8]) {
    load8_any<AL>(p.next_weight, p.weight_type, i, H, c);
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] += p.weight_offset;
  };
  auto make_c2 = [&](uint32_t i, float (&c)[8]) {
    float g[8];
    if (post) load8_any<AL>(p.post_weight, p.weight_type, i, H, c);
    if (kind == GATE_CHANNEL) load8_any<AL>(p.gate, p.gate_type, i, H, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = (post ? c[k] + p.weight_offset : 1.0f) * (kind == GATE_CHANNEL ? g[k] : 1.0f);
  };
  if constexpr (LDSC) {
    for (uint32_t i = (threadIdx.y * blockDim.x + threadIdx.x) * 8; i < H; i += blockDim.x * R * 8) {
      float c[8];
      if (next) {
        make_c1(i, c);
        store8<RT_F32, true>(dyn, i, H8, c);
      }
      if (has_y) {
        make_c2(i, c);
        store8<RT_F32, true>(dyn + H8, i, H8, c);
      }
    }
    __syncthreads();
  }
  auto c1_at = [&](uint32_t i, float (&c)[8]) {
    if constexpr (LDSC) load8<RT_F32, true>(dyn, i, H8, c);
    else make_c1(i, c);
  };
  auto c2_at = [&](uint32_t i, float (&c)[8]) {
    if constexpr (LDSC) load8<RT_F32, true>(dyn + H8, i, H8, c);
    else make_c2(i, c);
  };
  float an[C][8], ap[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int k = 0; k < 8; ++k) an[c][k] = ap[c][k] = 0.0f;
  int side = 0;
  for (int64_t t0 = (int64_t)blockIdx.x * R; t0 < p.T; t0 += (int64_t)gridDim.x * R, side ^= 1) {
    const int64_t t = t0 + own_row();
    const bool row = t < p.T;
    Raw8<YT> yr[C], gr[C], zr[C];
    Raw8<RT> hr[C], dr[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t i = piece(c);
      if (!row || i >= H) continue;
      if (next) {
        zr[c] = load_raw8<YT, AL>(static_cast<const uint8_t*>(d.g_z) + t * d.ldgz * rt_size(YT), i, H);
        hr[c] = load_raw8<RT, AL>(static_cast<const uint8_t*>(p.h) + t * p.ldh * rt_size(RT), i, H);
      }
      if (d.g_h) dr[c] = load_raw8<RT, AL>(static_cast<const uint8_t*>(d.g_h) + t * d.ldgh * rt_size(RT), i, H);
      if (has_y) yr[c] = load_raw8<YT, AL>(static_cast<const uint8_t*>(p.y) + t * p.ldy * rt_size(YT), i, H);
      if (kind == GATE_FULL)
        gr[c] = load_raw8<YT, AL>(static_cast<const uint8_t*>(p.gate) + t * p.ldg * rt_size(YT), i, H);
    }
    const float rh = next && row ? p.rstd_h[t] : 0.0f, ry = post && row ? p.rstd_y[t] : 1.0f;
    const float gt = kind == GATE_TOKEN && row ? one_any(p.gate, p.gate_type, t) : 1.0f;
    float s1[1] = {0.0f};
    if (next) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t i = piece(c);
        if (!row || i >= H) continue;
        float q[8], n[8], w[8];
        raw8_values<YT>(zr[c], q);
        raw8_values<RT>(hr[c], n);
        c1_at(i, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float m = q[k] * (n[k] * rh);
          an[c][k] += m;
          s1[0] += m * w[k];
        }
      }
      row_sums<1>(s1, red1[side], W);
      s1[0] *= invH;
    }
    float g[C][8];  // H'
    float s2[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t i = piece(c);
      if (!row || i >= H) continue;
      float v[8], w[8];
      if (next) {
        float q[8];
        raw8_values<YT>(zr[c], q);
        raw8_values<RT>(hr[c], v);
        c1_at(i, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[c][k] = rh * (q[k] * w[k] - v[k] * rh * s1[0]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) g[c][k] = 0.0f;
      }
      if (d.g_h) {
        raw8_values<RT>(dr[c], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[c][k] += v[k];
      }
      if (d.d_residual) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p.residual_scale * g[c][k];
        store8<RT, AL>(static_cast<uint8_t*>(d.d_residual) + t * H * rt_size(RT), i, H, v);
      }
      if (!has_y) continue;
      float b[8];
      raw8_values<YT>(yr[c], b);
      c2_at(i, w);
      if (kind == GATE_FULL) raw8_values<YT>(gr[c], v);
      float dg[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float u = g[c][k] * (b[k] * ry);
        const float gate = kind == GATE_FULL ? v[k] : gt;  // (a gate per channel is in w)
        ap[c][k] += gate * u;
        dg[k] = p.scale * u * w[k];
        s2[0] += gate * u * w[k];
        s2[1] += dg[k];
      }
      if (kind == GATE_FULL && d.d_gate)
        store8<YT, AL>(static_cast<uint8_t*>(d.d_gate) + t * H * rt_size(YT), i, H, dg);
    }
    if (!has_y) continue;
    const bool token = kind == GATE_TOKEN && d.d_gate;
    if (post || token) row_sums<2>(s2, red2[side], W);
    if (token && row && threadIdx.x == 0) {
      if (p.gate_type == RT_BF16) static_cast<uint16_t*>(d.d_gate)[t] = f32_to_bf16(s2[1]);
      else if (p.gate_type == RT_F32) static_cast<float*>(d.d_gate)[t] = s2[1];
      else static_cast<_Float16*>(d.d_gate)[t] = (_Float16)s2[1];
    }
    if (!d.d_y) continue;
    const float off = post ? s2[0] * invH : 0.0f, by = p.scale * ry;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t i = piece(c);
      if (!row || i >= H) continue;
      float b[8], w[8], v[8];
      raw8_values<YT>(yr[c], b);
      c2_at(i, w);
      if (kind == GATE_FULL) raw8_values<YT>(gr[c], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float gate = kind == GATE_FULL ? v[k] : gt;
        const float q = gate * (g[c][k] * w[k]);
        g[c][k] = by * (post ? q - b[k] * ry * off : q);
      }
      store8<YT, AL>(static_cast<uint8_t*>(d.d_y) + t * H * rt_size(YT), i, H, g[c]);
    }
  }
  if (!parts) return;
  float* out = parts + (int64_t)blockIdx.x * 2 * H;
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) {
    if (k2 == 0 ? !(next && d.d_next_weight) : !has_y) continue;
    float (&a)[C][8] = k2 == 0 ? an : ap;
    for (int r = 1; r < R; ++r) {  // the other rows' sums, one row after the other
      __syncthreads();
      if ((int)threadIdx.y == r)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (piece(c) < H) store8<RT_F32, true>(dyn, piece(c), H8, a[c]);
      __syncthreads();
      if (threadIdx.y == 0)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (piece(c) < H) {
            float v[8];
            load8<RT_F32, true>(dyn, piece(c), H8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) a[c][k] += v[k];
          }
    }
    if (threadIdx.y == 0)
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (piece(c) < H) store8<RT_F32, AL>(out + k2 * H, piece(c), H, a[c]);
  }
}

// Columns 64 x .. of sum y: parts of all workgroups, 16 at a time, then across
// them, and the factors of the two gradients that the second is for
__global__ __launch_bounds__(1024) void block_join_kernel(const float* parts, int groups, const qmoe_block_desc p,
                                                          const qmoe_block_grads d) {
  __shared__ float s[16][64];
  const int k2 = blockIdx.y, c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const bool post = p.y && p.post_weight, channel = p.gate_kind == GATE_CHANNEL;
  if (k2 == 0 ? !d.d_next_weight : !((post && d.d_post_weight) || (channel && d.d_gate))) return;
  const int64_t i = (int64_t)blockIdx.x * 64 + c;
  float v = 0.0f;
  if (i < p.H) {
#pragma unroll 8
    for (int g = r; g < groups; g += 16) v += parts[((int64_t)g * 2 + k2) * p.H + i];
  }
  s[r][c] = v;
  __syncthreads();
  if (r || i >= p.H) return;
  for (int k = 1; k < 16; ++k) v += s[k][c];
  auto put = [&](void* out, int type, float x) {
    if (type == RT_BF16) static_cast<uint16_t*>(out)[i] = f32_to_bf16(x);
    else if (type == RT_F32) static_cast<float*>(out)[i] = x;
    else static_cast<_Float16*>(out)[i] = (_Float16)x;
  };
  if (k2 == 0) return put(d.d_next_weight, p.weight_type, v);
  v *= p.scale;
  if (post && d.d_post_weight) put(d.d_post_weight, p.weight_type, v * (channel ? one_any(p.gate, p.gate_type, i) : 1.0f));
  if (channel && d.d_gate)
    put(d.d_gate, p.gate_type, v * (post ? p.weight_offset + one_any(p.post_weight, p.weight_type, i) : 1.0f));
}

// ---------------------------------------------------------------- launches

struct BlockShape {
  int pieces, waves, rows;
};

// pieces of 8 per lane, wavefronts of a row, rows of a workgroup. Rows of up to 8
// wavefronts, then (forward) two pieces per lane, or (gradient, whose sums take
// registers) up to 16 wavefronts. 8192 rows of 7168 bf16, one / two pieces: forward
// 115 / 98 us, gradient 160 / 167.
BlockShape block_shape(int64_t H, bool grad) {
  const int64_t chunks = cdiv<int64_t>(H, 8);
  const int C = chunks <= (grad ? 1024 : 512) ? 1 : 2;
  const int W = (int)cdiv<int64_t>(chunks, 64 * C);
  return {C, W, W > 8 ? 1 : 8 / W};
}

// workgroups of the gradient: two per CU, one of more than 8 wavefronts. Each adds its rows
// one after the other: T / (512 rows of a workgroup) float32 additions in a chain, 16 of 8192
// rows of 4096, 8192 of the 2^24 rows of 1024 that a call may have.
int grad_groups(int64_t T, BlockShape s) {
  const int64_t g = cdiv<int64_t>(T, s.rows), most = s.waves > 8 ? 256 : 512;
  return (int)(g < most ? g : most);
}

bool aligned16(const void* p, int64_t ld, int size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0);
}

// whether rows and vectors are read and written 16 bytes at a time
bool wide(const qmoe_block_desc* p) {
  const int ys = rt_size(p->y_type), rs = rt_size(p->residual_type);
  bool ok = p->H % 8 == 0 && aligned16(p->y, p->ldy, ys) && aligned16(p->residual, p->ldr, rs) &&
            aligned16(p->h, p->ldh, rs) && aligned16(p->z, p->ldz, ys) && aligned16(p->post_weight, 0, 1) &&
            aligned16(p->next_weight, 0, 1);
  if (p->gate_kind == GATE_FULL) ok = ok && aligned16(p->gate, p->ldg, ys);
  if (p->gate_kind == GATE_CHANNEL) ok = ok && aligned16(p->gate, 0, 1);
  return ok;
}

int check(const qmoe_block_desc* p) {
  if (!p || p->T < 1 || p->T > kMaxRows || p->H < 1 || p->H > kMaxRow) return QMOE_ERR_ARG;
  if (p->y_type < 0 || p->y_type > 2 || p->residual_type < 0 || p->residual_type > 2 || p->weight_type < 0 ||
      p->weight_type > 2 || p->gate_type < 0 || p->gate_type > 2 || p->gate_kind < 0 || p->gate_kind > GATE_FULL)
    return QMOE_ERR_ARG;
  // the residual is of the block's type or float32
  if (p->residual_type != p->y_type && p->residual_type != RT_F32) return QMOE_ERR_ARG;
  if (!p->y && (p->post_weight || p->gate_kind || !p->next_weight)) return QMOE_ERR_ARG;
  if (p->gate_kind && !p->gate) return QMOE_ERR_ARG;
  if (p->gate_kind == GATE_FULL && p->gate_type != p->y_type) return QMOE_ERR_ARG;
  if ((p->y && p->ldy < p->H) || (p->gate_kind == GATE_FULL && p->ldg < p->H)) return QMOE_ERR_ARG;
  return QMOE_OK;
}

// the instance for the types, pieces and alignment
template <int YT, int RT, typename F>
void with_pieces(BlockShape s, bool al, F&& f) {
#define QMOE_BLOCK(CC, TH)                                                                                         \
  if (al) f(std::integral_constant<int, YT>(), std::integral_constant<int, RT>(), std::integral_constant<int, CC>(), \
            std::integral_constant<int, TH>(), std::true_type());                                                  \
  else f(std::integral_constant<int, YT>(), std::integral_constant<int, RT>(), std::integral_constant<int, CC>(),   \
         std::integral_constant<int, TH>(), std::false_type())
  if (s.pieces == 1 && s.waves <= 8) QMOE_BLOCK(1, 512);
  else if (s.pieces == 1) QMOE_BLOCK(1, 1024);
  else if (s.waves <= 8) QMOE_BLOCK(2, 512);
  else QMOE_BLOCK(2, 1024);
#undef QMOE_BLOCK
}
template <typename F>
void with_types(int yt, int rt, BlockShape s, bool al, F&& f) {
  if (yt == RT_F32) with_pieces<RT_F32, RT_F32>(s, al, f);
  else if (yt == RT_BF16 && rt == RT_BF16) with_pieces<RT_BF16, RT_BF16>(s, al, f);
  else if (yt == RT_BF16) with_pieces<RT_BF16, RT_F32>(s, al, f);
  else if (rt == RT_F16) with_pieces<RT_F16, RT_F16>(s, al, f);
  else with_pieces<RT_F16, RT_F32>(s, al, f);
}

}  // namespace

// See include/qmoe.h for the contract.
extern "C" int qmoe_block_residual(const qmoe_block_desc* p, hipStream_t stream) {
  if (const int st = check(p)) return st;
  if (!p->residual || p->ldr < p->H || (p->y && (!p->h || p->ldh < p->H)) ||
      (p->next_weight && (!p->z || p->ldz < p->H)))
    return QMOE_ERR_ARG;
  const BlockShape s = block_shape(p->H, false);
  const dim3 grid = row_groups(cdiv<int64_t>(p->T, s.rows)), block(64 * s.waves, s.rows);
  with_types(p->y_type, p->residual_type, s, wide(p), [&](auto yt, auto rt, auto c, auto th, auto al) {
    if constexpr (th() == 512 || c() == 2)  // (one piece and more than 8 wavefronts: the gradient's)
      hipLaunchKernelGGL((block_residual_kernel<yt(), rt(), c(), th(), al()>), grid, block, 0, stream, *p);
  });
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_block_residual_grad_workspace_size(int64_t T, int64_t H, int64_t* bytes) {
  if (T < 1 || T > kMaxRows || H < 1 || H > kMaxRow || !bytes) return QMOE_ERR_ARG;
  *bytes = (int64_t)grad_groups(T, block_shape(H, true)) * 2 * H * 4;
  return QMOE_OK;
}

extern "C" int qmoe_block_residual_grad(const qmoe_block_desc* p, const qmoe_block_grads* d, void* workspace,
                                        int64_t ws_bytes, hipStream_t stream) {
  if (const int st = check(p)) return st;
  if (!d || (!d->g_h && !d->g_z) || (d->g_z && !p->next_weight)) return QMOE_ERR_ARG;
  // (outputs of operands that are not there, or that no gradient reaches)
  if ((d->d_next_weight && !d->g_z) || (d->d_y && !p->y) || (d->d_gate && !p->gate_kind) ||
      (d->d_post_weight && !p->post_weight))
    return QMOE_ERR_ARG;
  const bool next = d->g_z != nullptr, post = p->y && p->post_weight;
  if (next && (!p->h || p->ldh < p->H || !p->rstd_h || d->ldgz < p->H)) return QMOE_ERR_ARG;
  if (post && !p->rstd_y) return QMOE_ERR_ARG;
  if (d->g_h && d->ldgh < p->H) return QMOE_ERR_ARG;
  const bool sums = (next && d->d_next_weight) || (post && d->d_post_weight) ||
                    (p->gate_kind == GATE_CHANNEL && d->d_gate);
  const BlockShape s = block_shape(p->H, true);
  const int groups = grad_groups(p->T, s);
  if (sums && (!workspace || !aligned16(workspace, 0, 1) || ws_bytes < (int64_t)groups * 2 * p->H * 4))
    return QMOE_ERR_WORKSPACE;
  const int ys = rt_size(p->y_type), rs = rt_size(p->residual_type);
  const bool al = wide(p) && aligned16(d->g_h, d->ldgh, rs) && aligned16(d->g_z, d->ldgz, ys) &&
                  aligned16(d->d_y, p->H, ys) && aligned16(d->d_residual, p->H, rs) &&
                  (p->gate_kind != GATE_FULL || aligned16(d->d_gate, p->H, ys));
  const dim3 block(64 * s.waves, s.rows);
  float* parts = sums ? static_cast<float*>(workspace) : nullptr;
  const bool lds = p->H <= kMaxLdsRow;
  const size_t dyn = (lds ? 8 : s.rows > 1 ? 4 : 0) * (size_t)(cdiv<int64_t>(p->H, 8) * 8);
  with_types(p->y_type, p->residual_type, s, al, [&](auto yt, auto rt, auto c, auto th, auto a) {
    constexpr bool kLds = c() == 1;  // (rows of up to 8192)
    if constexpr (th() == 512 && c() == 2) {
      return;  // (the forward's)
    } else {
      if (a() && next && post)
        hipLaunchKernelGGL((block_residual_grad_kernel<yt(), rt(), c(), th(), a(), a() ? 1 : 0, kLds>), dim3(groups), block,
                           dyn, stream, *p, *d, parts);
      else if (a() && next && !p->y)
        hipLaunchKernelGGL((block_residual_grad_kernel<yt(), rt(), c(), th(), a(), a() ? 2 : 0, kLds>), dim3(groups), block,
                           dyn, stream, *p, *d, parts);
      else
        hipLaunchKernelGGL((block_residual_grad_kernel<yt(), rt(), c(), th(), a(), 0, kLds>), dim3(groups), block, dyn,
                           stream, *p, *d, parts);
    }
  });
  if (sums)
    hipLaunchKernelGGL(block_join_kernel, dim3((unsigned)cdiv<int64_t>(p->H, 64), 2), dim3(1024), 0, stream, parts, groups,
                       *p, *d);
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
