// A whole MoE layer for a few tokens (1..16) in two launches: routing, gate_up
// with its activation, down and the weighted sum.
//
//   s = score(logits), (w, e) = top k of s (moe_route.h's rule, float32 weights)
//   h[t, j]  = bf16(act(W13[e] x[t] + b13[e]))          j < k, e = e[t, j]
//   out[t]   = bf16(sum over j of w[t, j] (W2[e] h[t, j] + b2[e]))
//
// What bounds it: the touched experts' weights, read once each from HBM; at one
// token the launches and the routing's latency weigh as much.
//
//  * Launch 1: every workgroup routes the tokens itself (a few microseconds
//    that replace a launch and its result's way through memory), then takes its
//    share of the (active expert, 16 gate rows + their 16 up rows) items.
//    Launch 2: a workgroup owns 16 output columns and walks the active
//    experts, so that the weighted sum stays in registers.
//  * Weights are read in granules of 16 rows x 64 bytes, a wavefront's load
//    instruction each (4 adjacent lanes per row segment), and turned into MFMA
//    operand order through 1 KB of LDS per granule; the K axis is dealt to
//    the wavefronts in pairs of granules (one 128-byte line per row), several
//    steps in flight per wavefront. Tokens are the other MFMA operand's 16
//    columns; a column without a token loads nothing, and what it holds stays
//    in its column.
//  * Sums are float32: per wavefront, then over the wavefronts in order; in
//    launch 2 over the experts in ascending order per wavefront.

#include <algorithm>

#include "../../include/qmoe.h"
#include "gemm_tile.h"
#include "moe_route.h"
#include "stream_load.h"

namespace {

enum { FF_MX = 0, FF_NV = 1, FF_I4 = 2, FF_F8 = 3, FF_BF = 4 };

constexpr int kFewTokens = 16, kFewRoutes = 128, kFewExperts = 512;

struct FewParams {
  const uint16_t* x;  // bf16 [T][ldx]
  int64_t ldx;
  int T, H, I, E, topk;
  const void* logits;
  int logits_f32, scoring, grouped, renormalize, num_group, topk_group, skip;
  const float* correction;
  float rsf;
  const uint8_t *w1, *w2;  // [E][2I][H], [E][H][I]
  const void *s1, *s2;     // scales
  const float *b1, *b2;    // [E][2I], [E][H] or nullptr
  int act;
  float act_p0, act_p1;
  int group_shift;  // FF_I4: log2 of the k per scale
  uint16_t* h;      // bf16 [T topk][I]
  int32_t* ids;     // [T topk] routes of launch 1
  float* wts;
  uint16_t* out;    // bf16 [T][ldo]
  int64_t ldo;
};

// One format: codes per 16-byte chunk, bytes per row of K
template <int F>
struct Fmt {
  static constexpr int kCodes = F == FF_F8 ? 16 : (F == FF_BF ? 8 : 32);
  static constexpr int kMfma = kCodes / 8;  // 16x16x32 MFMAs per granule
  QMOE_HD static int row_bytes(int K) { return F == FF_BF ? 2 * K : (F == FF_F8 ? K : K / 2); }
  // bytes of a row's scales
  QMOE_HD static int scale_bytes(int K, int group_shift) {
    return F == FF_MX ? K / 32 : (F == FF_NV ? K / 8 : (F == FF_I4 ? (K >> group_shift) * 2 : (F == FF_F8 ? K / 32 : 0)));
  }
};

using qmoe_stream::kOob;
using qmoe_stream::make_rsrc;
using qmoe_stream::rsrc_t;

// One step of a wavefront: NT granules (16 rows x 64 bytes each), their
// scales and the tokens' values at the same k
template <int F, int NT>
struct Step {
  uint4 w[NT];
  uint32_t s[NT];
  uint4 x[Fmt<F>::kMfma];
};

__device__ __forceinline__ uint4 load16(rsrc_t r, uint32_t off) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// The scale word of the lane's chunk (row r = lane & 15, chunk c of its row)
template <int F>
__device__ __forceinline__ uint32_t load_scale(rsrc_t r, uint32_t row_off, int c, int group_shift, bool in) {
  if constexpr (F == FF_MX) return __builtin_amdgcn_raw_buffer_load_b8(r, in ? row_off + c : kOob, 0, 0);
  else if constexpr (F == FF_NV) return __builtin_amdgcn_raw_buffer_load_b32(r, in ? row_off + c * 4 : kOob, 0, 0);
  else if constexpr (F == FF_I4) return __builtin_amdgcn_raw_buffer_load_b16(r, in ? row_off + ((c * 32) >> group_shift) * 2 : kOob, 0, 0);
  else if constexpr (F == FF_F8) return __builtin_amdgcn_raw_buffer_load_b32(r, in ? row_off + (c >> 3) * 4 : kOob, 0, 0);
  else return 0;
}

union Bf8 {
  uint4 u;
  bf16x8 v;
};

__device__ __forceinline__ uint4 e2m1x8_to_bf16(uint32_t d, float scale) {
  union {
    bf16x2 h[4];
    uint4 u;
  } r;
  r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 0);
  r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 1);
  r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 2);
  r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 3);
  return r.u;
}

// 8 e4m3 codes (two dwords) times a float32 scale, each rounded once to bf16
__device__ __forceinline__ uint4 e4m3x8_to_bf16(uint32_t a, uint32_t b, float s) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f f0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)a, false), f1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)a, true);
  const v2f f2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, false), f3 = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, true);
  union {
    bf16x2 h[4];
    uint4 u;
  } r;
  r.h[0] = __builtin_convertvector(f32x2{f0[0] * s, f0[1] * s}, bf16x2);
  r.h[1] = __builtin_convertvector(f32x2{f1[0] * s, f1[1] * s}, bf16x2);
  r.h[2] = __builtin_convertvector(f32x2{f2[0] * s, f2[1] * s}, bf16x2);
  r.h[3] = __builtin_convertvector(f32x2{f3[0] * s, f3[1] * s}, bf16x2);
  return r.u;
}

// The i-th 8 codes of a 16-byte chunk as bf16
template <int F>
__device__ __forceinline__ uint4 expand8(const uint4& c, int i, uint32_t s) {
  const uint32_t d[4] = {c.x, c.y, c.z, c.w};
  if constexpr (F == FF_MX) return e2m1x8_to_bf16(d[i], e8m0_to_f32(s));
  else if constexpr (F == FF_NV) return nvfp4x8_to_bf16(d[i], bf16_to_f32((uint16_t)(i < 2 ? s : s >> 16)));
  else if constexpr (F == FF_I4) return int4x8_to_bf16(d[i], bf16_to_f32((uint16_t)s));
  else if constexpr (F == FF_F8) return e4m3x8_to_bf16(d[2 * i], d[2 * i + 1], bits_f32(s));
  else return c;
}

// acc[t] += granule t . tokens. `tr`: this wavefront's LDS, NT KB. Row r's
// 16-byte chunk c lies at slot c ^ (r / 4), so that neither the writes (4
// chunks of a row by 4 adjacent lanes) nor the reads (one chunk of 16 rows)
// meet in a bank.
template <int F, int NT>
__device__ __forceinline__ void consume(const Step<F, NT>& st, uint4* tr, f32x4 (&acc)[NT]) {
  const int lane = threadIdx.x & 63, wr = lane >> 2, r = lane & 15, kg = lane >> 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) tr[t * 64 + wr * 4 + ((lane & 3) ^ (wr >> 2))] = st.w[t];
  qmoe_moe::wave_lds_sync();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint4 c = tr[t * 64 + r * 4 + (kg ^ (r >> 2))];
#pragma unroll
    for (int i = 0; i < Fmt<F>::kMfma; ++i) {
      Bf8 a, b;
      a.u = expand8<F>(c, i, st.s[t]);
      b.u = st.x[i];
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc[t], 0, 0, 0);
    }
  }
  qmoe_moe::wave_lds_sync();  // the slots are free for the next step
}

// The routes of the tokens and what follows from them, in LDS
struct FewRoutes {
  int32_t ids[kFewRoutes];
  float w[kFewRoutes];
  uint32_t mask[kFewExperts / 32];  // experts with a route
  int16_t active[kFewRoutes];       // experts with a route, ascending
  int16_t route[kFewRoutes][kFewTokens];  // (active slot, token) -> route or -1
  int num;                          // active experts
};

// From ids / w (visible to the workgroup) to the rest; every thread calls
__device__ __forceinline__ void few_active(FewRoutes& s, const FewParams& p) {
  const int tid = threadIdx.x, R = p.T * p.topk;
  auto valid = [&](int r) {
    const int id = s.ids[r];
    return id >= 0 && id < p.E && !(p.skip && (f32_to_bf16(s.w[r]) & 0x7fffu) == 0);
  };
  if (tid < kFewExperts / 32) s.mask[tid] = 0;
  for (int i = tid; i < kFewRoutes * kFewTokens; i += blockDim.x) (&s.route[0][0])[i] = -1;
  __syncthreads();
  if (tid < R && valid(tid)) atomicOr(&s.mask[s.ids[tid] >> 5], 1u << (s.ids[tid] & 31));
  __syncthreads();
  if (tid < R && valid(tid)) {
    const int id = s.ids[tid];
    int slot = __popc(s.mask[id >> 5] & ((1u << (id & 31)) - 1u));
    for (int i = 0; i < (id >> 5); ++i) slot += __popc(s.mask[i]);
    s.active[slot] = (int16_t)id;
    s.route[slot][tid / p.topk] = (int16_t)tid;
  }
  if (tid == 0) {
    int n = 0;
    for (int i = 0; i < kFewExperts / 32; ++i) n += __popc(s.mask[i]);
    s.num = n;
  }
  __syncthreads();
}

// The wavefront's i-th granule of a row of `granules`: pairs dealt in turn
template <int NW>
__device__ __forceinline__ int granule_of(int wave, int i) { return (i >> 1) * 2 * NW + wave * 2 + (i & 1); }

constexpr int kUpWaves = 4, kUpAhead = 4;

template <int F, int S>
__global__ __launch_bounds__(kUpWaves * 64) void few_up_kernel(const FewParams p) {
  __shared__ FewRoutes s;
  __shared__ float choice[kUpWaves][qmoe_route::kChoiceLds];
  __shared__ __align__(16) uint4 tr[kUpWaves][2 * 64];
  __shared__ __align__(16) f32x4 red[kUpWaves][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = p.T * p.topk;
  for (int t = wave; t < p.T; t += kUpWaves)
    qmoe_route::route_token_any<S>(p.scoring, p.grouped, p.logits, p.logits_f32, t, p.E, p.topk, p.correction,
                                   p.renormalize, p.rsf, p.num_group, p.topk_group, s.w, s.ids, choice[wave], nullptr,
                                   nullptr, 1);
  __syncthreads();
  if (blockIdx.x == 0 && tid < R) {
    p.ids[tid] = s.ids[tid];
    p.wts[tid] = s.w[tid];
  }
  few_active(s, p);

  const int tiles = p.I / 16, items = __builtin_amdgcn_readfirstlane(s.num) * tiles;
  const int it0 = (int)((int64_t)blockIdx.x * items / gridDim.x), it1 = (int)((int64_t)(blockIdx.x + 1) * items / gridDim.x);
  if (it0 >= it1) return;
  const int rb = Fmt<F>::row_bytes(p.H), sb = Fmt<F>::scale_bytes(p.H, p.group_shift), granules = (rb + 63) / 64;
  // steps per item, the same for every wavefront (those past a row's end load
  // nothing and add zeros)
  const int chunks = (cdiv(granules, 2 * kUpWaves) * 2 + kUpAhead - 1) / kUpAhead;
  const int r = lane & 15, kg = lane >> 4;
  const rsrc_t xr = make_rsrc(p.x, (int64_t)p.T * p.ldx * 2);

  // where the loads are: item, chunk of it
  rsrc_t wr[2], sr[2];
  uint32_t xrow = kOob;  // byte offset of the lane's token row
  auto seek = [&](int item) {
    const int slot = item / tiles, tile = item - slot * tiles;
    const int e = __builtin_amdgcn_readfirstlane(s.active[slot]);
    const int route = s.route[slot][r];  // column r: token r, where it takes this expert
    xrow = route >= 0 ? (uint32_t)(r * p.ldx * 2) : kOob;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = (int64_t)e * 2 * p.I + t * p.I + tile * 16;
      wr[t] = make_rsrc(p.w1 + row * rb, (int64_t)16 * rb);
      sr[t] = make_rsrc(static_cast<const uint8_t*>(p.s1) + row * sb, (int64_t)16 * sb);
    }
  };
  Step<F, 2> st[kUpAhead];
  auto issue = [&](Step<F, 2>& d, int i, bool live) {
    const int g = granule_of<kUpWaves>(wave, i);
    const int lc = g * 4 + (lane & 3), mc = g * 4 + kg;  // chunk of the row: as loaded, as multiplied
    const bool lin = live && lc * 16 < rb, min_ = live && mc * 16 < rb;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      d.w[t] = load16(wr[t], lin ? (uint32_t)((lane >> 2) * rb + lc * 16) : kOob);
      d.s[t] = load_scale<F>(sr[t], (uint32_t)(r * sb), mc, p.group_shift, min_);
    }
#pragma unroll
    for (int k = 0; k < Fmt<F>::kMfma; ++k)
      d.x[k] = load16(xr, min_ ? xrow + (uint32_t)((mc * Fmt<F>::kCodes + k * 8) * 2) : kOob);
  };
  seek(it0);
#pragma unroll
  for (int u = 0; u < kUpAhead; ++u) issue(st[u], u, true);
  for (int item = it0; item < it1; ++item) {
    f32x4 acc[2] = {};
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 < chunks, next = item + 1 < it1;
      if (!more && next) seek(item + 1);
#pragma unroll
      for (int u = 0; u < kUpAhead; ++u) {
        consume<F, 2>(st[u], tr[wave], acc);
        issue(st[u], (more ? (c + 1) * kUpAhead : 0) + u, more || next);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // sums of the wavefronts in order, bias, activation
    red[wave][0][lane] = acc[0];
    red[wave][1][lane] = acc[1];
    stage_barrier();
    if (wave == 0) {
      const int slot = item / tiles, n0 = (item - slot * tiles) * 16 + kg * 4;
      const int route = s.route[slot][r];
      f32x4 g = red[0][0][lane], u = red[0][1][lane];
#pragma unroll
      for (int w = 1; w < kUpWaves; ++w) {
        g += red[w][0][lane];
        u += red[w][1][lane];
      }
      if (route >= 0) {
        if (p.b1) {
          const float* b = p.b1 + (int64_t)s.active[slot] * 2 * p.I + n0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            g[q] += b[q];
            u[q] += b[p.I + q];
          }
        }
        uint16_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = f32_to_bf16(qmoe_act(p.act, g[q], u[q], p.act_p0, p.act_p1));
        *reinterpret_cast<uint2*>(p.h + (int64_t)route * p.I + n0) =
            make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
      }
    }
    stage_barrier();  // the sums have been read
  }
}

constexpr int kDownWaves = 8, kDownAhead = 6;

template <int F>
__global__ __launch_bounds__(kDownWaves * 64) void few_down_kernel(const FewParams p) {
  __shared__ FewRoutes s;
  __shared__ __align__(16) uint4 tr[kDownWaves][64];
  __shared__ __align__(16) f32x4 red[kDownWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = p.T * p.topk;
  if (tid < R) {
    s.ids[tid] = p.ids[tid];
    s.w[tid] = p.wts[tid];
  }
  few_active(s, p);
  const int num = __builtin_amdgcn_readfirstlane(s.num), n0 = blockIdx.x * 16;
  const int rb = Fmt<F>::row_bytes(p.I), sb = Fmt<F>::scale_bytes(p.I, p.group_shift), granules = (rb + 63) / 64;
  const int r = lane & 15, kg = lane >> 4;
  const rsrc_t hr = make_rsrc(p.h, (int64_t)R * p.I * 2);

  // the wavefront's i-th step is granule granule_of(wave, i) of all experts' rows
  // laid end to end
  const int total = num * granules;
  struct At {
    int slot, g;
  };
  auto at = [&](int i) {
    const int L = granule_of<kDownWaves>(wave, i), slot = L / granules;
    return At{slot, L - slot * granules};
  };
  Step<F, 1> st[kDownAhead];
  auto issue = [&](Step<F, 1>& d, int i) {
    const At a = at(i);
    const bool live = a.slot < num;
    const int e = live ? __builtin_amdgcn_readfirstlane(s.active[a.slot]) : 0;
    const int route = live ? s.route[a.slot][r] : -1;
    const int64_t row = (int64_t)e * p.H + n0;
    const rsrc_t wr = make_rsrc(p.w2 + row * rb, (int64_t)16 * rb);
    const rsrc_t sr = make_rsrc(static_cast<const uint8_t*>(p.s2) + row * sb, (int64_t)16 * sb);
    const int lc = a.g * 4 + (lane & 3), mc = a.g * 4 + kg;
    const bool lin = live && lc * 16 < rb, min_ = live && mc * 16 < rb;
    d.w[0] = load16(wr, lin ? (uint32_t)((lane >> 2) * rb + lc * 16) : kOob);
    d.s[0] = load_scale<F>(sr, (uint32_t)(r * sb), mc, p.group_shift, min_);
#pragma unroll
    for (int k = 0; k < Fmt<F>::kMfma; ++k)
      d.x[k] = load16(hr, min_ && route >= 0 ? (uint32_t)(((int64_t)route * p.I + mc * Fmt<F>::kCodes + k * 8) * 2) : kOob);
  };
  f32x4 sum = {}, acc[1] = {};
  auto flush = [&](int slot) {
    const int route = s.route[slot][r];
    const float w = route >= 0 ? s.w[route] : 0.0f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (route >= 0) sum[q] += w * acc[0][q];
      acc[0][q] = 0.0f;
    }
  };
#pragma unroll
  for (int u = 0; u < kDownAhead; ++u) issue(st[u], u);
  int slot = -1;
  for (int i0 = 0; granule_of<kDownWaves>(wave, i0) < total; i0 += kDownAhead) {
#pragma unroll
    for (int u = 0; u < kDownAhead; ++u) {
      const At a = at(i0 + u);
      if (a.slot < num) {
        if (a.slot != slot && slot >= 0) flush(slot);
        slot = a.slot;
        consume<F, 1>(st[u], tr[wave], acc);
      }
      issue(st[u], i0 + u + kDownAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (slot >= 0) flush(slot);
  if (p.b2)
    for (int k = wave; k < num; k += kDownWaves) {
      const int route = s.route[k][r];
      const float* b = p.b2 + (int64_t)s.active[k] * p.H + n0 + kg * 4;
      if (route >= 0)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += s.w[route] * b[q];
    }
  red[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && r < p.T) {
    f32x4 v = red[0][lane];
#pragma unroll
    for (int w = 1; w < kDownWaves; ++w) v += red[w][lane];
    uint16_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = f32_to_bf16(v[q]);
    *reinterpret_cast<uint2*>(p.out + (int64_t)r * p.ldo + n0 + kg * 4) =
        make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
  }
}

template <int F, int S>
void launch_up(const FewParams& p, hipStream_t st) {
  const int64_t items = (int64_t)std::min(p.E, p.T * p.topk) * (p.I / 16);
  hipLaunchKernelGGL((few_up_kernel<F, S>), dim3((unsigned)std::min<int64_t>(items, 768)), dim3(kUpWaves * 64), 0, st, p);
}

template <int F>
void launch_few(const FewParams& p, hipStream_t st) {
  const int S = qmoe_route::route_slots(p.E);
  if (S <= 2) launch_up<F, 2>(p, st);
  else if (S == 4) launch_up<F, 4>(p, st);
  else launch_up<F, 8>(p, st);
  hipLaunchKernelGGL((few_down_kernel<F>), dim3((unsigned)(p.H / 16)), dim3(kDownWaves * 64), 0, st, p);
}

int64_t few_layout(int64_t R, int64_t I, int64_t (&off)[3]) {
  off[0] = 0;
  off[1] = (R * I * 2 + 255) / 256 * 256;
  off[2] = off[1] + (R * 4 + 255) / 256 * 256;
  return off[2] + (R * 4 + 255) / 256 * 256;
}

int few_ok(const qmoe_moe_few_desc* d) {
  if (!d || d->format < FF_MX || d->format > FF_BF) return 0;
  if (d->T < 1 || d->T > kFewTokens || d->E < 1 || d->E > kFewExperts) return 0;
  if (!qmoe_route::route_args_ok(d->T, d->E, d->topk, d->scoring, d->num_group, d->topk_group)) return 0;
  if ((int64_t)d->T * d->topk > kFewRoutes) return 0;
  if (d->H < 32 || d->H > 65536 || d->H % 32 || d->I < 32 || d->I > 65536 || d->I % 32) return 0;
  if (d->format == FF_I4 && ((d->group != 32 && d->group != 64 && d->group != 128) || d->H % d->group || d->I % d->group))
    return 0;
  if (d->format == FF_F8 && (d->H % 128 || d->I % 128)) return 0;
  if (d->act <= QMOE_ACT_NONE || d->act > QMOE_ACT_SITU) return 0;
  if (d->ldx < d->H || d->ldx % 8 || d->ldx >= (int64_t)1 << 26 || d->ldo < d->H || d->ldo % 4) return 0;
  return 1;
}

}  // namespace

// See include/qmoe.h for the contract.
extern "C" int qmoe_moe_few_workspace_size(const qmoe_moe_few_desc* d, int64_t* bytes) {
  if (!few_ok(d) || !bytes) return QMOE_ERR_ARG;
  int64_t off[3];
  *bytes = few_layout((int64_t)d->T * d->topk, d->I, off);
  return QMOE_OK;
}

extern "C" int qmoe_moe_few(const qmoe_moe_few_desc* d, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  if (!few_ok(d)) return QMOE_ERR_ARG;
  if (!d->x || !d->router_logits || !d->w1 || !d->w2 || !d->out) return QMOE_ERR_ARG;
  if ((d->format != FF_BF) != (d->w1_scale != nullptr) || (d->format != FF_BF) != (d->w2_scale != nullptr)) return QMOE_ERR_ARG;
  auto aligned = [](const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; };
  if (!aligned(d->x, 16) || !aligned(d->w1, 16) || !aligned(d->w2, 16) || !aligned(d->out, 8) ||
      !aligned(d->w1_scale, 4) || !aligned(d->w2_scale, 4) || !aligned(d->w1_bias, 4) || !aligned(d->w2_bias, 4))
    return QMOE_ERR_ARG;
  int64_t off[3];
  const int64_t R = (int64_t)d->T * d->topk;
  if (!workspace || ws_bytes < few_layout(R, d->I, off)) return QMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  FewParams p{};
  p.x = static_cast<const uint16_t*>(d->x);
  p.ldx = d->ldx;
  p.T = d->T, p.H = d->H, p.I = d->I, p.E = d->E, p.topk = d->topk;
  p.logits = d->router_logits;
  p.logits_f32 = d->logits_f32;
  p.scoring = d->scoring;
  p.grouped = d->num_group > 1 && d->topk_group < d->num_group;
  p.renormalize = d->renormalize;
  p.num_group = d->num_group, p.topk_group = d->topk_group;
  p.skip = d->skip_padded;
  p.correction = d->correction_bias;
  p.rsf = d->routed_scaling_factor;
  p.w1 = static_cast<const uint8_t*>(d->w1);
  p.w2 = static_cast<const uint8_t*>(d->w2);
  p.s1 = d->w1_scale, p.s2 = d->w2_scale;
  p.b1 = d->w1_bias, p.b2 = d->w2_bias;
  p.act = d->act, p.act_p0 = d->act_p0, p.act_p1 = d->act_p1;
  p.group_shift = d->format == FF_I4 ? __builtin_ctz(d->group) : 0;
  p.h = reinterpret_cast<uint16_t*>(ws + off[0]);
  p.ids = reinterpret_cast<int32_t*>(ws + off[1]);
  p.wts = reinterpret_cast<float*>(ws + off[2]);
  p.out = static_cast<uint16_t*>(d->out);
  p.ldo = d->ldo;
  switch (d->format) {
    case FF_MX: launch_few<FF_MX>(p, stream); break;
    case FF_NV: launch_few<FF_NV>(p, stream); break;
    case FF_I4: launch_few<FF_I4>(p, stream); break;
    case FF_F8: launch_few<FF_F8>(p, stream); break;
    default: launch_few<FF_BF>(p, stream); break;
  }
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
