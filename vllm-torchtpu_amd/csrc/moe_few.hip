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
//    share of the (slot, 16 gate rows + their 16 up rows) items; a slot is up to
//    kRows tokens of one expert (experts with more have several slots, which
//    read the weights again, from L2). Launch 2: a workgroup owns 16 output
//    columns and walks the slots, so that the weighted sum stays in registers.
//  * Weights are read as whole 128-byte lines of 16 rows, two load instructions
//    of 8 rows each, and turned into MFMA operand order through 2 KB of LDS per
//    wavefront. (64 bytes of 16 rows per instruction, the other half of each
//    line by the next one: the L1 stalled on pending lines 37 % of the time.)
//    The K axis is dealt to the wavefronts line by line, several in flight.
//  * A 16-byte chunk of 4-bit codes feeds four MFMAs, each with 8 tokens'
//    values per lane. The 16 columns of the other operand hold all four for
//    kRows = 4 tokens (column 4 r + i: token r's values for MFMA i) in one
//    load, instead of one load per MFMA; each MFMA has its own sums, of which
//    only its own columns count, and the four columns are added at the end.
//    (8-bit codes: two MFMAs, 8 tokens; bf16: one, 16.)
//  * Sums are float32: per wavefront, then over the wavefronts in order; in
//    launch 2 over the slots in ascending order per wavefront.
//  * Rounded to bf16 are the matrix cores' operands: h, and code x scale of the
//    4- and 8-bit formats (exact for MXFP4; the float32 scales of FP8 are
//    rounded to bf16 before the product), as in the other bf16-activation paths;
//    and out, once.
//
// Measured, launch 1 + 2, median (fastest) of 30: one token, MXFP4, 4 of 128 experts
// of 2880 x 2880 15.7 (15.4) + 8.8 (8.6) us; 16 tokens 121 (114) + 81 (73), 443 and 232
// MiB read, 3.8 and 3.0 TB/s (17 us of launch 1 are the routing of 16 tokens and
// latency, and launch 2 has 180 workgroups for 256 CUs); 8 tokens, NVFP4, 8 of 256
// experts of 2048 x 7168 211 (177) + 112 (93), 746 and 371 MiB, 3.7 and 3.5 TB/s, both
// in 272 to 297 us a call without the profiler.

#include <algorithm>

#include "../../include/qmoe.h"
#include "gemm_tile.h"
#include "moe_route.h"
#include "stream_load.h"

namespace {

enum { FF_MX = 0, FF_NV = 1, FF_I4 = 2, FF_F8 = 3, FF_BF = 4 };

constexpr int kFewTokens = 16, kFewRoutes = 128, kFewExperts = 512;

// What follows from the tokens' routes (route: t * topk + j)
struct FewTables {
  int32_t num;                             // slots
  float w[kFewRoutes];                     // route -> weight
  int16_t active[kFewRoutes];              // slot -> expert, ascending
  int16_t route[kFewRoutes * kFewTokens];  // (slot, row < kRows) -> route or -1, rows of a slot together
};

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
  FewTables* tables;  // from launch 1 to launch 2
  uint16_t* out;    // bf16 [T][ldo]
  int64_t ldo;
};

// One format: codes per 16-byte chunk, bytes per row of K
template <int F>
struct Fmt {
  static constexpr int kCodes = F == FF_F8 ? 16 : (F == FF_BF ? 8 : 32);
  static constexpr int kMfma = kCodes / 8;  // 16x16x32 MFMAs per chunk
  static constexpr int kRows = 16 / kMfma;  // tokens of a slot
  QMOE_HD static int row_bytes(int K) { return F == FF_BF ? 2 * K : (F == FF_F8 ? K : K / 2); }
  // bytes of a row's scales
  QMOE_HD static int scale_bytes(int K, int group_shift) {
    return F == FF_MX ? K / 32 : (F == FF_NV ? K / 8 : (F == FF_I4 ? (K >> group_shift) * 2 : (F == FF_F8 ? K / 32 : 0)));
  }
};

using qmoe_stream::kOob;
using qmoe_stream::make_rsrc;
using qmoe_stream::rsrc_t;

__device__ __forceinline__ uint4 load16(rsrc_t r, uint32_t off) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// The words that hold the scales of the lane's chunks c and c + 1 (c even) of
// the row at row_off, and where in them: FF_MX a byte each, FF_I4 a bf16, FF_NV a
// pair of bf16, FF_F8 one float32. (Whole, aligned words: the compiler extends a
// narrower load right behind it, where it waits for every load in flight.)
template <int F>
struct Scales {
  uint32_t w[2];
};
template <int F>
__device__ __forceinline__ uint32_t scale_off(uint32_t row_off, int c, int group_shift) {
  return row_off + (F == FF_MX ? c : (F == FF_NV ? c * 4 : (F == FF_I4 ? ((c * 32) >> group_shift) * 2 : (c >> 3) * 4)));
}
template <int F>
__device__ __forceinline__ Scales<F> load_scales(rsrc_t r, uint32_t row_off, int c, int group_shift, bool in) {
  Scales<F> s;
  if constexpr (F == FF_BF) {
    s.w[0] = s.w[1] = 0;
  } else {
    const uint32_t a = scale_off<F>(row_off, c, group_shift) & ~3u, b = scale_off<F>(row_off, c + 1, group_shift) & ~3u;
    s.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, in ? a : kOob, 0, 0);
    if constexpr (F == FF_F8) s.w[1] = s.w[0];
    // (mostly the same word: no request then)
    else s.w[1] = __builtin_amdgcn_raw_buffer_load_b32(r, in && b != a ? b : kOob, 0, 0);
  }
  return s;
}
// Scale of chunk c + u from its words, as expand8 takes it
template <int F>
__device__ __forceinline__ uint32_t scale_of(const uint32_t (&w)[2], uint32_t row_off, int c, int u, int group_shift) {
  if constexpr (F == FF_MX || F == FF_I4) {
    const uint32_t a = scale_off<F>(row_off, c, group_shift), o = scale_off<F>(row_off, c + u, group_shift);
    const uint32_t word = u && (o & ~3u) != (a & ~3u) ? w[1] : w[0];
    return (word >> ((o & 3u) * 8)) & (F == FF_MX ? 0xffu : 0xffffu);
  } else {
    return w[u];
  }
}

// One step of a wavefront: a 128-byte line of 16 rows for each of NT tiles
// (lane -> row 8 v + l / 8, chunk l % 8), their scales (lane -> row l % 16, chunks 2
// kg and 2 kg + 1, kg = l / 16) and the tokens' values for those two chunks
template <int F, int NT>
struct Step {
  uint4 w[NT][2];
  Scales<F> s[NT];
  uint4 x[2];
};

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

// 8 e4m3 codes (two dwords) times a scale, each product rounded once to bf16
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
  else if constexpr (F == FF_F8) return e4m3x8_to_bf16(d[2 * i], d[2 * i + 1], bf16_round(bits_f32(s)));
  else return c;
}

// acc[t][i] += line t . tokens, MFMA i of each chunk; `first`: the line's first
// chunk of the row, `end`: the row's chunks, row_off: the lane's scale row. `tr`: this wavefront's LDS,
// 2 KB per tile. Row r's chunk c lies at slot c ^ (r / 2), so that neither the
// writes (the 8 chunks of a row by 8 adjacent lanes) nor the reads (one chunk of
// 16 rows) meet in a bank.
template <int F, int NT>
__device__ __forceinline__ void consume(const Step<F, NT>& st, uint4* tr, uint32_t row_off, int first, int end,
                                        int group_shift, f32x4 (&acc)[NT][Fmt<F>::kMfma]) {
  const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
  // the scale words are taken as loaded only here: their conversions, moved up
  // to the loads of the step before, would wait for every load in flight
  uint32_t sc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    sc[t][0] = st.s[t].w[0];
    sc[t][1] = st.s[t].w[1];
    if constexpr (F != FF_BF) asm volatile("" : "+v"(sc[t][0]), "+v"(sc[t][1]));
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int row = 8 * v + (lane >> 3);
      tr[t * 128 + row * 8 + ((lane & 7) ^ (row >> 1))] = st.w[t][v];
    }
  qmoe_moe::wave_lds_sync();
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint4 c = tr[t * 128 + r * 8 + ((2 * kg + u) ^ (r >> 1))];
      // (behind a row's end lies the next row's scale: an infinity or NaN there, times the zero codes, is not this row's)
      const uint32_t scale = first + 2 * kg + u < end ? scale_of<F>(sc[t], row_off, first + 2 * kg, u, group_shift) : 0u;
      Bf8 b;
      b.u = st.x[u];
#pragma unroll
      for (int i = 0; i < Fmt<F>::kMfma; ++i) {
        Bf8 a;
        a.u = expand8<F>(c, i, scale);
        acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc[t][i], 0, 0, 0);
      }
    }
  qmoe_moe::wave_lds_sync();  // the slots are free for the next step
}

// The sums of the lane's token, from the kMfma columns it is spread over
template <int M>
__device__ __forceinline__ f32x4 own_sums(const f32x4 (&acc)[M]) {
  const int i = threadIdx.x & (M - 1);
  f32x4 v = acc[0];
#pragma unroll
  for (int k = 1; k < M; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = i == k ? acc[k][q] : v[q];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (M >= 2) v[q] += qmoe_route::dpp_f<0xB1>(v[q]);
    if constexpr (M >= 4) v[q] += qmoe_route::dpp_f<0x4E>(v[q]);
  }
  return v;
}

// From the routes (ids and tb.w, visible to the workgroup) to the tables; every
// thread calls. Slots in ascending order of (expert, token).
template <int ROWS>
__device__ __forceinline__ void few_tables(FewTables& tb, const int32_t* ids, uint32_t* tokens, int32_t* first,
                                           const FewParams& p) {
  const int tid = threadIdx.x, R = p.T * p.topk;
  auto valid = [&](int r) {
    return ids[r] >= 0 && ids[r] < p.E && !(p.skip && (f32_to_bf16(tb.w[r]) & 0x7fffu) == 0);
  };
  if (p.T == 1 && !p.skip) {  // a token's experts are distinct: a slot each
    if (tid < R) {
      tb.active[tid] = (int16_t)ids[tid];
      tb.route[tid * ROWS] = (int16_t)tid;
#pragma unroll
      for (int i = 1; i < ROWS; ++i) tb.route[tid * ROWS + i] = -1;
    }
    if (tid == 0) tb.num = R;
    __syncthreads();
    return;
  }
  for (int i = tid; i < kFewExperts; i += blockDim.x) tokens[i] = 0;
  for (int i = tid; i < R * ROWS; i += blockDim.x) tb.route[i] = -1;
  __syncthreads();
  if (tid < R && valid(tid)) atomicOr(&tokens[ids[tid]], 1u << (tid / p.topk));
  __syncthreads();
  if (tid < 64) {  // slots before an expert's first: lane l owns experts 8 l .. 8 l + 7
    int n[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      n[j] = (__popc(tokens[tid * 8 + j]) + ROWS - 1) / ROWS;
      sum += n[j];
    }
    int total;
    int at = qmoe_moe::wave_excl_scan(sum, tid, total);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      first[tid * 8 + j] = at;
      at += n[j];
    }
    if (tid == 0) tb.num = total;
  }
  __syncthreads();
  if (tid < R && valid(tid)) {
    const int e = ids[tid], rank = __popc(tokens[e] & ((1u << (tid / p.topk)) - 1u)), slot = first[e] + rank / ROWS;
    if (rank % ROWS == 0) tb.active[slot] = (int16_t)e;
    tb.route[slot * ROWS + rank % ROWS] = (int16_t)tid;
  }
  __syncthreads();
}

constexpr int kUpWaves = 4;

// A: steps in flight per wavefront
template <int F, int S, int A>
__global__ __launch_bounds__(kUpWaves * 64, 3) void few_up_kernel(const FewParams p) {
  constexpr int ROWS = Fmt<F>::kRows, M = Fmt<F>::kMfma;
  __shared__ FewTables tb;
  __shared__ int32_t ids[kFewRoutes];
  __shared__ union {
    float choice[kUpWaves][qmoe_route::kChoiceLds];
    struct {
      uint32_t tokens[kFewExperts];
      int32_t first[kFewExperts];
    } t;
  } tmp;
  __shared__ __align__(16) uint4 tr[kUpWaves][2 * 128];
  __shared__ __align__(16) f32x4 red[2][kUpWaves][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = p.T * p.topk;
  for (int t = wave; t < p.T; t += kUpWaves)
    qmoe_route::route_token_any<S>(p.scoring, p.grouped, p.logits, p.logits_f32, t, p.E, p.topk, p.correction,
                                   p.renormalize, p.rsf, p.num_group, p.topk_group, tb.w, ids, tmp.choice[wave], nullptr,
                                   nullptr, 1);
  __syncthreads();
  few_tables<ROWS>(tb, ids, tmp.t.tokens, tmp.t.first, p);
  const int num = __builtin_amdgcn_readfirstlane(tb.num);
  if (blockIdx.x == 0) {
    if (tid == 0) p.tables->num = num;
    if (tid < R) p.tables->w[tid] = tb.w[tid];
    if (tid < num) p.tables->active[tid] = tb.active[tid];
    for (int i = tid; i < num * ROWS; i += kUpWaves * 64) p.tables->route[i] = tb.route[i];
  }

  const int tiles = p.I / 16, items = num * tiles;
  const int it0 = (int)((int64_t)blockIdx.x * items / gridDim.x), it1 = (int)((int64_t)(blockIdx.x + 1) * items / gridDim.x);
  if (it0 >= it1) return;
  const int rb = Fmt<F>::row_bytes(p.H), sb = Fmt<F>::scale_bytes(p.H, p.group_shift);
  // steps per item, the same for every wavefront (those past a row's end load
  // nothing and add zeros)
  const int chunks = cdiv(cdiv(cdiv(rb, 128), kUpWaves), A);
  const int r = lane & 15, kg = lane >> 4;
  const rsrc_t xr = make_rsrc(p.x, (int64_t)p.T * p.ldx * 2);

  // where the loads are
  rsrc_t wr[2], sr[2];
  uint32_t xrow = kOob;  // byte offset of the column's token, at its MFMA's values
  auto seek = [&](int item) {
    const int slot = item / tiles, tile = item - slot * tiles;
    const int e = __builtin_amdgcn_readfirstlane(tb.active[slot]);
    const int route = tb.route[slot * ROWS + r / M];
    xrow = route >= 0 ? (uint32_t)((route / p.topk) * p.ldx * 2) + (r % M) * 16 : kOob;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = (int64_t)e * 2 * p.I + t * p.I + tile * 16;
      wr[t] = make_rsrc(p.w1 + row * rb, (int64_t)16 * rb);
      sr[t] = make_rsrc(static_cast<const uint8_t*>(p.s1) + row * sb, (int64_t)16 * sb);
    }
  };
  Step<F, 2> st[A];
  const uint32_t wlane = (uint32_t)((lane >> 3) * rb + (lane & 7) * 16), slane = (uint32_t)(r * sb);
  auto issue = [&](Step<F, 2>& d, int i, bool live) {
    const int line = (wave + kUpWaves * i) * 128;  // byte of the row
    const bool lin = live && line + (lane & 7) * 16 < rb;
    const int c = line / 16 + 2 * kg;  // the first chunk that the lane multiplies
    const bool in = live && c * 16 < rb;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int v = 0; v < 2; ++v) d.w[t][v] = load16(wr[t], lin ? wlane + (uint32_t)(8 * v * rb + line) : kOob);
      d.s[t] = load_scales<F>(sr[t], slane, c, p.group_shift, in);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      d.x[u] = load16(xr, live && (c + u) * 16 < rb ? xrow + (uint32_t)((c + u) * Fmt<F>::kCodes * 2) : kOob);
  };
  seek(it0);
  // (in this order: the loop's waits count the loads behind a step's own)
#pragma unroll
  for (int u = 0; u < A; ++u) {
    issue(st[u], u, true);
    __builtin_amdgcn_sched_barrier(0);
  }
  typedef const float __attribute__((address_space(4))) CFloat;
  for (int item = it0; item < it1; ++item) {
    const int slot = item / tiles, tile = item - slot * tiles;
    // the item's biases by scalar loads, in time for its end: a vector load's
    // wait there would drain the next item's weight loads
    float bg[16], bu[16];
    if (p.b1) {
      CFloat* b = (CFloat*)(uintptr_t)(p.b1 + (int64_t)__builtin_amdgcn_readfirstlane(tb.active[slot]) * 2 * p.I + tile * 16);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        bg[k] = b[k];
        bu[k] = b[p.I + k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) bg[k] = bu[k] = 0.0f;
    }
    f32x4 acc[2][M] = {};
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 < chunks, next = item + 1 < it1;
      if (!more && next) seek(item + 1);
#pragma unroll
      for (int u = 0; u < A; ++u) {
        consume<F, 2>(st[u], tr[wave], slane, (wave + kUpWaves * (c * A + u)) * 8, rb / 16, p.group_shift, acc);
        issue(st[u], (more ? (c + 1) * A : 0) + u, more || next);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // the wavefronts' sums in order, bias, activation (by one wavefront, while
    // the others go on: the next item's sums lie elsewhere)
    f32x4(&rd)[kUpWaves][2][64] = red[item & 1];
    rd[wave][0][lane] = own_sums<M>(acc[0]);
    rd[wave][1][lane] = own_sums<M>(acc[1]);
    stage_barrier();
    if (wave == item % kUpWaves && r % M == 0) {
      const int n0 = tile * 16 + kg * 4, route = tb.route[slot * ROWS + r / M];
      f32x4 g = rd[0][0][lane], u = rd[0][1][lane];
#pragma unroll
      for (int w = 1; w < kUpWaves; ++w) {
        g += rd[w][0][lane];
        u += rd[w][1][lane];
      }
      if (route >= 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          g[q] += kg == 0 ? bg[q] : (kg == 1 ? bg[4 + q] : (kg == 2 ? bg[8 + q] : bg[12 + q]));
          u[q] += kg == 0 ? bu[q] : (kg == 1 ? bu[4 + q] : (kg == 2 ? bu[8 + q] : bu[12 + q]));
        }
        uint16_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = f32_to_bf16(qmoe_act(p.act, g[q], u[q], p.act_p0, p.act_p1));
        *reinterpret_cast<uint2*>(p.h + (int64_t)route * p.I + n0) =
            make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
      }
    }
  }
}

constexpr int kDownAhead = 2, kDownWaves = 8;

template <int F>
__global__ __launch_bounds__(kDownWaves * 64) void few_down_kernel(const FewParams p) {
  constexpr int NW = kDownWaves, ROWS = Fmt<F>::kRows, M = Fmt<F>::kMfma;
  __shared__ FewTables tb;
  __shared__ __align__(16) uint4 tr[NW][128];
  __shared__ __align__(16) f32x4 tot[NW][64];  // [token][4 columns x 4]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = p.T * p.topk;
  // (every entry that a slot could have, so that no load waits for their number)
  const int num = __builtin_amdgcn_readfirstlane(p.tables->num);
  if (tid < R) {
    tb.w[tid] = p.tables->w[tid];
    tb.active[tid] = p.tables->active[tid];
  }
  for (int i = tid; i < R * ROWS; i += NW * 64) tb.route[i] = p.tables->route[i];
  __syncthreads();
  const int n0 = blockIdx.x * 16;
  const int rb = Fmt<F>::row_bytes(p.I), sb = Fmt<F>::scale_bytes(p.I, p.group_shift), lines = cdiv(rb, 128);
  const int r = lane & 15, kg = lane >> 4;
  const rsrc_t hr = make_rsrc(p.h, (int64_t)R * p.I * 2);

  // the wavefront's i-th step is line wave + NW i of all slots' rows laid end to
  // end; a cursor goes over them for the loads, another for the products
  struct Cursor {
    int slot, line;
  };
  auto settle = [&](Cursor& c) {
    while (c.line >= lines) {
      c.line -= lines;
      ++c.slot;
    }
  };
  Step<F, 1> st[kDownAhead];
  const uint32_t wlane = (uint32_t)((lane >> 3) * rb + (lane & 7) * 16), slane = (uint32_t)(r * sb);
  auto issue = [&](Step<F, 1>& d, Cursor& at) {
    settle(at);
    const bool live = at.slot < num;
    const int e = live ? __builtin_amdgcn_readfirstlane(tb.active[at.slot]) : 0;
    const int route = live ? tb.route[at.slot * ROWS + r / M] : -1;
    const int64_t row = (int64_t)e * p.H + n0;
    const rsrc_t wr = make_rsrc(p.w2 + row * rb, (int64_t)16 * rb);
    const rsrc_t sr = make_rsrc(static_cast<const uint8_t*>(p.s2) + row * sb, (int64_t)16 * sb);
    const int line = at.line * 128, c = line / 16 + 2 * kg;
    const bool lin = live && line + (lane & 7) * 16 < rb;
#pragma unroll
    for (int v = 0; v < 2; ++v) d.w[0][v] = load16(wr, lin ? wlane + (uint32_t)(8 * v * rb + line) : kOob);
    d.s[0] = load_scales<F>(sr, slane, c, p.group_shift, live && c * 16 < rb);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      d.x[u] = load16(hr, route >= 0 && (c + u) * 16 < rb
                              ? (uint32_t)(((int64_t)route * p.I + (c + u) * Fmt<F>::kCodes + (r % M) * 8) * 2)
                              : kOob);
    at.line += NW;
  };
  tot[wave][lane] = f32x4{};
  f32x4 acc[1][M] = {};
  // the slot's sums, weighted, into its tokens' (this wavefront's, in LDS)
  auto flush = [&](int slot) {
    const f32x4 v = own_sums<M>(acc[0]);
    const int route = tb.route[slot * ROWS + r / M];
    if (route >= 0 && r % M == 0) {
      const float w = tb.w[route];
      f32x4& t = tot[wave][route / p.topk * 4 + kg];
      t = t + w * v;
    }
#pragma unroll
    for (int i = 0; i < M; ++i) acc[0][i] = f32x4{};
  };
  // biases: the wavefront's first slot's is loaded ahead of the weights
  auto bias_of = [&](int k) {
    const float* b = p.b2 + (int64_t)tb.active[k] * p.H + n0 + kg * 4;
    return f32x4{b[0], b[1], b[2], b[3]};
  };
  auto add_bias = [&](int k, f32x4 b) {
    const int route = tb.route[k * ROWS + r / M];
    if (route >= 0 && r % M == 0) {
      f32x4& t = tot[wave][route / p.topk * 4 + kg];
      t = t + tb.w[route] * b;
    }
  };
  const bool biased = p.b2 && wave < num;
  f32x4 first_bias = {};
  if (biased) first_bias = bias_of(wave);
  Cursor ahead{0, wave}, now{0, wave};
#pragma unroll
  for (int u = 0; u < kDownAhead; ++u) {
    issue(st[u], ahead);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (biased) add_bias(wave, first_bias);
  int slot = -1;
  settle(now);
  while (now.slot < num) {
#pragma unroll
    for (int u = 0; u < kDownAhead; ++u) {
      if (now.slot < num) {
        if (now.slot != slot && slot >= 0) flush(slot);
        slot = now.slot;
        consume<F, 1>(st[u], tr[wave], slane, now.line * 8, rb / 16, p.group_shift, acc);
      }
      issue(st[u], ahead);
      now.line += NW;
      settle(now);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (slot >= 0) flush(slot);
  if (p.b2)
    for (int k = wave + NW; k < num; k += NW) add_bias(k, bias_of(k));
  __syncthreads();
  if (tid < p.T * 4) {  // token tid / 4, columns 4 (tid % 4) .. + 3
    f32x4 v = tot[0][tid];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += tot[w][tid];
    uint16_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = f32_to_bf16(v[q]);
    *reinterpret_cast<uint2*>(p.out + (int64_t)(tid >> 2) * p.ldo + n0 + (tid & 3) * 4) =
        make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
  }
}

template <int F, int S>
void launch_up(const FewParams& p, hipStream_t st) {
  // as many workgroups as fit (three per CU; 512 or 1536 instead: 118 or 119 us for
  // 113 with 16 tokens, MXFP4, 128 x 2880 x 2880; 207 or 212 for 189 with 8, NVFP4,
  // 256 x 2048 x 7168)
  const int64_t items = (int64_t)std::min(p.E, p.T * p.topk) * (p.I / 16);
  const dim3 grid((unsigned)std::min<int64_t>(items, 768)), block(kUpWaves * 64);
  // three steps in flight, or two where three leave more of them empty (the NVFP4
  // case, 7 lines per wavefront: 189 us by three, 176 by two; the MXFP4 one, 3
  // lines: 113 and 121; four: 210, 162)
  const int lines = cdiv(cdiv(Fmt<F>::row_bytes(p.H), 128), kUpWaves);
  if (cdiv(lines, 2) * 2 < cdiv(lines, 3) * 3) hipLaunchKernelGGL((few_up_kernel<F, S, 2>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((few_up_kernel<F, S, 3>), grid, block, 0, st, p);
}

template <int F>
void launch_few(const FewParams& p, hipStream_t st) {
  const int S = qmoe_route::route_slots(p.E);
  if (S <= 2) launch_up<F, 2>(p, st);
  else if (S == 4) launch_up<F, 4>(p, st);
  else launch_up<F, 8>(p, st);
  hipLaunchKernelGGL((few_down_kernel<F>), dim3((unsigned)(p.H / 16)), dim3(kDownWaves * 64), 0, st, p);
}

int64_t few_layout(int64_t R, int64_t I, int64_t (&off)[2]) {
  off[0] = 0;
  off[1] = (R * I * 2 + 255) / 256 * 256;
  return off[1] + ((int64_t)sizeof(FewTables) + 255) / 256 * 256;
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
  int64_t off[2];
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
  int64_t off[2];
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
  p.tables = reinterpret_cast<FewTables*>(ws + off[1]);
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
