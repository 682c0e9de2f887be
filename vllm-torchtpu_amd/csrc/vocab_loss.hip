// Softmax cross entropy of a projection onto the vocabulary table, in pieces
// of the vocabulary, without keeping the logits:
//
//   l[t, v] = s[v] x[t] . w[v]       (s: one scale per row of a 1-byte table, else 1)
//   lse[t]  = log sum_v exp l[t, v]
//   loss[t] = lse[t] - l[t, target[t]], 0 where target[t] is the ignored index
//
// and with g the gradients of loss (of scored tokens) and h of lse
//
//   P[t, v] = exp(l[t, v] - lse[t]) (g[t] + h[t]) - [v == target[t]] g[t]
//   dx[t]   = sum_v P[t, v] s[v] w[v],      dw[v] = sum_t P[t, v] x[t]
//
// What bounds it: four matrix products of 2 T V H operations on the bf16 matrix
// cores (the logits twice: keeping them would take T V values), or, for few
// tokens, one read of the table.
//
// Every product is the same tile, 256 "A" rows x 64, 128 or 256 "B" rows per
// workgroup, with the stage ring of gemm_t8.hip and an epilogue of its own:
//   logits : A = table rows, B = tokens; per token and tile the maximum and the
//            sum of exponentials (one pass), and the target's logit
//   probs  : the same product again; P as [t][v]
//   dx     : A = columns of the table piece, B = P rows; float32 sums added over
//            the pieces
//   dw     : A = columns of x (transposed once), B = columns of P; K = tokens
// Rows run along K, the contiguous axis, or, of the table in dx and of P in dw,
// across it: those are copied as they lie, 64 K rows of a stage, and transposed
// on their way from LDS to registers by ds_read_b64_tr_b16. (With a transposed
// copy of each table piece and P stored both ways instead: 892 us against 766 at
// 333 tokens x 50021 x 2880, 14.26 ms against 14.15 at 4096 x 131072 x 4096.)
// For the gradients the tokens that have one are gathered first, in order, so
// that masked ones cost nothing and whatever they hold is not read: their number
// stays on the device, and tiles behind it end at once (333 tokens x 50021 x 2880,
// 101 of them not scored: 541 -> 488 us for loss and gradients).
// Sums are float32; P is rounded to bf16 once, as the operand of the products.

#include <algorithm>
#include <type_traits>

#include "../../include/qmoe.h"
#include "gemm_across.h"

namespace {

constexpr int kVThreads = 512;
constexpr int kVN = 256;  // A rows of a tile

enum { VE_LSE = 0, VE_PROB = 1, VE_SUM = 2, VE_STORE = 3 };

struct VocabGemm {
  const uint8_t* a;  // rows [na][lda bytes] of bf16, or codes where the kernel says so
  int64_t lda;
  int na;
  const uint8_t* b;  // bf16 rows [nb][ldb bytes]
  int64_t ldb;
  int nb;
  int K;  // a multiple of 8
  int n_tiles, m_tiles;
  // logits / probs: A row r is table row v0 + r; B rows are tokens
  const float* row_scale;  // of the piece (from v0 on), or nullptr
  int64_t v0, V;
  const void* targets;
  int targets_i64;
  int64_t ignore;
  float2* part;     // [tiles of all pieces][nb] maximum and sum of exponentials
  int part_tile;    // first tile of the piece
  float* tgt;       // [nb] the target's logit
  const float *lse, *g_loss, *g_lse;  // g_lse may be nullptr
  const int32_t *live, *count;        // gradients: the tokens that have one, and how many (x, P and sums hold these)
  uint16_t* p;      // [nb][ldp] P
  int64_t ldp;
  // dx / dw: out[b row][a row]
  float* sum;       // [nb][ldsum] float32 sums of the pieces before, or nullptr
  int64_t ldsum;
  int kr;           // K rows of the operand that lies across K: those from kr on meet zeros
  int first, last;  // first / last piece
  int kslice;       // K split: slice z takes the K range from z * kslice on ...
  float* slices;    // ... and leaves its sums in [z][nb][ldsum]; kslice 0: no split
  uint16_t* y;      // [nb][ldy]
  int64_t ldy;
};

__device__ __forceinline__ int64_t load_target(const VocabGemm& p, int t) {
  return p.targets_i64 ? static_cast<const int64_t*>(p.targets)[t]
                       : (int64_t) static_cast<const int32_t*>(p.targets)[t];
}

// Which operand lies across K
constexpr bool tr_a(int epi) { return epi == VE_SUM; }
constexpr bool tr_b(int epi) { return epi == VE_STORE; }

// (maximum, sum of exponentials below it) of two disjoint sets; the base of the
// exponentials is 0 where the maximum is infinite, so that infinite logits give
// an infinite sum and a set without any (-inf, 0)
__device__ __forceinline__ float lse_base(float m) { return fabsf(m) == __builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float2 lse_merge(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), base = lse_base(m);
  // a sum is relative to its own base
  const float sa = a.x == -__builtin_inff() ? a.y : a.y * __expf(lse_base(a.x) - base);
  const float sb = b.x == -__builtin_inff() ? b.y : b.y * __expf(lse_base(b.x) - base);
  return make_float2(m, sa + sb);
}

// The epilogues. A tile's wavefront (wn, wm), wn < WN, wm < 2, holds NI x MJ
// blocks of 32 x 32: register quad q of block (i, j) is A rows (wn NI + i) 32 + 8
// q + 4 kh .. + 3 and B row (2 j + wm) 32 + rl, rl = lane % 32, kh = lane / 32.
// The logits are reduced in registers; the others pass 64 B rows at a time
// through LDS (A row n of B row t at n ^ 4 f(t)), so that a thread stores 8
// consecutive values. `smem`: 74 KB of LDS that no copy or read uses any more.
template <int EPI, int BM, int WN, int NI, int MJ>
__device__ __forceinline__ void vocab_epilogue(const VocabGemm& p, f32x16 (&acc)[NI][MJ], uint8_t* smem, int nt, int m0,
                                               int arows, int brows, int wn, int wm) {
  constexpr int BN = WN * NI * 32, THREADS = WN * 128;
  static_assert(BN == kVN, "tile height");
  const int tid = threadIdx.x, lane = tid & 63, rl = lane & 31, kh = lane >> 5, n0 = nt * BN;
  float* s_scale = reinterpret_cast<float*>(smem);
  float* reg = reinterpret_cast<float*>(smem + 9216);  // [64][BN]
  if constexpr (EPI == VE_LSE || EPI == VE_PROB) {
    for (int i = tid; i < BN; i += THREADS) s_scale[i] = p.row_scale ? p.row_scale[n0 + min(i, arows - 1)] : 1.0f;
    __syncthreads();
  }
  if constexpr (EPI == VE_LSE) {
    float2* s_part = reinterpret_cast<float2*>(smem + 1024);  // [WN][BM]
    constexpr float kLog2e = 1.4426950408889634f;
    const bool plain = p.row_scale == nullptr && arows == BN;  // neither scales nor rows to leave out
    const int n1 = wn * NI * 32 + kh * 4;
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      const int tb = (2 * j + wm) * 32 + rl;
      float m = -__builtin_inff(), s = 0.0f;
      if (!plain) {
        const int lim = opaque_s(arows);
        const float* sc = s_scale + opaque_v(n1);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int n = i * 32 + q * 8 + r;
              acc[i][j][q * 4 + r] = n1 + n < lim ? acc[i][j][q * 4 + r] * sc[n] : -__builtin_inff();
            }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
      const float base = lse_base(m), b2 = base * kLog2e;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, -b2));
      // the target's logit, if its row is one of this lane's
      if (tb < brows) {
        const int64_t at = load_target(p, m0 + tb) - p.v0 - n0 - n1;
        if (at >= 0 && at < NI * 32 && at < arows - n1 && (at & 4) == 0) {
          float l = 0.0f;
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) l = (int)at == i * 32 + (r / 4) * 8 + r % 4 ? acc[i][j][r] : l;
          p.tgt[m0 + tb] = l;
        }
      }
      const float2 both = lse_merge(make_float2(m, s), make_float2(__shfl_xor(m, 32, 64), __shfl_xor(s, 32, 64)));
      if (kh == 0) s_part[wn * BM + tb] = both;
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    for (int t = tid; t < brows; t += THREADS) {
      float2 v = s_part[t];
#pragma unroll
      for (int w = 1; w < WN; ++w) v = lse_merge(v, s_part[w * BM + t]);
      p.part[(int64_t)(p.part_tile + nt) * p.nb + m0 + t] = v;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int tl = wm * 32 + rl, tb = 64 * j + tl;  // B row of the 64, of the tile
    if (64 * j >= brows) break;
    if (j) __syncthreads();  // the rows before have been read
    const int n1 = opaque_v(wn * NI * 32 + kh * 4);
    if constexpr (EPI == VE_PROB) {
      const bool valid = tb < brows;
      float hot = 0.0f, coef = 0.0f, lse2 = 0.0f;
      int at = -1;
      if (valid) {
        const int t = p.live[m0 + tb];
        const int64_t tg = load_target(p, t);
        const float g = p.g_loss[t];  // (0 for a target outside the table: its NaN loss went nowhere)
        hot = tg == p.ignore || g == 0.0f ? 0.0f : (tg >= 0 && tg < p.V ? g : __builtin_nanf(""));
        coef = hot + (p.g_lse ? p.g_lse[t] : 0.0f);
        lse2 = p.lse[t] * 1.4426950408889634f;
        const int64_t in = tg - p.v0 - n0;
        at = in >= 0 && in < arows ? (int)in : -1;
      }
      const int lim = opaque_s(arows);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int n = n1 + i * 32 + q * 8 + r;
            // a token without a gradient leaves zeros, whatever its logits are
            float e = __builtin_amdgcn_exp2f(fmaf(acc[i][j][q * 4 + r] * s_scale[n], 1.4426950408889634f, -lse2)) * coef;
            e = n < lim && coef != 0.0f ? e : 0.0f;
            v[r] = n == at ? e - hot : e;
          }
          const int n = n1 + i * 32 + q * 8;
          *reinterpret_cast<float4*>(reg + tl * BN + (n ^ vg_row_swz(tl))) = make_float4(v[0], v[1], v[2], v[3]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n1 + i * 32 + q * 8;
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = acc[i][j][q * 4 + r];
          }
          *reinterpret_cast<float4*>(reg + tl * BN + (n ^ vg_row_swz(tl))) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    __syncthreads();
    // 8 consecutive A rows of a B row per thread
    constexpr int CH = BN / 8;
    const int c = (tid % CH) * 8;
#pragma unroll 2
    for (int t = tid / CH; t < 64; t += THREADS / CH) {
      const int64_t row = m0 + 64 * j + t;
      if (64 * j + t >= brows) break;
      const float4 lo = *reinterpret_cast<const float4*>(reg + t * BN + (c ^ vg_row_swz(t)));
      const float4 hi = *reinterpret_cast<const float4*>(reg + t * BN + ((c + 4) ^ vg_row_swz(t)));
      float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if constexpr (EPI == VE_PROB) {
        // P times the row scales is what multiplies the codes
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= s_scale[c + k];
        *reinterpret_cast<uint4*>(p.p + row * p.ldp + n0 + c) = make_uint4(
            pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      } else if (c < arows) {  // (A rows come in multiples of 8)
        if constexpr (EPI == VE_SUM) {
          float4* dst = reinterpret_cast<float4*>(p.sum + row * p.ldsum + n0 + c);
          if (!p.first) {
            const float4 a = dst[0], b = dst[1];
            v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
            v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
          }
          if (!p.last) {
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            continue;
          }
        }
        *reinterpret_cast<uint4*>(p.y + (EPI == VE_SUM ? p.live[row] : row) * p.ldy + n0 + c) = make_uint4(
            pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      }
    }
  }
}

// This workgroup's slice of a K split (dx only)
template <int EPI>
__device__ __forceinline__ void take_slice(VocabGemm& p) {
  if constexpr (EPI == VE_SUM) {
    if (p.kslice) {
      const int k0 = blockIdx.y * p.kslice;
      p.a += k0 * p.lda;
      p.b += (int64_t)k0 * 2;
      p.K = min(p.kslice, p.K - k0);
      p.kr -= k0;
      p.sum = p.slices + (int64_t)blockIdx.y * p.nb * p.ldsum;
      p.first = 1, p.last = 0;
    }
  }
}

// B rows of the problem: tokens with a gradient of P and dx; of dw they are K
template <int EPI>
__device__ __forceinline__ int live_rows(VocabGemm& p) {
  if constexpr (EPI == VE_LSE) return p.nb;
  const int n = __builtin_amdgcn_readfirstlane(*p.count);
  if constexpr (EPI == VE_STORE) {
    p.kr = n;
    p.K = (n + 63) / 64 * 64;
    return p.nb;
  }
  return n;
}

// 8 codes of a chunk as bf16 (exact)
template <int AT>
__device__ __forceinline__ bf16x8 codes8_to_bf16(uint32_t lo, uint32_t hi) {
  union {
    bf16x2 h[4];
    bf16x8 v;
  } r;
  if constexpr (AT == 3) {
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true);
  } else if constexpr (AT == 5) {
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)lo, 1.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)lo, 1.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)hi, 1.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)hi, 1.0f, true);
  } else {
    const uint32_t d[2] = {lo, hi};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      r.h[k] = __builtin_convertvector(
          f32x2{(float)(int8_t)(d[k / 2] >> (16 * (k & 1))), (float)(int8_t)(d[k / 2] >> (16 * (k & 1) + 8))}, bf16x2);
  }
  return r.v;
}

// Tiles of 256 A rows x BM B rows (64 or 128) by eight wavefronts, two per SIMD,
// for problems that the 256 x 256 tiles below would leave CUs idle or pad, and
// for few tokens, where reading the table is all that counts (one token, 131072
// x 4096 bf16: 169 us, 6.4 TB/s; 16 tokens, 131072 x 7168 e4m3: 177 us, 5.3
// TB/s): with codes (AT 3 e4m3, 4 int8, 5 e5m2) the table is read as it is stored
// and expanded between LDS and the matrix cores. Stages of 64 k of every row in a ring of
// as many as fit.
// ONE: a stage at a time, without a ring, so that two workgroups share a CU and
// each one's copies and stores run under the other's products (kShortK).
template <int EPI, int BM, int AT, bool ONE = false>
__global__ __launch_bounds__(kVThreads, ONE ? 4 : 2) void vocab_gemm_kernel(const VocabGemm args) {
  constexpr int BN = kVN, NI = 2, MJ = BM / 64;
  constexpr bool TRA = tr_a(EPI), TRB = tr_b(EPI);
  constexpr int AB = AT ? 64 : 128;  // bytes of an A row per stage
  constexpr int WB = BN * AB, STG = WB + BM * 128;
  constexpr int RING = ONE ? 1 : (163840 / STG < 6 ? 163840 / STG : 6), EPILOGUE = 9216 + 65536;
  __shared__ __align__(1024) uint8_t smem[RING * STG > EPILOGUE ? RING * STG : EPILOGUE];
  static_assert(ONE ? sizeof(smem) <= 81920 : RING >= 3 && sizeof(smem) <= 163840, "workgroups of a CU, ring");
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  VocabGemm p = args;
  take_slice<EPI>(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 3, wm = wave >> 2, rl = lane & 31, kh = lane >> 5;
  int mt, nt;
  if (!tile_dense(blockIdx.x, p.m_tiles, p.n_tiles, mt, nt)) return;
  const int n0 = nt * BN, m0 = mt * BM;
  const int arows = min(BN, p.na - n0), brows = min(BM, live_rows<EPI>(p) - m0);
  if ((EPI == VE_PROB || EPI == VE_SUM) && brows <= 0) return;

  // copies: one instruction = 8 rows x 128 bytes (lane -> row l >> 3, slot l & 7;
  // the slot of chunk c of row r is c ^ vg_swz(r)) or, of codes, 16 rows x 64
  // bytes (lane -> row l >> 2, slot l & 3, chunk c at c ^ (r / 4) % 4); wavefront w
  // moves the groups w, w + 8, ... of both operands; rows past the end repeat
  // the last one (their products are dropped)
  constexpr int WI = WB / 8192, XI = BM / 64;
  const int xchunk = (lane & 7) ^ ((lane >> 3) ^ (wave & 1));
  const int achunk = AT ? (lane & 3) ^ ((lane >> 4) & 3) : xchunk;
  const uint8_t* abase = p.a + (int64_t)n0 * p.lda;
  const uint8_t* bbase = p.b + (int64_t)m0 * p.ldb;
  uint32_t aoff[WI], boff[XI];
  // the operand across K: an instruction is 1 KB of K rows; K rows past the last
  // repeat it, by the bytes from the stage's first row that a lane stays below
  constexpr int TB = TRA ? BN * 2 : BM * 2, TL = TB / 16;  // bytes, lanes of a K row
  const int trow = lane / TL, tchunk = (lane % TL) ^ tr_swz<TB>(wave * (64 / TL) + trow);
  const uint32_t tcol = TRA ? (uint32_t)min(tchunk, arows / 8 - 1) * 16 : (uint32_t)tchunk * 16;
  const int64_t tld = TRA ? p.lda : p.ldb;
  if constexpr (TRA) abase = p.a + n0 * 2;
  if constexpr (TRB) bbase = p.b + m0 * 2;
  const int64_t astep = TRA ? 64 * p.lda : AB, bstep = TRB ? 64 * p.ldb : 128;
#pragma unroll
  for (int j = 0; j < WI; ++j) {
    if constexpr (TRA) {
      aoff[j] = (uint32_t)((wave + 8 * j) * (64 / TL) + trow) * (uint32_t)tld + tcol;
      continue;
    }
    const int r = AT ? (wave + 8 * j) * 16 + (lane >> 2) : (wave + 8 * j) * 8 + (lane >> 3);
    aoff[j] = (uint32_t)min(r, arows - 1) * (uint32_t)p.lda + achunk * 16;
  }
#pragma unroll
  for (int j = 0; j < XI; ++j)
    boff[j] = TRB ? (uint32_t)((wave + 8 * j) * (64 / TL) + trow) * (uint32_t)tld + tcol
                  : (uint32_t)min((wave + 8 * j) * 8 + (lane >> 3), brows - 1) * (uint32_t)p.ldb + xchunk * 16;
  const int KF = p.K / 64;  // whole stages
  const uint32_t cw = lds0 + wave * 1024;
  // stage s to slot `slot` (stages past the last one copy it again, into slots
  // nobody reads)
  auto copy_stage = [&](int s, int slot) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(cw + slot * STG);
    const int k = min(s, KF - 1);
    const uint8_t *as = uniform_ptr(abase + k * astep), *bs = uniform_ptr(bbase + k * bstep);
    uint32_t end = 0;
    if constexpr (TRA || TRB) end = (uint32_t)min(63, p.kr - 64 * k - 1) * (uint32_t)tld + tcol;
#pragma unroll
    for (int j = 0; j < WI; ++j) lds_copy16(as, TRA ? min(aoff[j], end) : aoff[j], d + j * 8192);
#pragma unroll
    for (int j = 0; j < XI; ++j) lds_copy16(bs, TRB ? min(boff[j], end) : boff[j], d + WB + j * 8192);
  };

  f32x16 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // operand reads and MFMAs of step q (16 k). bf16: lane -> row l & 31, chunk 2 q
  // + kh of both operands. Codes: a 16-byte chunk, 2 (q / 2) + kh, holds the
  // lane's codes of two steps, so the B chunk is 4 (q / 2) + 2 kh + q % 2.
  union B8 {
    uint4 u;
    bf16x8 v;
  };
  B8 wf[2][NI], xf[2][MJ];
  const uint32_t tlane = tr_lane<TB>(lane);
  auto read_q = [&](int slot, int q) {
    const uint8_t* sW = smem + slot * STG;
    if constexpr (TRA) {
#pragma unroll
      for (int i = 0; i < NI; ++i) wf[q & 1][i].u = tr_read<TB>(sW + q * 16 * TB + (tlane ^ (wn * NI + i) * 64));
    } else if constexpr (AT) {
      if (q % 2 == 0)
#pragma unroll
        for (int i = 0; i < NI; ++i)
          wf[q / 2][i].u = *reinterpret_cast<const uint4*>(sW + (wn * 64 + i * 32 + rl) * 64 +
                                                            (((2 * (q / 2) + kh) ^ (rl >> 2)) & 3) * 16);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i)
        wf[q & 1][i].u =
            *reinterpret_cast<const uint4*>(sW + (wn * 64 + i * 32 + rl) * 128 + ((2 * q + kh) ^ vg_swz(rl)) * 16);
    }
    const int c = AT ? 4 * (q / 2) + 2 * kh + (q & 1) : 2 * q + kh;
#pragma unroll
    for (int j = 0; j < MJ; ++j)
      if constexpr (TRB) xf[q & 1][j].u = tr_read<TB>(sW + WB + q * 16 * TB + (tlane ^ (2 * j + wm) * 64));
      else xf[q & 1][j].u =
          *reinterpret_cast<const uint4*>(sW + WB + ((2 * j + wm) * 32 + rl) * 128 + (c ^ vg_swz(rl)) * 16);
  };
  auto mma = [&](int q) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      bf16x8 a;
      if constexpr (AT) {
        const uint4 c = wf[q / 2][i].u;
        a = q & 1 ? codes8_to_bf16<AT>(c.z, c.w) : codes8_to_bf16<AT>(c.x, c.y);
      } else {
        a = wf[q & 1][i].v;
      }
#pragma unroll
      for (int j = 0; j < MJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, xf[q & 1][j].v, acc[i][j], 0, 0, 0);
    }
  };
  // Per stage: all but the last MFMA step run while the next step's operands are
  // read; then the next stage's copies have landed -> barrier: everybody holds
  // this stage's last operands, so that its slot takes the copies of stage s +
  // RING -> the last step, while the next stage's first operands are read.
  if constexpr (ONE) {
    for (int s = 0; s < KF; ++s) {
      copy_stage(s, 0);
      wait_copies_upto<0>();
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        read_q(0, q);
        mma(q);
      }
      __syncthreads();
    }
  } else if (KF > 0) {
#pragma unroll
    for (int r = 0; r < RING; ++r) copy_stage(r, r);
    wait_copies_upto<(RING - 1) * (WI + XI)>();
    stage_barrier();
    read_q(0, 0);
    int slot = 0;
    for (int s = 0; s < KF; ++s) {
      const int next = slot == RING - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        read_q(slot, q + 1);
        mma(q);
      }
      wait_copies_upto<(RING - 2) * (WI + XI)>();
      stage_barrier();
      copy_stage(s + RING, slot);
      asm volatile("" ::: "memory");
      read_q(next, 0);
      mma(3);
      slot = next;
    }
    wait_copies_upto<0>();
    __syncthreads();
  }
  // the last, partial stage: zeros behind the rows' ends (K is a multiple of 16
  // for codes, 8 else; that of dx and dw of 64)
  if ((EPI == VE_LSE || EPI == VE_PROB) && p.K % 64) {
    const uint8_t *as = abase + (int64_t)KF * AB, *bs = bbase + (int64_t)KF * 128;
    const bool ain = KF * 64 + achunk * (AT ? 16 : 8) < p.K, bin = KF * 64 + xchunk * 8 < p.K;
    const uint8_t* z = reinterpret_cast<const uint8_t*>(kZeroChunk);
#pragma unroll
    for (int j = 0; j < WI; ++j) lds_copy16(ain ? as + aoff[j] : z, cw + j * 8192);
#pragma unroll
    for (int j = 0; j < XI; ++j) lds_copy16(bin ? bs + boff[j] : z, cw + WB + j * 8192);
    wait_copies_upto<0>();
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      read_q(0, q);
      mma(q);
    }
    __syncthreads();
  }
  vocab_epilogue<EPI, BM, 4, NI, MJ>(p, acc, smem, nt, m0, arows, brows, wn, wm);
}

// The slices of a K split and the pieces before -> the running sums, or, after
// the last piece, dx
__global__ __launch_bounds__(256) void vocab_slices_kernel(const VocabGemm p, int slices) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, n = (int64_t)p.nb * p.ldsum;
  if (i >= (int64_t)*p.count * p.ldsum) return;
  const int64_t row = i / p.ldsum;
  const int c = (int)(i - row * p.ldsum);
  float4 v = p.first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *reinterpret_cast<const float4*>(p.sum + i);
  for (int z = 0; z < slices; ++z) {
    const float4 a = *reinterpret_cast<const float4*>(p.slices + z * n + i);
    v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
  }
  if (!p.last) *reinterpret_cast<float4*>(p.sum + i) = v;
  else *reinterpret_cast<uint2*>(p.y + p.live[row] * p.ldy + c) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// The same product in tiles of 256 x 256 (or 192: 4 x 3 blocks) by four wavefronts
// of 4 x 4 blocks (one per SIMD, the sums in accumulation registers). A wavefront of 64 x 128 reads
// 24 KB of operands from LDS per 32 MFMAs, one of 128 x 128 32 KB per 64: with
// eight of the former per CU the reads and the copies' writes fill LDS's 128
// bytes per cycle, which is what bounds that kernel.
//
// Stages of 64 k: 32 KB of A rows and 32 KB of B rows, in a ring of five such
// slots (all of LDS): A(s), B(s), A(s + 1), B(s + 1), A(s + 2). At the barrier of
// stage s every wavefront holds its last operands, and the stage's two slots
// take B(s + 2) and A(s + 3). Their copies go out four per MFMA step and one at a
// time between the MFMAs: four wavefronts' copies at once would keep the
// address unit busy, and the matrix cores idle, for half a step. Whole
// 128-byte lines per row: with 64-byte rows in a ring of four smaller stages the
// second half of a line is asked for while the first is pending, and the L1
// stalls on it (dw of 4096 tokens, 16384 x 4096: 458 us; by lines 417). Codes
// (AT) take 64 bytes of a row and are expanded on their way to the matrix cores.
//
// 4096 tokens: logits of 131072 x 4096 3.11 ms, 1.41 PFLOP/s; of 16384 rows the
// probabilities 454 us, 1.21 PFLOP/s (their stores wait for nothing, but no
// product runs meanwhile), dx 397, 1.38, dw 418, 1.31. A plain product of 8192 on
// each side by the library reaches 1.25 to 1.54 on the same card.
// TAIL: K is not a multiple of 64 (an instance of its own: the extra stage costs
// the others registers).
constexpr int kBThreads = 256;

template <int EPI, int BM, int AT, bool TAIL>
__global__ __launch_bounds__(kBThreads, 1) void vocab_big_kernel(const VocabGemm args) {
  constexpr int BN = kVN, NI = 4, MJ = BM / 64, BI = 2 * MJ;  // BI: a wavefront's copies of B rows per stage
  constexpr uint32_t SLOT = BN * 128, RING = 5 * SLOT;
  constexpr bool TRA = tr_a(EPI), TRB = tr_b(EPI);
  constexpr int AB = AT ? 64 : 128, AI = AT ? 4 : 8;  // bytes of an A row per stage, a wavefront's copies of them
  constexpr int TB = 512;  // bytes of a K row of the operand across K
  static_assert(!TRB || BM == 256, "K rows of 512 bytes");
  __shared__ __align__(1024) uint8_t smem[RING];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  VocabGemm p = args;
  take_slice<EPI>(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = wave >> 1, rl = lane & 31, kh = lane >> 5;
  int mt, nt;
  if (!tile_dense(blockIdx.x, p.m_tiles, p.n_tiles, mt, nt)) return;
  const int n0 = nt * BN, m0 = mt * BM;
  const int arows = min(BN, p.na - n0), brows = min(BM, live_rows<EPI>(p) - m0);
  if ((EPI == VE_PROB || EPI == VE_SUM) && brows <= 0) return;

  // copies: one instruction = 8 rows x 128 bytes (lane -> row l >> 3, slot l & 7;
  // the slot of chunk c of row r is c ^ vg_swz(r)); wavefront w moves the row
  // groups w, w + 4, ... of both operands; rows past the end repeat the last
  // one (their products are dropped)
  const int chunk16 = (lane & 7) ^ ((lane >> 3) ^ (wave & 1)), achunk = (lane & 3) ^ ((lane >> 4) & 3);
  const uint8_t* abase = p.a + (int64_t)n0 * p.lda;
  const uint8_t* bbase = p.b + (int64_t)m0 * p.ldb;
  // (the operand across K: 2 K rows per instruction; K rows past the last repeat
  // it, by the bytes from the stage's first row that a lane stays below)
  const int trow = lane >> 5, tchunk = (lane & 31) ^ tr_swz<TB>(2 * wave + trow);
  const uint32_t tcol = TRA ? (uint32_t)min(tchunk, arows / 8 - 1) * 16 : (uint32_t)tchunk * 16;
  if constexpr (TRA) abase = p.a + n0 * 2;
  if constexpr (TRB) bbase = p.b + m0 * 2;
  const int64_t astep = TRA ? 64 * p.lda : AB, bstep = TRB ? 64 * p.ldb : 128;
  const uint32_t tld = (uint32_t)(TRA ? p.lda : p.ldb);
  uint32_t aoff[8], boff[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = (wave + 4 * j) * 8 + (lane >> 3);
    const uint32_t t = (uint32_t)(2 * (wave + 4 * j) + trow) * tld + tcol;
    aoff[j] = TRA ? t : (uint32_t)min(r, arows - 1) * (uint32_t)p.lda + chunk16 * 16;
    if constexpr (AT) {  // (16 rows x 64 bytes, as in the kernel above)
      const int ra = ((wave + 4 * j) & 15) * 16 + (lane >> 2);
      aoff[j] = (uint32_t)min(ra, arows - 1) * (uint32_t)p.lda + achunk * 16;
    }
    boff[j] = TRB ? t : (uint32_t)min(r, brows - 1) * (uint32_t)p.ldb + chunk16 * 16;
  }
  const int KF = p.K / 64;  // whole stages
  const uint32_t cw = lds0 + wave * 1024;
  union B8 {
    uint4 u;
    bf16x8 v;
  };
  B8 wf[2][NI], xf[2][MJ];
  // operand reads of step q of a stage: lane -> row l & 31, chunk 2 q + kh
  const uint32_t wpo = (uint32_t)(wn * NI * 4096 + rl * 128), xpo = (uint32_t)(wm * 4096 + rl * 128);
  const uint32_t tlane = tr_lane<TB>(lane) ^ (TRA ? wn * NI * 64 : wm * 64);
  auto read_w = [&](uint32_t slot, int q) {
    if constexpr (TRA) {
#pragma unroll
      for (int i = 0; i < NI; ++i) wf[q & 1][i].u = tr_read<TB>(smem + slot + q * 16 * TB + (tlane ^ i * 64));
      return;
    }
    if constexpr (AT) {  // 16 codes: of this step and the next
      if (q & 1) return;
      const uint8_t* b = smem + slot + wpo / 2 + (((q + kh) ^ (rl >> 2)) & 3) * 16;
#pragma unroll
      for (int i = 0; i < NI; ++i) wf[q / 2][i].u = *reinterpret_cast<const uint4*>(b + i * 2048);
      return;
    }
    const uint8_t* b = smem + slot + wpo + ((2 * q + kh) ^ vg_swz(rl)) * 16;
#pragma unroll
    for (int i = 0; i < NI; ++i) wf[q & 1][i].u = *reinterpret_cast<const uint4*>(b + i * 4096);
  };
  auto read_x = [&](uint32_t slot, int q) {
    if constexpr (TRB) {
#pragma unroll
      for (int j = 0; j < MJ; ++j) xf[q & 1][j].u = tr_read<TB>(smem + slot + q * 16 * TB + (tlane ^ j * 128));
      return;
    }
    const int c = AT ? 4 * (q / 2) + 2 * kh + (q & 1) : 2 * q + kh;
    const uint8_t* b = smem + slot + xpo + (c ^ vg_swz(rl)) * 16;
#pragma unroll
    for (int j = 0; j < MJ; ++j) xf[q & 1][j].u = *reinterpret_cast<const uint4*>(b + j * 8192);
  };
  f32x16 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  auto mma_row = [&](int q, int i) {
    bf16x8 a;
    if constexpr (AT) {
      const uint4 c = wf[q / 2][i].u;
      a = q & 1 ? codes8_to_bf16<AT>(c.z, c.w) : codes8_to_bf16<AT>(c.x, c.y);
    } else {
      a = wf[q & 1][i].v;
    }
#pragma unroll
    for (int j = 0; j < MJ; ++j)
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, xf[q & 1][j].v, acc[i][j], 0, 0, 0);
  };
  if (KF > 0) {
    // (stages past the last one copy it again, into slots nobody reads)
    auto asrc = [&](int s) { return uniform_ptr(abase + min(s, KF - 1) * astep); };
    auto bsrc = [&](int s) { return uniform_ptr(bbase + min(s, KF - 1) * bstep); };
    auto end_of = [&](int s) { return (uint32_t)min(63, p.kr - 64 * min(s, KF - 1) - 1) * tld + tcol; };
    auto copy_a = [&](const uint8_t* base, int j, uint32_t end, uint32_t to) {
      lds_copy16(base, TRA ? min(aoff[j], end) : aoff[j], to);
    };
    auto copy_b = [&](const uint8_t* base, int j, uint32_t end, uint32_t to) {
      lds_copy16(base, TRB ? min(boff[j], end) : boff[j], to);
    };
    auto dst = [&](uint32_t slot) { return (uint32_t)__builtin_amdgcn_readfirstlane(cw + slot); };
    auto wrap = [](uint32_t slot) { return slot >= RING ? slot - RING : slot; };
#pragma unroll
    for (int j = 0; j < AI; ++j) copy_a(asrc(0), j, end_of(0), dst(0) + j * 4096);
#pragma unroll
    for (int j = 0; j < BI; ++j) copy_b(bsrc(0), j, end_of(0), dst(SLOT) + j * 4096);
#pragma unroll
    for (int j = 0; j < AI; ++j) copy_a(asrc(1), j, end_of(1), dst(2 * SLOT) + j * 4096);
#pragma unroll
    for (int j = 0; j < BI / 2; ++j) copy_b(bsrc(1), j, end_of(1), dst(3 * SLOT) + j * 4096);
    wait_copies_upto<AI + BI / 2>();  // the first stage
    stage_barrier();
    read_w(0, 0);
    read_x(SLOT, 0);
    uint32_t sa = 0;  // slot of A(s); B(s), A(s + 1), ... follow
    for (int s = 0; s < KF; ++s) {
      const uint32_t sb = wrap(sa + SLOT), sa1 = wrap(sa + 2 * SLOT), sb1 = wrap(sa + 3 * SLOT), sa2 = wrap(sa + 4 * SLOT);
      const uint8_t *b1 = bsrc(s + 1), *a2 = asrc(s + 2), *b2 = bsrc(s + 2);
      const uint32_t e1 = end_of(s + 1), e2 = end_of(s + 2);
      const uint32_t db1 = dst(sb1) + BI / 2 * 4096, da2 = dst(sa2), db2 = dst(sa);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (q == 3) {
          wait_copies_upto<AI>();  // stage s + 1 has landed
          stage_barrier();        // and everybody holds this stage's last operands
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (i == 0) read_w(q < 3 ? sa : sa1, (q + 1) & 3);
          if (i == 1) read_x(q < 3 ? sb : sb1, (q + 1) & 3);
          if (q == 1 || q == 2) {
            if (4 * (q - 1) + i < AI) copy_a(a2, 4 * (q - 1) + i, e2, da2 + (4 * (q - 1) + i) * 4096);
          }
          else if (i < BI / 2 && q == 0) copy_b(b1, BI / 2 + i, e1, db1 + i * 4096);
          else if (i < BI / 2) copy_b(b2, i, e2, db2 + i * 4096);
          mma_row(q, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      sa = sa1;
    }
    wait_copies_upto<0>();
    __syncthreads();
  }
  if constexpr (TAIL) {  // the last, partial stage: zeros behind the rows' ends
    const uint8_t *as = abase + (int64_t)KF * AB, *bs = bbase + (int64_t)KF * 128;
    const bool ain = KF * 64 + (AT ? achunk * 16 : chunk16 * 8) < p.K, in = KF * 64 + chunk16 * 8 < p.K;
    const uint8_t* z = reinterpret_cast<const uint8_t*>(kZeroChunk);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < AI) lds_copy16(ain ? as + aoff[j] : z, cw + j * 4096);
      if (j < BI) lds_copy16(in ? bs + boff[j] : z, cw + SLOT + j * 4096);
    }
    wait_copies_upto<0>();
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      read_w(0, q);
      read_x(SLOT, q);
#pragma unroll
      for (int i = 0; i < NI; ++i) mma_row(q, i);
    }
    __syncthreads();
  }
  vocab_epilogue<EPI, BM, 2, NI, MJ>(p, acc, smem, nt, m0, arows, brows, wn, wm);
}

// Joins the tiles of a token (one wavefront): lse, loss
__global__ __launch_bounds__(256) void vocab_loss_join_kernel(const float2* part, int tiles, int T, const float* tgt,
                                                              const void* targets, int targets_i64, int64_t ignore,
                                                              int64_t V, float* loss, float* lse) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= T) return;
  float2 v = make_float2(-__builtin_inff(), 0.0f);
  for (int i = lane; i < tiles; i += 64) v = lse_merge(v, part[(int64_t)i * T + t]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = lse_merge(v, make_float2(__shfl_xor(v.x, o, 64), __shfl_xor(v.y, o, 64)));
  if (lane) return;
  const int64_t tg = targets_i64 ? static_cast<const int64_t*>(targets)[t]
                                 : (int64_t) static_cast<const int32_t*>(targets)[t];
  const float all = lse_base(v.x) + logf(v.y);
  lse[t] = all;
  loss[t] = tg == ignore ? 0.0f : (tg >= 0 && tg < V ? all - tgt[t] : __builtin_nanf(""));
}

// Rows of codes -> bf16 rows; 8 codes per thread
template <int WT>
__global__ __launch_bounds__(256) void vocab_expand_kernel(const uint8_t* w, int64_t ldw, int64_t rows, int H8,
                                                           uint16_t* out, int64_t ldo) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * H8) return;
  const int64_t r = i / H8;
  const int c = (int)(i - r * H8) * 8;
  const uint2 d = *reinterpret_cast<const uint2*>(w + r * ldw + c);
  *reinterpret_cast<bf16x8*>(out + r * ldo + c) = codes8_to_bf16<WT>(d.x, d.y);
}

// The tokens with a gradient, in order: live[k] = t, place[t] = k or -1, *count. One
// workgroup, 1024 tokens at a time.
__global__ __launch_bounds__(1024) void vocab_live_kernel(int T, const void* targets, int targets_i64, int64_t ignore,
                                                          const float* g_loss, const float* g_lse, int32_t* live,
                                                          int32_t* place, int32_t* count) {
  __shared__ int part[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  int base = 0;
  for (int t0 = 0, side = 0; t0 < T; t0 += 1024, side ^= 1) {
    const int t = t0 + tid;
    bool is = false;
    if (t < T) {
      const int64_t tg = targets_i64 ? static_cast<const int64_t*>(targets)[t]
                                     : (int64_t) static_cast<const int32_t*>(targets)[t];
      is = (tg != ignore && g_loss[t] != 0.0f) || (g_lse && g_lse[t] != 0.0f);
    }
    const uint64_t m = __ballot(is);
    if (lane == 0) part[side][wave] = __popcll(m);
    __syncthreads();  // (the other side is written next)
    int before = base;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += part[side][w];
      base += part[side][w];
    }
    const int k = before + __popcll(m & below);
    if (is) live[k] = t;
    if (t < T) place[t] = is ? k : -1;
  }
  if (tid == 0) *count = base;
}

// Rows of x of the tokens with a gradient, one after the other, and zeros in dx
// (when not null) for the others. A workgroup per row.
__global__ __launch_bounds__(256) void vocab_gather_kernel(const uint16_t* x, int64_t ldx, int H, const int32_t* place,
                                                           uint16_t* out, uint16_t* dx, int64_t lddx) {
  const int64_t t = blockIdx.x;
  const int k = place[t];
  const uint4* src = reinterpret_cast<const uint4*>(x + t * ldx);
  uint4* dst = reinterpret_cast<uint4*>(k >= 0 ? out + (int64_t)k * H : dx + t * lddx);
  if (k < 0 && !dx) return;
  for (int c = threadIdx.x; c < H / 8; c += 256) dst[c] = k >= 0 ? src[c] : make_uint4(0, 0, 0, 0);
}

// Their rows [*count][C] -> out [C][ldo], columns from *count on zero. 64 x 64 tiles
// through LDS.
__global__ __launch_bounds__(256) void vocab_transpose_kernel(const uint8_t* src, int64_t ld, const int32_t* count, int C,
                                                              uint16_t* out, int64_t ldo) {
  __shared__ uint16_t tile[64][66];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, R = *count;
  const int tid = threadIdx.x;
  {
    const int c = (tid & 7) * 8;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = (tid >> 3) + 32 * k;
      const bool live = r0 + r < R && c0 + c < C;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (live) v = *reinterpret_cast<const uint4*>(src + (int64_t)(r0 + r) * ld + (int64_t)(c0 + c) * 2);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[r][c + i] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
    }
  }
  __syncthreads();
  const int r = (tid & 7) * 8;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = (tid >> 3) + 32 * k;
    if (c0 + c >= C) continue;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = tile[r + 2 * i][c] | (uint32_t)tile[r + 2 * i + 1][c] << 16;
    *reinterpret_cast<uint4*>(out + (int64_t)(c0 + c) * ldo + r0 + r) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// K of a tile up to which two workgroups per CU without a ring, whose copies, products
// and stores overlap each other's, beat the ring in tiles that store or reduce
// much. dw of 50021 x 2880: 64 tokens 66 us, by 256 x 256 106; 128 90, 122; 333
// 156, 178; 768 264, 272; 1024 333, 331. Probabilities of 333 tokens x 50021, H
// 512, 1024, 2048: 37, 58, 103, by the ring 49, 65, 99; logits 31, 56, 100, by the
// ring 36, 54, 90; of 2048 tokens 115, 204 (H 512, 1024), by the ring 138, 218.
constexpr int64_t kShortK = 1024;

// What a round of tiles over the 256 CUs costs: 256 x 256 and 256 x 192 by four
// wavefronts, 256 x 128 by eight. (333 tokens x 50021 x 2880, 2, 2 and 3 rounds:
// logits 142, 118, 136 us; probabilities 162, 128, 147.)
int tile_cost(int bm) { return bm == 256 ? 160 : (bm == 192 ? 130 : 100); }

// Tile of a problem of na A rows and nb B rows, by the rounds that it takes. (dw
// has no 192 and no 64: K rows of P are copied by 256 or 512 bytes.)
int vocab_bm(int64_t na, int64_t nb, bool dw = false) {
  const int64_t n = cdiv(na, (int64_t)kVN);
  if (nb <= 64 && !dw) return 64;
  if (nb <= 128) return 128;
  auto cost = [&](int bm) { return cdiv(n * cdiv(nb, (int64_t)bm), (int64_t)256) * tile_cost(bm); };
  const int big = dw || cost(256) <= cost(192) ? 256 : 192;
  return cost(big) <= cost(128) ? big : 128;
}

template <int EPI, int BM, int AT>
void launch_small(const VocabGemm& g, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((vocab_gemm_kernel<EPI, BM, AT>), grid, dim3(kVThreads), 0, st, g);
}

template <int EPI>
void launch_short(const VocabGemm& g, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((vocab_gemm_kernel<EPI, 128, 0, true>), grid, dim3(kVThreads), 0, st, g);
}

template <int EPI, int BM, int AT>
void launch_big_at(const VocabGemm& g, dim3 grid, hipStream_t st) {
  constexpr bool kLogits = EPI == VE_LSE || EPI == VE_PROB;  // (the K of dx and dw is a multiple of 64)
  if (kLogits && g.K % 64) hipLaunchKernelGGL((vocab_big_kernel<EPI, BM, AT, kLogits>), grid, dim3(kBThreads), 0, st, g);
  else hipLaunchKernelGGL((vocab_big_kernel<EPI, BM, AT, false>), grid, dim3(kBThreads), 0, st, g);
}
template <int EPI, int BM>
void launch_big(const VocabGemm& g, int at, dim3 grid, hipStream_t st) {
  if constexpr (EPI == VE_LSE) {
    if (at == 3) return launch_big_at<EPI, BM, 3>(g, grid, st);
    if (at == 4) return launch_big_at<EPI, BM, 4>(g, grid, st);
    if (at == 5) return launch_big_at<EPI, BM, 5>(g, grid, st);
  }
  launch_big_at<EPI, BM, 0>(g, grid, st);
}

// Whether a product whose tiles would be bm rows high takes the ones without a
// ring. at: type of the A rows, 0 bf16 or the codes' table type (logits)
template <int EPI>
bool ringless(int at, int64_t nb, int64_t K, int bm) {
  return EPI == VE_STORE ? bm == 128 || K <= kShortK : EPI != VE_SUM && at == 0 && nb > 128 && K <= kShortK;
}

template <int EPI>
void launch_gemm(VocabGemm g, int at, int bm, int slices, hipStream_t st) {
  const bool one = ringless<EPI>(at, g.nb, g.K, bm);
  if (one) bm = 128;
  g.n_tiles = cdiv(g.na, kVN);
  g.m_tiles = cdiv(g.nb, bm);
  const dim3 grid((unsigned)(cdiv(g.n_tiles * g.m_tiles, kXcds) * kXcds), (unsigned)slices);
  if (bm == 256) {
    launch_big<EPI, 256>(g, at, grid, st);
  } else if (bm == 192) {
    if constexpr (!tr_b(EPI)) launch_big<EPI, 192>(g, at, grid, st);
  } else if (at == 0) {
    if constexpr (EPI == VE_SUM) launch_small<EPI, 64, 0>(g, grid, st);
    else if (EPI == VE_STORE || one) launch_short<EPI>(g, grid, st);
    else if constexpr (EPI != VE_STORE) bm == 128 ? launch_small<EPI, 128, 0>(g, grid, st) : launch_small<EPI, 64, 0>(g, grid, st);
  } else if constexpr (EPI == VE_LSE) {
    if (at == 3) bm == 128 ? launch_small<EPI, 128, 3>(g, grid, st) : launch_small<EPI, 64, 3>(g, grid, st);
    else if (at == 4) bm == 128 ? launch_small<EPI, 128, 4>(g, grid, st) : launch_small<EPI, 64, 4>(g, grid, st);
    else bm == 128 ? launch_small<EPI, 128, 5>(g, grid, st) : launch_small<EPI, 64, 5>(g, grid, st);
  }
}

void launch_expand(int wt, const uint8_t* w, int64_t ldw, int64_t rows, int64_t H, uint16_t* out, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(rows * (H / 8), (int64_t)256));
  if (wt == 3) hipLaunchKernelGGL(vocab_expand_kernel<3>, grid, dim3(256), 0, st, w, ldw, rows, (int)(H / 8), out, H);
  else if (wt == 4) hipLaunchKernelGGL(vocab_expand_kernel<4>, grid, dim3(256), 0, st, w, ldw, rows, (int)(H / 8), out, H);
  else hipLaunchKernelGGL(vocab_expand_kernel<5>, grid, dim3(256), 0, st, w, ldw, rows, (int)(H / 8), out, H);
}

struct LossArgs {
  const void* x;
  int64_t ldx, T;
  const void* w;
  int wtype;
  int64_t ldw;
  const float* row_scale;
  int64_t V, H;
  const void* targets;
  int targets_i64;
  int64_t ignore;
};

// sizes whose tile counts, and the threads of their grids, fit 32 bits
constexpr int64_t kMaxTokens = (int64_t)1 << 20, kMaxVocab = (int64_t)1 << 24, kMaxHidden = (int64_t)1 << 16;


bool loss_sizes_ok(int64_t T, int64_t V, int64_t H) {
  return T >= 0 && T <= kMaxTokens && V > 0 && V <= kMaxVocab && H > 0 && H <= kMaxHidden && H % 8 == 0 &&
         cdiv(V, (int64_t)kVN) * cdiv(T, (int64_t)128) <= ((int64_t)1 << 22);
}

int loss_args_ok(const LossArgs& a) {
  if (!loss_sizes_ok(a.T, a.V, a.H)) return 0;
  if (a.wtype != 0 && (a.wtype < 3 || a.wtype > 5)) return 0;
  if (a.ldx < a.H || a.ldw < a.H || a.ldx % 8 || a.ldw % 8) return 0;
  if (a.ldx >= (int64_t)1 << 22 || a.ldw >= (int64_t)1 << 22) return 0;  // 256 rows of a tile within 32-bit offsets
  if (a.T == 0) return 1;
  if (!a.x || !a.w || !a.targets || ((a.wtype != 0) != (a.row_scale != nullptr))) return 0;
  if ((reinterpret_cast<uintptr_t>(a.x) & 15) || (reinterpret_cast<uintptr_t>(a.w) & (a.wtype ? 7 : 15))) return 0;
  return 1;
}

// Whether codes go to the tiles as they are stored: whole 16-byte chunks. (Else
// pieces are expanded first. e4m3, 131072 x 4096: 192 tokens 0.19 ms as stored,
// 0.78 expanded; 1024 0.92, 1.23; 4096 3.61, 3.90. int8, whose expansion takes
// the most instructions, 32003 x 2880: 1024 tokens 200 us, 248; 4096 793, 785.)
bool codes_direct(const void* w, int64_t ldw, int64_t H) {
  return H % 16 == 0 && ldw % 16 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
}

// Table rows of a piece of the forward pass where codes are expanded first: 128
// MB of them
int64_t loss_piece(int64_t V, int64_t H) {
  return std::min(up(V, kVN), std::max<int64_t>((int64_t)(64 << 20) / H / kVN * kVN, kVN));
}

int64_t loss_layout(int64_t T, int64_t V, int64_t H, int wtype, int64_t (&off)[3]) {
  int64_t at = 0;
  off[0] = at;  // partial (maximum, sum) of every tile
  at += up(cdiv(V, (int64_t)kVN) * T * 8, 256);
  off[1] = at;  // the targets' logits
  at += up(T * 4, 256);
  off[2] = at;  // expanded rows
  if (wtype) at += up(loss_piece(V, H) * H * 2, 256);
  return at;
}

// Table rows of a piece of the gradients: P, and for codes the expanded rows, of
// a piece take up to 128 MB each
int64_t grad_piece(int64_t T, int64_t V, int64_t H, int wtype) {
  const int64_t width = std::max<int64_t>(up(T, 64), wtype ? H : 0);
  return std::min(up(V, kVN), std::max<int64_t>((int64_t)(64 << 20) / width / kVN * kVN, kVN));
}

// dx of a piece: T x H outputs, a K axis as long as the piece. As many K slices
// as fill the CUs, of at least 512 (V 50021, H 2880 without the split: 489 us at
// 64 tokens, 685 at 333; with it 87 and 104). Tile height by the padded rows'
// cost; 64 by eight wavefronts up to 64 tokens (1, 64 tokens: 72, 87 us; of 192:
// 84, 94), and above no 128 by eight (100, 333 tokens: 98, 200 us; of 192: 100,
// 104): eight wavefronts' transposed reads keep LDS busy.
struct DxPlan {
  int bm, slices, kslice;
};
DxPlan dx_plan(int64_t T, int64_t H, int64_t K) {
  DxPlan d{};
  auto cost = [&](int bm) { return cdiv(T, (int64_t)bm) * tile_cost(bm); };
  d.bm = T <= 64 ? 64 : (cost(256) <= cost(192) ? 256 : 192);
  const int64_t tiles = cdiv(H, (int64_t)kVN) * cdiv(T, (int64_t)d.bm);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(256 / tiles, K / 512));
  d.kslice = (int)up(cdiv(K, want), 64);
  d.slices = (int)cdiv(K, (int64_t)d.kslice);
  return d;
}

// P, x transposed, float32 sums, K slices, expanded rows, x gathered, the tokens' list
int64_t grad_layout(int64_t T, int64_t V, int64_t H, int wtype, int need_dx, int need_dw, int64_t (&off)[7]) {
  const int64_t Vc = grad_piece(T, V, H, wtype), Tw = up(T, 64);
  const bool pieces = Vc < V;
  int64_t at = 0;
  off[0] = at;
  at += up(T * Vc * 2, 256);
  off[1] = at;
  if (need_dw) at += up(H * Tw * 2, 256);
  off[2] = at;
  if (need_dx && pieces) at += up(T * H * 4, 256);
  off[3] = at;
  if (need_dx) {
    const DxPlan d = dx_plan(T, H, up(std::min(Vc, V), 64));
    if (d.slices > 1) at += up(d.slices * T * H * 4, 256);
  }
  off[4] = at;
  if (wtype) at += up(Vc * H * 2, 256);
  off[5] = at;
  at += up(T * H * 2, 256);
  off[6] = at;
  return at + up((2 * T + 1) * 4, 256);
}

}  // namespace

// See include/qmoe.h for the contracts.
extern "C" int qmoe_vocab_loss_workspace_size(int64_t T, int64_t V, int64_t H, int wtype, int64_t* bytes) {
  if (!loss_sizes_ok(T, V, H) || (wtype != 0 && (wtype < 3 || wtype > 5)) || !bytes) return QMOE_ERR_ARG;
  int64_t off[3];
  *bytes = loss_layout(T, V, H, wtype, off);
  return QMOE_OK;
}

extern "C" int qmoe_vocab_loss(const void* x, int64_t ldx, int64_t T, const void* w, int wtype, int64_t ldw,
                               const float* row_scale, int64_t V, int64_t H, const void* targets, int targets_i64,
                               int64_t ignore_index, float* loss, float* lse, void* workspace, int64_t ws_bytes,
                               hipStream_t stream) {
  const LossArgs a{x, ldx, T, w, wtype, ldw, row_scale, V, H, targets, targets_i64, ignore_index};
  if (!loss_args_ok(a)) return QMOE_ERR_ARG;
  if (T == 0) return QMOE_OK;
  if (!loss || !lse) return QMOE_ERR_ARG;
  int64_t off[3];
  if (!workspace || ws_bytes < loss_layout(T, V, H, wtype, off)) return QMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  VocabGemm g{};
  g.b = static_cast<const uint8_t*>(x);
  g.ldb = ldx * 2;
  g.nb = (int)T;
  g.K = (int)H;
  g.V = V;
  g.targets = targets;
  g.targets_i64 = targets_i64;
  g.ignore = ignore_index;
  g.part = reinterpret_cast<float2*>(ws + off[0]);
  g.tgt = reinterpret_cast<float*>(ws + off[1]);
  const bool direct = wtype && codes_direct(w, ldw, H);
  const int64_t Vc = wtype && !direct ? loss_piece(V, H) : V;
  for (int64_t v0 = 0; v0 < V; v0 += Vc) {
    const uint8_t* rows = static_cast<const uint8_t*>(w) + v0 * ldw * (wtype ? 1 : 2);
    const int64_t n = std::min(Vc, V - v0);
    g.a = rows;
    g.lda = ldw * (wtype ? 1 : 2);
    if (wtype && !direct) {
      uint16_t* e = reinterpret_cast<uint16_t*>(ws + off[2]);
      launch_expand(wtype, rows, ldw, n, H, e, stream);
      g.a = reinterpret_cast<const uint8_t*>(e);
      g.lda = H * 2;
    }
    g.na = (int)n;
    g.v0 = v0;
    g.row_scale = row_scale ? row_scale + v0 : nullptr;
    g.part_tile = (int)(v0 / kVN);
    launch_gemm<VE_LSE>(g, direct ? wtype : 0, vocab_bm(n, T), 1, stream);
  }
  hipLaunchKernelGGL(vocab_loss_join_kernel, dim3((unsigned)cdiv(T, (int64_t)4)), dim3(256), 0, stream, g.part,
                     (int)cdiv(V, (int64_t)kVN), (int)T, g.tgt, targets, targets_i64, ignore_index, V, loss, lse);
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_vocab_loss_plan(int64_t T, int64_t V, int64_t H, int wtype, qmoe_vocab_loss_tiles* plan) {
  if (!loss_sizes_ok(T, V, H) || T == 0 || (wtype != 0 && (wtype < 3 || wtype > 5)) || !plan) return QMOE_ERR_ARG;
  const bool direct = wtype && H % 16 == 0;
  const int at = direct ? wtype : 0;
  auto pieces = [&](int64_t Vc) { return (int32_t)cdiv(V, Vc); };
  auto tile = [](bool one, int bm) { return one ? 1 : bm; };
  const int64_t lc = wtype && !direct ? loss_piece(V, H) : V, gc = grad_piece(T, V, H, wtype), ln = std::min(lc, V),
                gn = std::min(gc, V), Tw = up(T, 64);
  const int lbm = vocab_bm(ln, T), pbm = vocab_bm(gn, T), wbm = vocab_bm(H, gn, true);
  const DxPlan dx = dx_plan(T, H, up(gn, 64));
  plan->logits = tile(ringless<VE_LSE>(at, T, H, lbm), lbm);
  plan->loss_pieces = pieces(lc);
  plan->probs = tile(ringless<VE_PROB>(0, T, H, pbm), pbm);
  plan->dx = dx.bm;
  plan->dx_slices = dx.slices;
  plan->dw = tile(ringless<VE_STORE>(0, gn, Tw, wbm), wbm);
  plan->grad_pieces = pieces(gc);
  return QMOE_OK;
}

extern "C" int qmoe_vocab_loss_grad_workspace_size(int64_t T, int64_t V, int64_t H, int wtype, int need_dx, int need_dw,
                                                   int64_t* bytes) {
  if (!loss_sizes_ok(T, V, H) || (wtype != 0 && (wtype < 3 || wtype > 5)) || !bytes) return QMOE_ERR_ARG;
  int64_t off[7];
  *bytes = grad_layout(T, V, H, wtype, need_dx, need_dw, off);
  return QMOE_OK;
}

extern "C" int qmoe_vocab_loss_grad(const void* x, int64_t ldx, int64_t T, const void* w, int wtype, int64_t ldw,
                                    const float* row_scale, int64_t V, int64_t H, const void* targets, int targets_i64,
                                    int64_t ignore_index, const float* lse, const float* g_loss, const float* g_lse,
                                    void* dx, int64_t lddx, void* dw, int64_t lddw, void* workspace, int64_t ws_bytes,
                                    hipStream_t stream) {
  const LossArgs a{x, ldx, T, w, wtype, ldw, row_scale, V, H, targets, targets_i64, ignore_index};
  if (!loss_args_ok(a) || T == 0 || !lse || !g_loss || (!dx && !dw)) return QMOE_ERR_ARG;
  if (dw && wtype) return QMOE_ERR_ARG;  // codes have no gradient
  if (dx && (lddx < H || lddx % 8 || (reinterpret_cast<uintptr_t>(dx) & 15))) return QMOE_ERR_ARG;
  if (dw && (lddw < H || lddw % 8 || (reinterpret_cast<uintptr_t>(dw) & 15))) return QMOE_ERR_ARG;
  int64_t off[7];
  if (!workspace || ws_bytes < grad_layout(T, V, H, wtype, dx != nullptr, dw != nullptr, off)) return QMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t Vc = grad_piece(T, V, H, wtype), Tw = up(T, 64);
  uint16_t* P = reinterpret_cast<uint16_t*>(ws + off[0]);
  uint16_t* XT = reinterpret_cast<uint16_t*>(ws + off[1]);
  uint16_t* X = reinterpret_cast<uint16_t*>(ws + off[5]);
  int32_t *live = reinterpret_cast<int32_t*>(ws + off[6]), *place = live + T, *count = place + T;
  hipLaunchKernelGGL(vocab_live_kernel, dim3(1), dim3(1024), 0, stream, (int)T, targets, targets_i64, ignore_index, g_loss,
                     g_lse, live, place, count);
  hipLaunchKernelGGL(vocab_gather_kernel, dim3((unsigned)T), dim3(256), 0, stream, static_cast<const uint16_t*>(x), ldx, (int)H,
                     place, X, static_cast<uint16_t*>(dx), lddx);
  if (dw)
    hipLaunchKernelGGL(vocab_transpose_kernel, dim3((unsigned)(Tw / 64), (unsigned)cdiv(H, (int64_t)64)), dim3(256), 0, stream,
                       reinterpret_cast<const uint8_t*>(X), H * 2, count, (int)H, XT, Tw);
  for (int64_t v0 = 0; v0 < V; v0 += Vc) {
    const uint8_t* rows = static_cast<const uint8_t*>(w) + v0 * ldw * (wtype ? 1 : 2);
    const int64_t n = std::min(Vc, V - v0), np = up(n, 64);
    VocabGemm g{};
    g.a = rows;
    g.lda = ldw * (wtype ? 1 : 2);
    if (wtype) {
      uint16_t* e = reinterpret_cast<uint16_t*>(ws + off[4]);
      launch_expand(wtype, rows, ldw, n, H, e, stream);
      g.a = reinterpret_cast<const uint8_t*>(e);
      g.lda = H * 2;
    }
    g.na = (int)n;
    g.b = reinterpret_cast<const uint8_t*>(X);
    g.ldb = H * 2;
    g.live = live;
    g.count = count;
    g.nb = (int)T;
    g.K = (int)H;
    g.row_scale = row_scale ? row_scale + v0 : nullptr;
    g.v0 = v0;
    g.V = V;
    g.targets = targets;
    g.targets_i64 = targets_i64;
    g.ignore = ignore_index;
    g.lse = lse;
    g.g_loss = g_loss;
    g.g_lse = g_lse;
    g.p = P;
    g.ldp = Vc;
    launch_gemm<VE_PROB>(g, 0, vocab_bm(n, T), 1, stream);
    if (dx) {
      VocabGemm d{};
      d.live = live;
      d.count = count;
      d.a = g.a;
      d.lda = g.lda;
      d.na = (int)H;
      d.b = reinterpret_cast<const uint8_t*>(P);
      d.ldb = Vc * 2;
      d.nb = (int)T;
      d.K = (int)np;
      d.kr = (int)n;
      d.sum = reinterpret_cast<float*>(ws + off[2]);
      d.ldsum = H;
      d.first = v0 == 0;
      d.last = v0 + Vc >= V;
      d.y = static_cast<uint16_t*>(dx);
      d.ldy = lddx;
      const DxPlan plan = dx_plan(T, H, up(std::min(Vc, V), 64));
      const int slices = (int)cdiv(np, (int64_t)plan.kslice);
      if (slices > 1) {
        d.kslice = plan.kslice;
        d.slices = reinterpret_cast<float*>(ws + off[3]);
      }
      launch_gemm<VE_SUM>(d, 0, plan.bm, slices, stream);
      if (slices > 1)
        hipLaunchKernelGGL(vocab_slices_kernel, dim3((unsigned)cdiv(T * H / 4, (int64_t)256)), dim3(256), 0, stream, d, slices);
    }
    if (dw) {
      VocabGemm d{};
      d.live = live;
      d.count = count;
      d.a = reinterpret_cast<const uint8_t*>(XT);
      d.lda = Tw * 2;
      d.na = (int)H;
      d.b = reinterpret_cast<const uint8_t*>(P);
      d.ldb = Vc * 2;
      d.nb = (int)n;
      d.K = (int)Tw;
      d.kr = (int)T;
      d.y = static_cast<uint16_t*>(dw) + v0 * lddw;
      d.ldy = lddw;
      launch_gemm<VE_STORE>(d, 0, vocab_bm(H, n, true), 1, stream);
    }
  }
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
