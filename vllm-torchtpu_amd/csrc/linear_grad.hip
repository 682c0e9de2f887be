// Gradients of a linear layer y = x w^T + bias whose input waited in 8 bits:
//
//   dx[t, k] = sum_n dy[t, n] w[n, k],   dw[n, k] = sum_t dy[t, n] x8[t, k],   dbias[n] = sum_t dy[t, n]
//
// What bounds it: two products of 2 T N K operations on the bf16 matrix cores, or,
// for few tokens, one read of w and one write of dw. The 8-bit values' scales
// change along the summed axis, so the codes are multiplied as bf16 (exact: 4 of
// its 8 significant bits): of up to 512 tokens by the tiles without a ring themselves
// (linear_codes), for other tiles and of more tokens expanded and transposed once on the
// way to dw (4096 x 4096: 14 us).
//
// The products (the layer's own among them) are the same tile: 256 "A" rows x BM "B"
// rows of a workgroup, a ring of LDS stages of 64 k filled by direct copies, and for
// the gradients an operand that lies across K (gemm_across.h):
//   dx : A = columns of w (across), B = rows of dy
//   dw : A = columns of x8 (rows of its transpose, padded with zeros to 64 k, or codes across K), B = columns
//        of dy (across)
//   y  : A = rows of w, B = rows of x (neither across)
// The last stage copies zeros where K has ended. Sums are float32; a K axis that
// is long for the number of tiles is cut into slices, added in order.

#include <algorithm>

#include "../../include/qmoe.h"
#include "eight_bits.h"
#include "gemm_across.h"

namespace {

constexpr int kAN = 256;  // A rows of a tile

QMOE_HD int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct LinearGemm {
  const uint8_t* a;  // rows along K [na][lda bytes], or across it [K][lda]
  int64_t lda;
  int na;
  const uint8_t* b;
  int64_t ldb;
  int nb;
  int K;
  int n_tiles, m_tiles;
  uint16_t* y;  // [nb][ldy]
  int64_t ldy;
  int kslice;   // K split: slice z takes the K range from z * kslice on and leaves float32 sums in [z][nb][na]
  float* slices;
  const float* bias;  // of the A rows, or nullptr
  const uint8_t* scales;  // of A where it is codes [K][na], bytes [K][na / 32]
};

// B row t of the 64 that a round holds, A row n of it at n ^ vg_row_swz(t): 8
// consecutive A rows per thread and store. 64 KB of LDS, once no copy or read uses it,
// or 128 (HALVES: wavefronts wm = 0 and 1 have the same rows, of half of k each).
template <int THREADS, int NI, int MJ, bool HALVES = false>
__device__ __forceinline__ void linear_epilogue(const LinearGemm& p, f32x16 (&acc)[NI][MJ], uint8_t* smem, int n0, int m0,
                                                int arows, int brows, int wn, int wm) {
  const int tid = threadIdx.x, lane = tid & 63, rl = lane & 31, kh = lane >> 5;
  float *reg = reinterpret_cast<float*>(smem), *reg2 = reg + 64 * kAN;  // [64][256]
  float* to = HALVES && wm ? reg2 : reg;
  constexpr int ROUND = HALVES ? 2 : 1;  // blocks of a wavefront in 64 rows
#pragma unroll
  for (int j = 0; j < MJ / ROUND; ++j) {
    if (64 * j >= brows) break;
    if (j) __syncthreads();  // the rows before have been read
    const int n1 = opaque_v(wn * NI * 32 + kh * 4);
#pragma unroll
    for (int jj = 0; jj < ROUND; ++jj)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n1 + i * 32 + q * 8, tl = (HALVES ? jj : wm) * 32 + rl;
          const f32x16& v = acc[i][j * ROUND + jj];
          *reinterpret_cast<float4*>(to + tl * kAN + (n ^ vg_row_swz(tl))) =
              make_float4(v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]);
        }
    __syncthreads();
    constexpr int CH = kAN / 8;
    const int c = (tid % CH) * 8;
#pragma unroll 2
    for (int t = tid / CH; t < 64; t += THREADS / CH) {
      const int64_t row = m0 + 64 * j + t;
      if (64 * j + t >= brows) break;
      if (c >= arows) continue;  // (A rows come in multiples of 8)
      const int at = t * kAN + (c ^ vg_row_swz(t)), at4 = t * kAN + ((c + 4) ^ vg_row_swz(t));
      float4 lo = *reinterpret_cast<const float4*>(reg + at), hi = *reinterpret_cast<const float4*>(reg + at4);
      if constexpr (HALVES) {
        const float4 l = *reinterpret_cast<const float4*>(reg2 + at), h = *reinterpret_cast<const float4*>(reg2 + at4);
        lo.x += l.x, lo.y += l.y, lo.z += l.z, lo.w += l.w;
        hi.x += h.x, hi.y += h.y, hi.z += h.z, hi.w += h.w;
      }
      if (p.kslice) {
        float4* dst = reinterpret_cast<float4*>(p.slices + ((int64_t)blockIdx.y * p.nb + row) * p.na + n0 + c);
        dst[0] = lo;
        dst[1] = hi;
      } else {
        float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (p.bias) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += p.bias[n0 + c + k];
        }
        *reinterpret_cast<uint4*>(p.y + row * p.ldy + n0 + c) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      }
    }
  }
}

// This workgroup's slice of K
template <bool TRA, bool TRB, bool CODES = false>
__device__ __forceinline__ void linear_slice(LinearGemm& p) {
  if (!p.kslice) return;
  const int64_t k0 = (int64_t)blockIdx.y * p.kslice;
  p.a += TRA ? k0 * p.lda : k0 * 2;
  if constexpr (CODES) p.scales += k0 * (p.na / 32);
  p.b += TRB ? k0 * p.ldb : k0 * 2;
  p.K = (int)min((int64_t)p.kslice, p.K - k0);
}

// Tiles of 256 x BM (64 or 128) by eight wavefronts of 64 x 64. HALVES (64 B rows): two
// of them have the same block, of half of every stage's k each, and their sums are added
// at the end: 64 KB of operands from LDS per stage where wavefronts of 64 x 32 read 96.
// 777 tokens, 4096 x 4096 forward / dx, each alone, 38.1 / 39.5 -> 35.5 / 34.9 us (208 tiles of
// 256 CUs, 740 TFLOP/s; 37.1 / 38.3 in a step, 35.4 / 37.4 at best); of 128 rows the same 2
// to 9 % slower. ONE: a stage at a time, without a ring, so that two workgroups share a CU
// (that case's dw 30). CODES: the A operand is x8
// itself, codes and scale bytes across K, expanded on the way to LDS (a thread 32
// columns of a row): no transposed copy of x8 before the product, whose launch and
// bytes count where the sums are short.
template <bool TRA, bool TRB, int BM, bool ONE, bool CODES>
__global__ __launch_bounds__(512, ONE ? 4 : 2) void linear_small_kernel(const LinearGemm args) {
  constexpr bool HALVES = BM == 64;
  constexpr int NI = 2, MJ = HALVES ? 2 : BM / 64, WB = kAN * 128, STG = WB + BM * 128;
  constexpr int RING = ONE ? 1 : (163840 / STG < 6 ? 163840 / STG : 6), EPILOGUE = HALVES ? 131072 : 65536;
  __shared__ __align__(1024) uint8_t smem[RING * STG > EPILOGUE ? RING * STG : EPILOGUE];
  static_assert(ONE ? sizeof(smem) <= 81920 : RING >= 3 && sizeof(smem) <= 163840, "workgroups of a CU, ring");
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  LinearGemm p = args;
  linear_slice<TRA, TRB, CODES>(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 3, wm = wave >> 2, rl = lane & 31, kh = lane >> 5;
  int mt, nt;
  if (!tile_dense(blockIdx.x, p.m_tiles, p.n_tiles, mt, nt)) return;
  const int n0 = nt * kAN, m0 = mt * BM;
  const int arows = min(kAN, p.na - n0), brows = min(BM, p.nb - m0);

  // copies: one instruction = 8 rows x 128 bytes (lane -> row l >> 3, slot l & 7,
  // chunk c of row r at c ^ vg_swz(r)), or 1 KB of K rows; wavefront w moves the
  // groups w, w + 8, ...; rows and columns past the end repeat the last
  constexpr int WI = WB / 8192, XI = BM / 64;
  constexpr bool COPY_A = TRA && !CODES;               // the operand across K that is copied
  constexpr int TB = COPY_A ? kAN * 2 : BM * 2, TL = TB / 16;  // bytes, lanes of its K row
  static_assert(!COPY_A || !TRB, "one copied operand across K");
  static_assert(!CODES || (ONE && TRA && TRB), "codes");
  const int chunk = (lane & 7) ^ ((lane >> 3) ^ (wave & 1));
  const int trow = lane / TL, tchunk = (lane % TL) ^ tr_swz<TB>(wave * (64 / TL) + trow);
  const uint32_t tcol = (uint32_t)min(tchunk, (COPY_A ? arows : brows) / 8 - 1) * 16;
  const uint8_t* abase = TRA ? p.a + n0 * 2 : p.a + (int64_t)n0 * p.lda;
  const uint8_t* bbase = TRB ? p.b + m0 * 2 : p.b + (int64_t)m0 * p.ldb;
  const int64_t astep = TRA ? 64 * p.lda : 128, bstep = TRB ? 64 * p.ldb : 128;
  uint32_t aoff[WI], boff[XI];
  auto krow = [&](int j) { return (wave + 8 * j) * (64 / TL) + trow; };  // of a stage, of copy j of the operand across K
#pragma unroll
  for (int j = 0; j < WI; ++j)
    aoff[j] = CODES ? 0u : TRA ? (uint32_t)krow(j) * (uint32_t)p.lda + tcol
                  : (uint32_t)min((wave + 8 * j) * 8 + (lane >> 3), arows - 1) * (uint32_t)p.lda + chunk * 16;
#pragma unroll
  for (int j = 0; j < XI; ++j)
    boff[j] = TRB ? (uint32_t)krow(j) * (uint32_t)p.ldb + tcol
                  : (uint32_t)min((wave + 8 * j) * 8 + (lane >> 3), brows - 1) * (uint32_t)p.ldb + chunk * 16;
  const int KF = p.K / 64, tail = p.K % 64;  // whole stages, k of the last
  const uint32_t cw = lds0 + wave * 1024;
  // stage s to slot `slot` (stages past the last whole one copy it again, into
  // slots nobody reads)
  auto copy_stage = [&](int s, int slot) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(cw + slot * STG);
    const int k = min(s, KF - 1);
    const uint8_t *as = uniform_ptr(abase + k * astep), *bs = uniform_ptr(bbase + k * bstep);
    if constexpr (!CODES) {
#pragma unroll
      for (int j = 0; j < WI; ++j) lds_copy16(as, aoff[j], d + j * 8192);
    }
#pragma unroll
    for (int j = 0; j < XI; ++j) lds_copy16(bs, boff[j], d + WB + j * 8192);
  };
  // the last, partial stage, with zeros where K has ended
  auto copy_tail = [&]() {
    const uint8_t *as = abase + KF * astep, *bs = bbase + KF * bstep, *z = reinterpret_cast<const uint8_t*>(kZeroChunk);
    if constexpr (!CODES) {
#pragma unroll
      for (int j = 0; j < WI; ++j)
        lds_copy16((TRA ? krow(j) : chunk * 8) < tail ? as + aoff[j] : z, __builtin_amdgcn_readfirstlane(cw + j * 8192));
    }
#pragma unroll
    for (int j = 0; j < XI; ++j)
      lds_copy16((TRB ? krow(j) : chunk * 8) < tail ? bs + boff[j] : z,
                 __builtin_amdgcn_readfirstlane(cw + WB + j * 8192));
  };

  f32x16 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  union B8 {
    uint4 u;
    bf16x8 v;
  };
  B8 wf[2][NI], xf[2][MJ];
  const uint32_t alane = tr_lane<kAN * 2>(lane), blane = tr_lane<BM * 2>(lane);
  // operands of step q (16 k) of a stage
  constexpr int QS = HALVES ? 2 : 4;  // steps of a wavefront in a stage
  auto read_q = [&](int slot, int u) {
    const uint8_t* s = smem + slot * STG;
    const int q = HALVES ? 2 * wm + u : u;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if constexpr (TRA) wf[u & 1][i].u = tr_read<kAN * 2>(s + q * 32 * kAN + (alane ^ (wn * NI + i) * 64));
      else wf[u & 1][i].u =
          *reinterpret_cast<const uint4*>(s + (wn * 64 + i * 32 + rl) * 128 + ((2 * q + kh) ^ vg_swz(rl)) * 16);
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      const int b = HALVES ? j : 2 * j + wm;  // block of 32 B rows
      if constexpr (TRB) xf[u & 1][j].u = tr_read<BM * 2>(s + WB + q * 32 * BM + (blane ^ b * 64));
      else xf[u & 1][j].u =
          *reinterpret_cast<const uint4*>(s + WB + (b * 32 + rl) * 128 + ((2 * q + kh) ^ vg_swz(rl)) * 16);
    }
  };
  auto mma = [&](int u) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[u & 1][i].v, xf[u & 1][j].v, acc[i][j], 0, 0, 0);
  };
  auto one_stage = [&]() {
    wait_copies_upto<0>();
    __syncthreads();
#pragma unroll
    for (int u = 0; u < QS; ++u) {
      read_q(0, u);
      mma(u);
    }
    __syncthreads();
  };
  // Ring: all but the last MFMA step run while the next step's operands are read;
  // then the next stage's copies have landed -> barrier: everybody holds this
  // stage's last operands, so that its slot takes the copies of stage s + RING ->
  // the last step, while the next stage's first operands are read.
  if constexpr (ONE) {
    // codes: row k of the stage, 32 columns from 32 g on; zeros behind the ends
    const int k = tid >> 3, g = tid & 7;
    const bool col = 32 * g < arows;
    const uint8_t *cp = p.a + (int64_t)k * p.lda + n0 + 32 * g, *sp = p.scales + (int64_t)k * (p.na / 32) + n0 / 32 + g;
    uint8_t* to = smem + k * kAN * 2 + ((g * 64) ^ (tr_swz<kAN * 2>(k) * 16));
    for (int s = 0; s < KF + (tail != 0); ++s) {
      uint4 c[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      uint32_t scale = 0;
      if constexpr (CODES) {
        if (col && 64 * s + k < p.K) {
          const uint4* at = reinterpret_cast<const uint4*>(cp + (int64_t)s * 64 * p.lda);
          c[0] = at[0];
          c[1] = at[1];
          scale = sp[(int64_t)s * 64 * (p.na / 32)];
        }
      }
      if (s < KF) copy_stage(s, 0);
      else copy_tail();
      if constexpr (CODES) {
        const uint32_t* d = reinterpret_cast<const uint32_t*>(c);
        const float f = bits_f32(scale << 23);  // (the conversion takes the exponent alone, 0 as 2^-127)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          union {
            bf16x2 h[4];
            uint4 u;
          } v;
          v.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d[2 * j], f, false);
          v.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d[2 * j], f, true);
          v.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d[2 * j + 1], f, false);
          v.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d[2 * j + 1], f, true);
          *reinterpret_cast<uint4*>(to + j * 16) = v.u;
        }
      }
      one_stage();
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
      for (int u = 0; u < QS - 1; ++u) {
        read_q(slot, u + 1);
        mma(u);
      }
      wait_copies_upto<(RING - 2) * (WI + XI)>();
      stage_barrier();
      copy_stage(s + RING, slot);
      asm volatile("" ::: "memory");
      read_q(next, 0);
      mma(QS - 1);
      slot = next;
    }
    wait_copies_upto<0>();
    __syncthreads();
  }
  if (!ONE && tail) {
    copy_tail();
    one_stage();
  }
  linear_epilogue<512, NI, MJ, HALVES>(p, acc, smem, n0, m0, arows, brows, wn, wm);
}

// The same without slices in 32 KB of LDS (at `region`), waiting for none of the copies
// that are in flight to the rest of it: a round takes 64 B rows of two of a wavefront's
// four blocks, row t's float n at n ^ 4 (t & 31), and leaves 128 bytes of each row.
template <int NI, int MJ>
__device__ __forceinline__ void linear_rows(const LinearGemm& p, f32x16 (&acc)[NI][MJ], uint8_t* region, int n0, int m0,
                                            int arows, int brows, int wn, int wm) {
  static_assert(NI == 4, "two halves");
  const int tid = threadIdx.x, lane = tid & 63, rl = lane & 31, kh = lane >> 5;
  float* reg = reinterpret_cast<float*>(region);  // [64][128]
  float* to = reg + (wm * 32 + rl) * 128;
  const int c = (tid & 15) * 8, t0 = tid >> 4, n = (c >> 6) * 128 + (c & 63);
  uint16_t* y = p.y + (int64_t)(m0 + t0) * p.ldy + n0 + n;
  float bias[2][8] = {};
  if (p.bias) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n + 64 * h < arows)
#pragma unroll
        for (int k = 0; k < 8; ++k) bias[h][k] = p.bias[n0 + n + 64 * h + k];
  }
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    if (64 * j >= brows) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (j || h) stage_barrier();  // the rows before have been read
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& v = acc[2 * h + i][j];
          *reinterpret_cast<float4*>(to + ((wn * 64 + i * 32 + q * 8 + kh * 4) ^ (4 * rl))) =
              make_float4(v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]);
        }
      stage_barrier();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = t0 + 16 * k;
        if (64 * j + t < brows && n + 64 * h < arows) {  // (A rows come in multiples of 8)
          const float4 lo = *reinterpret_cast<const float4*>(reg + t * 128 + (c ^ (4 * (t & 31))));
          const float4 hi = *reinterpret_cast<const float4*>(reg + t * 128 + ((c + 4) ^ (4 * (t & 31))));
          const float* b = bias[h];
          *reinterpret_cast<uint4*>(y + (int64_t)(64 * j + 16 * k) * p.ldy + 64 * h) =
              make_uint4(pack_bf16(lo.x + b[0], lo.y + b[1]), pack_bf16(lo.z + b[2], lo.w + b[3]),
                         pack_bf16(hi.x + b[4], hi.y + b[5]), pack_bf16(hi.z + b[6], hi.w + b[7]));
        }
      }
    }
  }
  stage_barrier();  // the last rows have been read
}

// The same products in tiles of 256 x BM (256 or 192) by four wavefronts of 4 x
// BM / 64 blocks, one per SIMD, the sums in accumulation registers: a wavefront of
// 128 x 128 reads 32 KB of operands from LDS per 64 MFMAs where one of 64 x 64
// reads 32 per 32, and eight of those fill LDS's 128 bytes per cycle.
//
// Stages of 64 k: 32 KB of A rows and up to 32 KB of B rows, in a ring of five such
// slots (all of LDS): A(s), B(s), A(s + 1), B(s + 1), A(s + 2). At the barrier of
// stage s every wavefront holds its last operands, and the stage's two slots
// take B(s + 2) and A(s + 3). The copies go out four per MFMA step, one at a time
// between the MFMAs.
// A workgroup goes on to the tile gridDim.x further: its first stages follow the
// last of the tile before in the ring, so that they are there when that tile's results
// have been stored (of two stages and more; one of a single stage has a tile only).
// 4096 tokens, 4096 x 28672, seven tiles each: forward 727 us (755 with a workgroup per
// tile) = 1323 TFLOP/s, dw 729 (740); one tile each, dx 709 = 1357 TFLOP/s. The matrix
// cores are busy for 70 to 75 % of the cycles, and the clock falls with more. Results
// stored straight from the registers, 64 bytes of a row at a time, cost 838 where rows
// lie a multiple of 4 KB apart.
// TAIL: K is not a multiple of 64 (an instance of its own: the extra stage costs
// the others registers), a tile per workgroup.
template <bool TRA, bool TRB, int BM, bool TAIL>
__global__ __launch_bounds__(256, 1) void linear_big_kernel(const LinearGemm args) {
  constexpr int NI = 4, MJ = BM / 64, AI = 8, BI = 2 * MJ;  // a wavefront's copies of A and B per stage
  constexpr uint32_t SLOT = kAN * 128, RING = 5 * SLOT;
  constexpr int TB = 512, TL = 32;  // bytes, lanes of a K row of the operand across K
  static_assert(!TRB || BM == 256, "K rows of 512 bytes");
  static_assert(!TRA || !TRB, "one operand across K");
  __shared__ __align__(1024) uint8_t smem[RING];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  LinearGemm p = args;
  linear_slice<TRA, TRB>(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = wave >> 1, rl = lane & 31, kh = lane >> 5;
  struct Tile {
    int n0, m0, arows, brows;
    const uint8_t *a, *b;
  };
  const int tiles = (int)up(p.m_tiles * p.n_tiles, kXcds);
  auto tile_of = [&](int b, Tile& t) {
    int mt, nt;
    if (b >= tiles || !tile_dense(b, p.m_tiles, p.n_tiles, mt, nt)) return false;
    t.n0 = nt * kAN;
    t.m0 = mt * BM;
    t.arows = min(kAN, p.na - t.n0);
    t.brows = min(BM, p.nb - t.m0);
    t.a = TRA ? p.a + t.n0 * 2 : p.a + (int64_t)t.n0 * p.lda;
    t.b = TRB ? p.b + t.m0 * 2 : p.b + (int64_t)t.m0 * p.ldb;
    return true;
  };
  int block = blockIdx.x;
  Tile cur, nxt;
  if (!tile_of(block, cur)) return;

  // copies as in the kernel above; wavefront w moves the groups w, w + 4, ...
  const int chunk = (lane & 7) ^ ((lane >> 3) ^ (wave & 1));
  const int trow = lane / TL, tchunk = (lane % TL) ^ tr_swz<TB>(2 * wave + trow);
  const int64_t astep = TRA ? 64 * p.lda : 128, bstep = TRB ? 64 * p.ldb : 128;
  uint32_t aoff[AI], boff[BI];
  auto place = [&](bool across, int j, int rows, int64_t ld) {
    if (across) return (uint32_t)(2 * (wave + 4 * j) + trow) * (uint32_t)ld + (uint32_t)min(tchunk, rows / 8 - 1) * 16;
    return (uint32_t)min((wave + 4 * j) * 8 + (lane >> 3), rows - 1) * (uint32_t)ld + chunk * 16;
  };
#pragma unroll
  for (int j = 0; j < AI; ++j) aoff[j] = place(TRA, j, cur.arows, p.lda);
#pragma unroll
  for (int j = 0; j < BI; ++j) boff[j] = place(TRB, j, cur.brows, p.ldb);
  const int KF = p.K / 64, tail = p.K % 64;
  const uint32_t cw = lds0 + wave * 1024;
  union B8 {
    uint4 u;
    bf16x8 v;
  };
  B8 wf[2][NI], xf[2][MJ];
  const uint32_t wpo = (uint32_t)(wn * NI * 4096 + rl * 128), xpo = (uint32_t)(wm * 4096 + rl * 128);
  const uint32_t tlane = tr_lane<TB>(lane) ^ (TRA ? wn * NI * 64 : wm * 64);
  auto read_w = [&](uint32_t slot, int q) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if constexpr (TRA) wf[q & 1][i].u = tr_read<TB>(smem + slot + q * 16 * TB + (tlane ^ i * 64));
      else wf[q & 1][i].u =
          *reinterpret_cast<const uint4*>(smem + slot + wpo + i * 4096 + ((2 * q + kh) ^ vg_swz(rl)) * 16);
  };
  auto read_x = [&](uint32_t slot, int q) {
#pragma unroll
    for (int j = 0; j < MJ; ++j)
      if constexpr (TRB) xf[q & 1][j].u = tr_read<TB>(smem + slot + q * 16 * TB + (tlane ^ j * 128));
      else xf[q & 1][j].u =
          *reinterpret_cast<const uint4*>(smem + slot + xpo + j * 8192 + ((2 * q + kh) ^ vg_swz(rl)) * 16);
  };
  f32x16 acc[NI][MJ];
  // (by a product of zeros: sums set to zero one register at a time pass through others)
  auto clear = [&]() {
    bf16x8 no = {};
    const f32x16 zero = {};
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        asm volatile("" : "+v"(no));  // (one product each: one for all would be copied)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(no, no, zero, 0, 0, 0);
      }
  };
  auto mma_row = [&](int q, int i) {
#pragma unroll
    for (int j = 0; j < MJ; ++j)
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[q & 1][i].v, xf[q & 1][j].v, acc[i][j], 0, 0, 0);
  };
  if constexpr (TAIL) clear();
  if (!TAIL || KF > 0) {
    bool more = !TAIL && KF > 1 && tile_of(block + gridDim.x, nxt);
    auto dst = [&](uint32_t slot) { return (uint32_t)__builtin_amdgcn_readfirstlane(cw + slot); };
    const uint8_t *a2 = uniform_ptr(cur.a), *b1 = uniform_ptr(cur.b), *b2;
#pragma unroll
    for (int j = 0; j < AI; ++j) lds_copy16(a2, aoff[j], dst(0) + j * 4096);
#pragma unroll
    for (int j = 0; j < BI; ++j) lds_copy16(b1, boff[j], dst(SLOT) + j * 4096);
    if (KF > 1) {
      a2 += astep;
      b1 += bstep;
    }
#pragma unroll
    for (int j = 0; j < AI; ++j) lds_copy16(a2, aoff[j], dst(2 * SLOT) + j * 4096);
#pragma unroll
    for (int j = 0; j < BI / 2; ++j) lds_copy16(b1, boff[j], dst(3 * SLOT) + j * 4096);
    a2 += astep;
    b2 = b1 + bstep;
    wait_copies_upto<AI + BI / 2>();  // the first stage
    stage_barrier();
    read_w(0, 0);
    read_x(SLOT, 0);
    uint32_t sa = 0, sb = SLOT, sa1 = 2 * SLOT, sb1 = 3 * SLOT, sa2 = 4 * SLOT;  // slots of A(s), B(s), A(s + 1), ...
    for (;;) {
      if constexpr (!TAIL) clear();
      for (int s = 0; s < KF; ++s) {
        if (s + 2 >= KF) {  // the next tile's stages; without one the last again, into slots nobody reads
          if (!more) {
            a2 -= astep;
            b2 -= bstep;
          } else if (s + 2 == KF) {
            a2 = uniform_ptr(nxt.a);
            b2 = uniform_ptr(nxt.b);
#pragma unroll
            for (int j = 0; j < AI; ++j) aoff[j] = place(TRA, j, nxt.arows, p.lda);
#pragma unroll
            for (int j = 0; j < BI / 2; ++j) boff[j] = place(TRB, j, nxt.brows, p.ldb);
          } else {
#pragma unroll
            for (int j = BI / 2; j < BI; ++j) boff[j] = place(TRB, j, nxt.brows, p.ldb);
          }
        }
        const uint32_t db1 = dst(sb1) + BI / 2 * 4096, da2 = dst(sa2), db2 = dst(sa);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q == 3) {
            wait_copies_upto<AI>();  // stage s + 1 has landed
            stage_barrier();         // and everybody holds this stage's last operands
          }
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            if (i == 0) read_w(q < 3 ? sa : sa1, (q + 1) & 3);
            if (i == 1) read_x(q < 3 ? sb : sb1, (q + 1) & 3);
            if (q == 1 || q == 2) lds_copy16(a2, aoff[4 * (q - 1) + i], da2 + (4 * (q - 1) + i) * 4096);
            else if (i < BI / 2 && q == 0) lds_copy16(b1, boff[BI / 2 + i], db1 + i * 4096);
            else if (i < BI / 2) lds_copy16(b2, boff[i], db2 + i * 4096);
            mma_row(q, i);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        a2 += astep;
        b1 = b2;
        b2 += bstep;
        const uint32_t s0 = sa, s1 = sb;
        sa = sa1, sb = sb1, sa1 = sa2, sb1 = s0, sa2 = s1;
      }
      if (TAIL || !more) wait_copies_upto<0>();
      if (TAIL || p.kslice) break;
      linear_rows<NI, MJ>(p, acc, smem + sa2, cur.n0, cur.m0, cur.arows, cur.brows, wn, wm);  // (A(s + 2)'s slot is free)
      if (!more) return;
      cur = nxt;
      block += gridDim.x;
      more = tile_of(block + gridDim.x, nxt);
    }
    __syncthreads();
  }
  if constexpr (TAIL) {  // the last, partial stage, with zeros where K has ended
    const uint8_t *as = cur.a + KF * astep, *bs = cur.b + KF * bstep, *z = reinterpret_cast<const uint8_t*>(kZeroChunk);
#pragma unroll
    for (int j = 0; j < AI; ++j)
      lds_copy16((TRA ? 2 * (wave + 4 * j) + trow : chunk * 8) < tail ? as + aoff[j] : z,
                 __builtin_amdgcn_readfirstlane(cw + j * 4096));
#pragma unroll
    for (int j = 0; j < BI; ++j)
      lds_copy16((TRB ? 2 * (wave + 4 * j) + trow : chunk * 8) < tail ? bs + boff[j] : z,
                 __builtin_amdgcn_readfirstlane(cw + SLOT + j * 4096));
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
  linear_epilogue<256, NI, MJ>(p, acc, smem, cur.n0, cur.m0, cur.arows, cur.brows, wn, wm);
}

// The K slices -> bf16 rows
__global__ __launch_bounds__(256) void linear_slices_kernel(const float* s, int slices, int64_t rows, int na,
                                                            const float* bias, uint16_t* y, int64_t ldy) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, n = rows * na;
  if (i >= n) return;
  const int64_t row = i / na;
  const int c = (int)(i - row * na);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int z = 0; z < slices; ++z) {
    const float4 a = *reinterpret_cast<const float4*>(s + z * n + i);
    v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
  }
  if (bias) v.x += bias[c], v.y += bias[c + 1], v.z += bias[c + 2], v.w += bias[c + 3];
  *reinterpret_cast<uint2*>(y + row * ldy + c) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// Codes [T][K] -> bf16 [K][Tw], columns from T on zero. 64 x 64 tiles through LDS.
__global__ __launch_bounds__(256) void linear_expand_kernel(const uint8_t* codes, const uint8_t* scales, int T, int K,
                                                            uint16_t* out, int64_t Tw) {
  __shared__ uint16_t tile[64][66];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, tid = threadIdx.x;
  {
    const int c = (tid & 7) * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (tid >> 3) + 32 * h, t = r0 + r;
      float v[8] = {};
      if (t < T && c0 + c < K)
        qmoe_row::decode8(*reinterpret_cast<const uint2*>(codes + (int64_t)t * K + c0 + c),
                          scales[(int64_t)t * (K / 32) + (c0 + c) / 32], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[r][c + i] = f32_to_bf16(v[i]);
    }
  }
  __syncthreads();
  const int r = (tid & 7) * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = (tid >> 3) + 32 * h;
    if (c0 + c >= K) continue;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (uint32_t)tile[r + 2 * i][c] | (uint32_t)tile[r + 2 * i + 1][c] << 16;
    *reinterpret_cast<uint4*>(out + (int64_t)(c0 + c) * Tw + r0 + r) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// Column sums of dy: workgroup (x, y) adds the rows y, y + gridDim.y, ... of 64
// columns, eight threads of 8 of them, 32 rows at a time -> parts [gridDim.y][N], or,
// alone, the sums themselves
__device__ __forceinline__ void put_bias(void* out, int f32, int n, float v) {
  if (f32) static_cast<float*>(out)[n] = v;
  else static_cast<uint16_t*>(out)[n] = f32_to_bf16(v);
}
__global__ __launch_bounds__(256) void linear_bias_kernel(const uint16_t* dy, int64_t lddy, int64_t T, int N,
                                                          float* parts, void* out, int f32) {
  __shared__ float s[32][65];
  const int c = (threadIdx.x & 7) * 8, r = threadIdx.x >> 3, n = blockIdx.x * 64 + c;
  float v[8] = {};
  if (n < N)
    for (int64_t t = (int64_t)blockIdx.y * 32 + r; t < T; t += (int64_t)gridDim.y * 32) {
      float d[8];
      qmoe_row::load8<qmoe_row::RT_BF16, true>(dy + t * lddy, n, N, d);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += d[k];
    }
#pragma unroll
  for (int k = 0; k < 8; ++k) s[r][c + k] = v[k];
  __syncthreads();
  if (threadIdx.x >= 64 || (int)(blockIdx.x * 64 + threadIdx.x) >= N) return;
  float sum = 0.0f;
#pragma unroll 8
  for (int k = 0; k < 32; ++k) sum += s[k][threadIdx.x];
  const int at = blockIdx.x * 64 + threadIdx.x;
  if (gridDim.y == 1) put_bias(out, f32, at, sum);
  else parts[(int64_t)blockIdx.y * N + at] = sum;
}

__global__ __launch_bounds__(256) void linear_bias_join_kernel(const float* parts, int n_parts, int N, void* out,
                                                               int f32) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float v = 0.0f;
#pragma unroll 8
  for (int k = 0; k < n_parts; ++k) v += parts[(int64_t)k * N + n];
  put_bias(out, f32, n, v);
}

// ---------------------------------------------------------------- launches

// Which operand of a product lies across K
enum LinearMode { LM_FORWARD = 0, LM_DX = 1, LM_DW = 2 };

// Tile rows (1: of 128, without a ring), K slices and their length of a product of
// na A rows, nb B rows and K
struct LinearPlan {
  int bm, slices, kslice;
};
// The least time of a model: rounds of the tiles on the chip times (stages times
// a stage's time + the rest of a tile), and for K slices their sums' way to memory
// and back. Times from sweeps of every tile and 1 to 16 slices over 16 sizes (1 to
// 8192 tokens, 256 x 1024 to 4096 x 28672), with a workgroup per tile; the plan's own time
// was within 5 % of the best of the sweep for most, 14 % at most. Both sides, us: 4096
// tokens x 4096 x 28672 forward / dx / dw tiles of 256 723 / 676 / 734, of 128 887 / 816 / 875;
// 777 x 4096 x 4096 dw without a ring 36.9, 256 rows 39.3; forward of 512 x 7168 x 7168 64 rows
// 58.7, 256 rows in 4 slices 65.7; of 200 x 1024 x 4096 64 rows 13.2, in 4 slices 18.9; of
// 64 x 4096 x 4096 16.8 in 8 slices.
LinearPlan linear_plan(int mode, int64_t na, int64_t nb, int64_t K) {
  struct Tile {
    int bm, cus, stage, fixed;  // workgroups of a round, ns of a stage and of the rest of a tile
  };
  // (dw: few stages and the most to write; without a ring one workgroup's stores run under the other's products)
  constexpr Tile kAlong[] = {{256, 256, 1680, 6000}, {192, 256, 1290, 5000}, {128, 256, 1050, 4000}, {1, 512, 2000, 5000},
                             {64, 256, 510, 5500}};
  constexpr Tile kDw[] = {{256, 256, 1680, 11000}, {128, 256, 1050, 8000}, {1, 512, 1900, 5000}, {64, 256, 700, 4000}};
  LinearPlan best{};
  int64_t least = INT64_MAX;
  const int64_t stages = cdiv(K, (int64_t)64), n = cdiv(na, (int64_t)kAN);
  for (int i = 0; i < (mode == LM_DW ? 4 : 5); ++i) {
    const Tile& t = mode == LM_DW ? kDw[i] : kAlong[i];
    const int64_t tiles = n * cdiv(nb, (int64_t)(t.bm == 1 ? 128 : t.bm));
    for (int64_t want = 1; want <= 16 && want <= stages; ++want) {
      const int64_t per = cdiv(stages, want), slices = cdiv(stages, per);
      // (each XCD takes an eighth of the tiles, of every slice)
      int64_t ns = cdiv(cdiv(tiles, (int64_t)kXcds) * slices, (int64_t)t.cus / kXcds) * (per * t.stage + t.fixed);
      if (slices > 1) ns += 3000 + slices * 300 + slices * na * nb * 8 / 7000;
      if (ns < least) {
        least = ns;
        best = LinearPlan{t.bm, (int)slices, (int)(per * 64)};
      }
    }
  }
  return best;
}

// Whether dw takes the codes as they are: tiles without a ring of up to 512 tokens. (The
// plan's times leave the transposed copy out, so that other tiles of so few tokens still
// make it, where their own time is less: 19 tokens x 2048 x 2048.)
// Every tile of N expands them again: 19 tokens x 2880 x 2880 10.4 us (13.4 with the
// transposed copy), 200 x 7168 x 2048 19.6 (22.1), 512 x 4096 x 4096 29.7 (30.0), but 777
// x 4096 x 4096 42.7 (38.9), 1500 x 14336 x 4096 235 (180).
bool linear_codes(int64_t N, int64_t K, int64_t T) { return T <= 512 && linear_plan(LM_DW, K, N, T).bm == 1; }

// (several tiles per workgroup where no K slice is a single stage)
template <bool TRA, bool TRB, int BM>
void launch_big(const LinearGemm& g, dim3 grid, hipStream_t st) {
  if (g.K % 64 == 0 && grid.y == 1 && g.K > 64 && grid.x > 256) grid.x = 256;
  if (g.K % 64) hipLaunchKernelGGL((linear_big_kernel<TRA, TRB, BM, true>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((linear_big_kernel<TRA, TRB, BM, false>), grid, dim3(256), 0, st, g);
}

template <int MODE>
void launch_linear(LinearGemm g, uint8_t* ws, hipStream_t st) {
  constexpr bool TRA = MODE == LM_DX, TRB = MODE == LM_DW;
  const LinearPlan d = linear_plan(MODE, g.na, g.nb, g.K);
  if (d.slices > 1) {
    g.kslice = d.kslice;
    g.slices = reinterpret_cast<float*>(ws);
  }
  g.n_tiles = cdiv(g.na, kAN);
  g.m_tiles = cdiv(g.nb, d.bm == 1 ? 128 : d.bm);
  const dim3 grid((unsigned)up((int64_t)g.n_tiles * g.m_tiles, kXcds), (unsigned)d.slices);
  if (d.bm == 256) launch_big<TRA, TRB, 256>(g, grid, st);
  else if (d.bm == 192) { if constexpr (!TRB) launch_big<TRA, TRB, 192>(g, grid, st); }
  else if (d.bm == 64) hipLaunchKernelGGL((linear_small_kernel<TRA, TRB, 64, false, false>), grid, dim3(512), 0, st, g);
  else if (d.bm == 128) hipLaunchKernelGGL((linear_small_kernel<TRA, TRB, 128, false, false>), grid, dim3(512), 0, st, g);
  else if (MODE == LM_DW && g.scales)
    hipLaunchKernelGGL((linear_small_kernel<TRA || MODE == LM_DW, TRB, 128, true, MODE == LM_DW>), grid, dim3(512), 0, st, g);
  else hipLaunchKernelGGL((linear_small_kernel<TRA, TRB, 128, true, false>), grid, dim3(512), 0, st, g);
  if (d.slices > 1)
    hipLaunchKernelGGL(linear_slices_kernel, dim3((unsigned)cdiv((int64_t)g.nb * g.na / 4, (int64_t)256)), dim3(256), 0, st,
                       g.slices, d.slices, (int64_t)g.nb, g.na, g.bias, g.y, g.ldy);
}

int64_t slice_bytes(int mode, int64_t na, int64_t nb, int64_t K) {
  const LinearPlan d = linear_plan(mode, na, nb, K);
  return d.slices > 1 ? up(4 * d.slices * na * nb, 256) : 0;
}

// Parts of the column sums: 128 rows of each at least (up to 255 tokens one launch), 2048
// workgroups at most. 128 rows x 4096 2.7 us (parts of 32 rows 4.8), 1500 x 1024 5.1 (of 512
// rows 7.5, one part 8.9), 4096 x 4096 8.1 (9.7, 22), but 256 x 4096 4.8 (3.3); 65536 x 4096 106
// (512 workgroups 152, 8192 107), but 4096 x 28672 46 (35, 40).
int bias_parts(int64_t T, int64_t N) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(T / 128, cdiv((int64_t)2048, cdiv(N, (int64_t)64))));
}

// x8 transposed, K slices (dx's, then dw's), bias parts
int64_t linear_layout(int64_t T, int64_t N, int64_t K, int need_dx, int need_dw, int need_dbias, int64_t (&off)[3]) {
  int64_t at = 0;
  off[0] = at;
  if (need_dw && !linear_codes(N, K, T)) at += up(K * up(T, 64) * 2, 256);
  off[1] = at;
  int64_t s = need_dx ? slice_bytes(LM_DX, K, T, N) : 0;
  if (need_dw) s = std::max(s, slice_bytes(LM_DW, K, N, T));
  at += s;
  off[2] = at;
  if (need_dbias) at += up(4 * N * bias_parts(T, N), 256);
  return at;
}

bool linear_sizes_ok(int64_t T, int64_t N, int64_t K) {
  return T >= 1 && T <= ((int64_t)1 << 20) && N >= 8 && N <= ((int64_t)1 << 18) && K >= 32 && K <= ((int64_t)1 << 16) &&
         N % 8 == 0 && K % 32 == 0;
}

// (256 rows of a tile, or 64 of a stage, lie within 32-bit offsets)
constexpr int64_t kMaxPitch = (int64_t)1 << 22;

bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// See include/qmoe.h for the contract.
extern "C" int qmoe_linear_workspace_size(int64_t T, int64_t N, int64_t K, int64_t* bytes) {
  if (!linear_sizes_ok(T, N, K) || !bytes) return QMOE_ERR_ARG;
  *bytes = slice_bytes(LM_FORWARD, N, T, K);
  return QMOE_OK;
}

extern "C" int qmoe_linear(const void* x, int64_t ldx, int64_t T, int64_t N, int64_t K, const void* w, int64_t ldw,
                           const float* bias, void* y, uint8_t* codes, uint8_t* scales, void* workspace,
                           int64_t ws_bytes, hipStream_t stream) {
  if (!linear_sizes_ok(T, N, K) || !x || !w || !y || ldx < K || ldx % 8 || ldx >= kMaxPitch || ldw < K || ldw % 8 ||
      ldw >= kMaxPitch || !at16(x) || !at16(w) || !at16(y))
    return QMOE_ERR_ARG;
  if (codes && (!scales || !at16(codes))) return QMOE_ERR_ARG;
  const int64_t need = slice_bytes(LM_FORWARD, N, T, K);
  if (need && (!workspace || !at16(workspace) || ws_bytes < need)) return QMOE_ERR_WORKSPACE;
  if (codes)
    if (const int st = qmoe_pack_8bit(x, ldx, T, K, codes, scales, stream)) return st;
  LinearGemm g{};
  g.a = static_cast<const uint8_t*>(w);
  g.lda = ldw * 2;
  g.na = (int)N;
  g.b = static_cast<const uint8_t*>(x);
  g.ldb = ldx * 2;
  g.nb = (int)T;
  g.K = (int)K;
  g.y = static_cast<uint16_t*>(y);
  g.ldy = N;
  g.bias = bias;
  launch_linear<LM_FORWARD>(g, static_cast<uint8_t*>(workspace), stream);
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_linear_plan(int64_t T, int64_t N, int64_t K, qmoe_linear_tiles* plan) {
  if (!linear_sizes_ok(T, N, K) || !plan) return QMOE_ERR_ARG;
  const LinearPlan y = linear_plan(LM_FORWARD, N, T, K), dx = linear_plan(LM_DX, K, T, N), dw = linear_plan(LM_DW, K, N, T);
  *plan = qmoe_linear_tiles{y.bm, y.slices, dx.bm, dx.slices, dw.bm, dw.slices, linear_codes(N, K, T)};
  return QMOE_OK;
}

extern "C" int qmoe_linear_grad_workspace_size(int64_t T, int64_t N, int64_t K, int need_dx, int need_dw, int need_dbias,
                                               int64_t* bytes) {
  if (!linear_sizes_ok(T, N, K) || !bytes) return QMOE_ERR_ARG;
  int64_t off[3];
  *bytes = linear_layout(T, N, K, need_dx, need_dw, need_dbias, off);
  return QMOE_OK;
}

extern "C" int qmoe_linear_grad(const void* dy, int64_t lddy, int64_t T, int64_t N, int64_t K, const void* w, int64_t ldw,
                                const uint8_t* codes, const uint8_t* scales, void* dx, void* dw, void* dbias,
                                int dbias_f32, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  if (!linear_sizes_ok(T, N, K) || !dy || lddy < N || lddy % 8 || lddy >= kMaxPitch || !at16(dy)) return QMOE_ERR_ARG;
  if (dx && (!w || ldw < K || ldw % 8 || ldw >= kMaxPitch || !at16(w) || !at16(dx))) return QMOE_ERR_ARG;
  if (dw && (!codes || !scales || !at16(codes) || !at16(dw))) return QMOE_ERR_ARG;
  int64_t off[3];
  const int64_t need = linear_layout(T, N, K, dx != nullptr, dw != nullptr, dbias != nullptr, off);
  if (need && (!workspace || !at16(workspace) || ws_bytes < need)) return QMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (dx) {
    LinearGemm g{};
    g.a = static_cast<const uint8_t*>(w);
    g.lda = ldw * 2;
    g.na = (int)K;
    g.b = static_cast<const uint8_t*>(dy);
    g.ldb = lddy * 2;
    g.nb = (int)T;
    g.K = (int)N;
    g.y = static_cast<uint16_t*>(dx);
    g.ldy = K;
    launch_linear<LM_DX>(g, ws + off[1], stream);
  }
  if (dw) {
    LinearGemm g{};
    if (linear_codes(N, K, T)) {
      g.a = codes;
      g.lda = K;
      g.scales = scales;
    } else {
      const int64_t Tw = up(T, 64);
      uint16_t* xt = reinterpret_cast<uint16_t*>(ws + off[0]);
      hipLaunchKernelGGL(linear_expand_kernel, dim3((unsigned)(Tw / 64), (unsigned)cdiv(K, (int64_t)64)), dim3(256), 0,
                         stream, codes, scales, (int)T, (int)K, xt, Tw);
      g.a = reinterpret_cast<const uint8_t*>(xt);
      g.lda = Tw * 2;
    }
    g.na = (int)K;
    g.b = static_cast<const uint8_t*>(dy);
    g.ldb = lddy * 2;
    g.nb = (int)N;
    g.K = (int)T;
    g.y = static_cast<uint16_t*>(dw);
    g.ldy = K;
    launch_linear<LM_DW>(g, ws + off[1], stream);
  }
  if (dbias) {
    float* parts = reinterpret_cast<float*>(ws + off[2]);
    const int n_parts = bias_parts(T, N);
    hipLaunchKernelGGL(linear_bias_kernel, dim3((unsigned)cdiv(N, (int64_t)64), (unsigned)n_parts), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(dy), lddy, T, (int)N, parts, dbias, dbias_f32);
    if (n_parts > 1)
      hipLaunchKernelGGL(linear_bias_join_kernel, dim3((unsigned)cdiv(N, (int64_t)256)), dim3(256), 0, stream, parts, n_parts,
                         (int)N, dbias, dbias_f32);
  }
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
