// Rows of the vocabulary table: lookup with scaling, and its gradient by
// sorted tokens.
//
//   out[n]  = round(scale * s[id[n]] * w[id[n]])       (s: one scale per row of a 1-byte table,
//                                                       rounded to the output type first)
//   dw[v]   = round(scale * sum over n with id[n] == v of g[n]), sums in float32 in the order of n,
//                                                       grouped by where the sorted ids are cut
//
// Both are bound by HBM: the lookup reads and writes N rows, the gradient reads
// N rows and writes V (all of a fresh gradient; only the touched ones when it
// is added into an existing one).
// Measured: 16384 rows of 7168 bf16 67 us (168 MiB read, repeated rows come from
// cache, 224 written: 6.1 TB/s), 8 rows of 4096 e4m3 3.5; gradient of 16384 rows
// of 4096 bf16 into a fresh 131072-row one 11 (sort) + 211 (sums and zeros, 125
// MiB read, 1035 written: 5.8 TB/s) + 19 (join).

#include <algorithm>

#include "../../include/qmoe.h"
#include "qmoe_common.h"

namespace {

enum { VT_BF16 = 0, VT_F32 = 1, VT_F16 = 2, VT_E4M3 = 3, VT_INT8 = 4, VT_E5M2 = 5 };

template <int T>
constexpr int vt_bytes() { return T == VT_F32 ? 4 : (T == VT_BF16 || T == VT_F16 ? 2 : 1); }

QMOE_HD int vt_size(int t) { return t == VT_F32 ? 4 : (t == VT_BF16 || t == VT_F16 ? 2 : 1); }

// NV values at `src` (aligned to their whole size when NV > 1) as float32, exactly
template <int T, int NV>
__device__ __forceinline__ void vt_load(const void* src, float (&v)[NV]) {
  constexpr int NB = NV * vt_bytes<T>();
  union {
    uint8_t b[NB];
    uint16_t h[NB / 2 > 0 ? NB / 2 : 1];
    float f[NB / 4 > 0 ? NB / 4 : 1];
    _Float16 e[NB / 2 > 0 ? NB / 2 : 1];
    uint4 q[NB / 16 > 0 ? NB / 16 : 1];
    uint2 d;
  } u;
  if constexpr (NB % 16 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) u.q[i] = static_cast<const uint4*>(src)[i];
  } else if constexpr (NB == 8) {
    u.d = *static_cast<const uint2*>(src);
  } else if constexpr (NB == 4) {
    u.f[0] = *static_cast<const float*>(src);
  } else if constexpr (NB == 2) {
    u.h[0] = *static_cast<const uint16_t*>(src);
  } else {
    u.b[0] = *static_cast<const uint8_t*>(src);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (T == VT_BF16) v[i] = bf16_to_f32(u.h[i]);
    else if constexpr (T == VT_F32) v[i] = u.f[i];
    else if constexpr (T == VT_F16) v[i] = (float)u.e[i];
    else if constexpr (T == VT_E4M3) v[i] = e4m3_to_f32(u.b[i]);
    else if constexpr (T == VT_E5M2) v[i] = e5m2_to_f32(u.b[i]);
    else v[i] = (float)(int8_t)u.b[i];
  }
}

// Round to nearest, ties to even, to the output type (one rounding)
template <int T>
__device__ __forceinline__ float vt_round(float f) {
  if constexpr (T == VT_BF16) return bf16_round(f);
  else if constexpr (T == VT_F16) return (float)(_Float16)f;
  else return f;
}

template <int T, int NV>
__device__ __forceinline__ void vt_store(void* dst, const float (&v)[NV]) {
  constexpr int NB = NV * vt_bytes<T>();
  union {
    uint16_t h[NB / 2];
    float f[NB / 4 > 0 ? NB / 4 : 1];
    _Float16 e[NB / 2];
    uint4 q[NB / 16 > 0 ? NB / 16 : 1];
  } u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (T == VT_BF16) u.h[i] = f32_to_bf16(v[i]);
    else if constexpr (T == VT_F32) u.f[i] = v[i];
    else u.e[i] = (_Float16)v[i];
  }
  if constexpr (NB % 16 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) static_cast<uint4*>(dst)[i] = u.q[i];
  } else if constexpr (NB == 4) {
    *static_cast<float*>(dst) = u.f[0];
  } else {
    *static_cast<uint16_t*>(dst) = u.h[0];
  }
}

__device__ __forceinline__ int64_t token_id(const void* ids, int i64, int64_t n) {
  return i64 ? static_cast<const int64_t*>(ids)[n] : (int64_t) static_cast<const int32_t*>(ids)[n];
}

// ---------------------------------------------------------------- lookup

struct LookupParams {
  const void* ids;
  int ids_i64;
  int64_t N, V, H;
  const uint8_t* w;
  int64_t ldw;  // bytes
  const float* row_scale;
  float scale;
  uint8_t* out;
  int64_t ldo;  // bytes
};

constexpr int kLookupThreads = 256;

// Workgroup (x, y): row x, columns from y * span on; a thread takes NV columns
// every 256 * NV of them, up to four such pieces, all loaded before the first
// is stored. An id outside the table gives a row of NaN and reads nothing.
template <int WT, int OT, int NV>
__global__ __launch_bounds__(kLookupThreads) void vocab_lookup_kernel(const LookupParams p, int64_t span) {
  const int64_t n = blockIdx.x;
  const int64_t id = token_id(p.ids, p.ids_i64, n);
  const bool ok = id >= 0 && id < p.V;
  constexpr bool kScaled = WT == VT_E4M3 || WT == VT_INT8 || WT == VT_E5M2;
  const float s = ok ? (kScaled ? vt_round<OT>(p.row_scale[id]) : 1.0f) : __builtin_nanf("");
  const uint8_t* row = p.w + (ok ? id : 0) * p.ldw;
  uint8_t* out = p.out + n * p.ldo;
  const int64_t c1 = min(p.H, ((int64_t)blockIdx.y + 1) * span);
  constexpr int kStep = kLookupThreads * NV, kPieces = 4;
  for (int64_t c0 = (int64_t)blockIdx.y * span + threadIdx.x * NV; c0 < c1; c0 += (int64_t)kPieces * kStep) {
    float v[kPieces][NV];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int64_t c = c0 + j * kStep;
      if (c < c1 && ok) {
        vt_load<WT, NV>(row + c * vt_bytes<WT>(), v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[j][i] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int64_t c = c0 + j * kStep;
      if (c < c1) {
        // code * row scale is rounded once by the store when scale == 1: an
        // 8-bit code times a 16-bit-format scale is exact in float32
#pragma unroll
        for (int i = 0; i < NV; ++i) v[j][i] = v[j][i] * s * p.scale;
        vt_store<OT, NV>(out + c * vt_bytes<OT>(), v[j]);
      }
    }
  }
}

template <int WT, int OT>
void launch_lookup(const LookupParams& p, bool vec, hipStream_t st) {
  const int nv = vec ? 8 : 1;
  // whole rows per workgroup, or pieces of one step where the rows alone
  // leave CUs without a workgroup (8 rows of 4096 e4m3: 4.1 us by whole rows, 3.5
  // by pieces; 16384 of 7168 bf16: 67 and 80)
  const int64_t step = (int64_t)kLookupThreads * nv, pieces = cdiv(p.H, step);
  const int64_t ny = p.N * cdiv(pieces, (int64_t)4) >= 1024 ? cdiv(pieces, (int64_t)4) : pieces;
  const int64_t span = cdiv(pieces, ny) * step;
  const dim3 grid((unsigned)p.N, (unsigned)cdiv(p.H, span));
  if (vec) hipLaunchKernelGGL((vocab_lookup_kernel<WT, OT, 8>), grid, dim3(kLookupThreads), 0, st, p, span);
  else hipLaunchKernelGGL((vocab_lookup_kernel<WT, OT, 1>), grid, dim3(kLookupThreads), 0, st, p, span);
}

template <int WT>
void launch_lookup_out(const LookupParams& p, int ot, bool vec, hipStream_t st) {
  if (ot == VT_BF16) launch_lookup<WT, VT_BF16>(p, vec, st);
  else if (ot == VT_F16) launch_lookup<WT, VT_F16>(p, vec, st);
  else launch_lookup<WT, VT_F32>(p, vec, st);
}

// ---------------------------------------------------------------- gradient
//
// 1. sort: workgroup b owns the table rows [b * rpw, ...). It reads every id
//    (from L2 after the first workgroup: N ids cost less than the N gradient
//    rows that follow), counts those below its rows, which is where its
//    stretch of the sorted order begins, and places its own ones by (row, n):
//    wavefront w scans the w-th part of the ids in order, so that the counts
//    per (wavefront, row), summed in that order, make the placement stable and
//    the order of the later sums fixed for given ids. No workgroup waits for another.
// 2. sum: workgroup c adds the gradient rows of the sorted entries
//    [c * chunk, ...), whatever rows they belong to, so that a token that
//    makes up a tenth of a batch costs as much per entry as a rare one. Runs
//    of equal ids inside the chunk are finished; a run that crosses the
//    chunk's start or end leaves float32 partial sums. Further workgroups
//    write the zeros of rows without a token.
// 3. join: the workgroup of the chunk in which a crossing run begins adds its
//    partial sums in order.

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortRows = 512;   // table rows of a workgroup at most (54 KB of LDS)
constexpr int kSortKept = 192;   // found ids that a wavefront keeps in LDS

struct GradParams {
  const void* ids;
  int ids_i64;
  int64_t N, V, H;
  int64_t padding;  // id whose gradient stays zero (-1: none)
  const uint8_t* g;
  int64_t ldg;  // bytes
  float scale;
  uint8_t* dw;
  int64_t lddw;  // bytes
  int add;       // dw holds a gradient to add to
  int rpw;       // sort: table rows per workgroup
  int chunk;     // sum: sorted entries per workgroup
  int64_t chunks;
  int32_t* pos;    // [N] token positions by (row, position)
  int32_t* row;    // [N] their rows
  int32_t* start;  // [V + 1] where each row's run starts
  float* part;     // [chunks][2][H]: the chunk's first and last, unfinished, runs
};

__global__ __launch_bounds__(kSortThreads) void vocab_sort_kernel(const GradParams p) {
  extern __shared__ int32_t lds[];
  int32_t* cnt = lds;                            // [kSortWaves][rpw]
  int32_t* scan = cnt + kSortWaves * p.rpw;      // [kSortThreads]
  int32_t* kept_pos = scan + kSortThreads;       // [kSortWaves][kSortKept]
  uint16_t* kept_row = reinterpret_cast<uint16_t*>(kept_pos + kSortWaves * kSortKept);
  __shared__ int32_t s_less[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t lo = (int64_t)blockIdx.x * p.rpw;
  const int nrows = (int)min((int64_t)p.rpw, p.V - lo);
  for (int i = tid; i < kSortWaves * p.rpw; i += kSortThreads) cnt[i] = 0;
  __syncthreads();

  const int64_t per = (cdiv(p.N, (int64_t)kSortWaves) + 63) / 64 * 64;
  const int64_t n0 = wave * per, n1 = min(p.N, n0 + per);
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  int less = 0, found = 0;
  // the ids of this wavefront's part, 64 at a time and four such reads ahead;
  // visit(row in the workgroup's range, position, taken)
  auto scan_ids = [&](auto visit) {
    for (int64_t n = n0; n < n1; n += 256) {
      int64_t id[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = n + j * 64 + lane;
        id[j] = at < n1 ? token_id(p.ids, p.ids_i64, at) : -1;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool valid = id[j] >= 0 && id[j] < p.V && id[j] != p.padding;
        visit(id[j] - lo, n + j * 64 + lane, valid);
      }
    }
  };
  scan_ids([&](int64_t r, int64_t at, bool valid) {
    const bool mine = valid && r >= 0 && r < nrows;
    less += valid && r < 0 ? 1 : 0;
    const uint64_t m = __ballot(mine);
    if (mine) {
      atomicAdd(&cnt[wave * p.rpw + (int)r], 1);
      const int k = found + __popcll(m & below);
      if (k < kSortKept) {
        kept_pos[wave * kSortKept + k] = (int32_t)at;
        kept_row[wave * kSortKept + k] = (uint16_t)r;
      }
    }
    found += __popcll(m);
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) less += __shfl_xor(less, o, 64);
  if (lane == 0) s_less[wave] = less;
  __syncthreads();

  // exclusive scan over the rows' totals (thread r owns row r)
  int total = 0;
  if (tid < nrows)
    for (int w = 0; w < kSortWaves; ++w) total += cnt[w * p.rpw + tid];
  scan[tid] = total;
  __syncthreads();
  for (int o = 1; o < kSortThreads; o <<= 1) {
    const int v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += s_less[w];
  if (tid < nrows) {
    int at = base + scan[tid] - total;
    p.start[lo + tid] = at;
    if (lo + tid == p.V - 1) p.start[p.V] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * p.rpw + tid];
      cnt[w * p.rpw + tid] = at;
      at += c;
    }
  }
  __syncthreads();

  // placement, 64 found ids at a time in order: the lanes of one row take
  // consecutive places
  int32_t* next = cnt + wave * p.rpw;
  auto place = [&](bool mine, int r, int32_t at) {
    uint64_t left = __ballot(mine);
    while (left) {
      const int rr = __builtin_amdgcn_readlane(r, __builtin_ctzll(left));
      const uint64_t same = __ballot(mine && r == rr);
      const int first = next[rr];  // (one address: a broadcast)
      if (mine && r == rr) {
        const int k = first + __popcll(same & below);
        p.pos[k] = at;
        p.row[k] = (int32_t)(lo + rr);
      }
      if (lane == 0) next[rr] = first + __popcll(same);
      // the write is read back by the whole wavefront at the row's next turn
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
      left &= ~same;
    }
  };
  if (found <= kSortKept) {
    for (int k = 0; k < found; k += 64) {
      const bool mine = k + lane < found;
      const int at = wave * kSortKept + min(k + lane, found - 1);
      place(mine, kept_row[at], kept_pos[at]);
    }
  } else {
    scan_ids([&](int64_t r, int64_t at, bool valid) {
      const bool mine = valid && r >= 0 && r < nrows;
      place(mine, mine ? (int)r : 0, (int32_t)at);
    });
  }
}

constexpr int kSumThreads = 256;
constexpr int kZeroRows = 16;  // rows that a zeroing workgroup looks at

template <int WT, int NV>
__device__ __forceinline__ void grad_finish(const GradParams& p, int64_t v, int64_t c, const float (&acc)[NV]) {
  uint8_t* dst = p.dw + v * p.lddw + c * vt_bytes<WT>();
  float o[NV];
  if (p.add) {
    vt_load<WT, NV>(dst, o);
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] += acc[i] * p.scale;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = acc[i] * p.scale;
  }
  vt_store<WT, NV>(dst, o);
}

// Workgroup (x, y): chunk x, or for x >= chunks kZeroRows table rows; columns
// from y * 256 * NV on.
template <int GT, int WT, int NV>
__global__ __launch_bounds__(kSumThreads) void vocab_grad_sum_kernel(const GradParams p) {
  const int64_t c = ((int64_t)blockIdx.y * kSumThreads + threadIdx.x) * NV;
  if (blockIdx.x >= p.chunks) {
    const int64_t v0 = ((int64_t)blockIdx.x - p.chunks) * kZeroRows;
    if (c >= p.H) return;
    const float zero[NV] = {};
    for (int64_t v = v0; v < min(p.V, v0 + kZeroRows); ++v)
      if (p.start[v] == p.start[v + 1]) vt_store<WT, NV>(p.dw + v * p.lddw + c * vt_bytes<WT>(), zero);
    return;
  }
  const int64_t M = p.start[p.V], e0 = (int64_t)blockIdx.x * p.chunk, e1 = min(M, e0 + p.chunk);
  if (e0 >= e1 || c >= p.H) return;
  const int before = e0 > 0 ? p.row[e0 - 1] : -1, after = e1 < M ? p.row[e1] : -1;
  float acc[NV] = {};
  bool crosses = p.row[e0] == before;  // the current run began before the chunk
  constexpr int kAhead = 4;
  for (int64_t e = e0; e < e1; e += kAhead) {
    float g[kAhead][NV];
    int row[kAhead + 1];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t k = min(e + j, e1 - 1);
      row[j] = p.row[k];
      vt_load<GT, NV>(p.g + (int64_t)p.pos[k] * p.ldg + c * vt_bytes<GT>(), g[j]);
    }
    row[kAhead] = e + kAhead < e1 ? p.row[e + kAhead] : after;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (e + j >= e1) break;
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] += g[j][i];
      const bool last = e + j + 1 >= e1;
      const int next = last ? after : row[j + 1];
      if (last ? true : next != row[j]) {  // the run ends here, or goes on behind the chunk
        if (crosses || next == row[j]) {
          // its first partial sums where it began before the chunk, else its last
          float* dst = p.part + ((int64_t)blockIdx.x * 2 + (crosses ? 0 : 1)) * p.H + c;
#pragma unroll
          for (int i = 0; i < NV; ++i) dst[i] = acc[i];
        } else {
          grad_finish<WT, NV>(p, row[j], c, acc);
        }
        crosses = false;
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
      }
    }
  }
}

// Workgroup (x, y): the run that begins in chunk x and goes on behind it
template <int WT, int NV>
__global__ __launch_bounds__(kSumThreads) void vocab_grad_join_kernel(const GradParams p) {
  const int64_t M = p.start[p.V], e1 = ((int64_t)blockIdx.x + 1) * p.chunk, e0 = e1 - p.chunk;
  if (e1 >= M) return;
  const int v = p.row[e1 - 1];
  const int64_t first = p.start[v], end = p.start[v + 1];  // the run's entries
  if (p.row[e1] != v || first < e0) return;
  const int64_t c = ((int64_t)blockIdx.y * kSumThreads + threadIdx.x) * NV;
  if (c >= p.H) return;
  float acc[NV];
  const float* src = p.part + ((int64_t)blockIdx.x * 2 + 1) * p.H + c;
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = src[i];
  const int64_t x1 = cdiv(end, (int64_t)p.chunk);  // chunks of the run: up to x1 - 1
  constexpr int kAhead = 8;
  for (int64_t x = (int64_t)blockIdx.x + 1; x < x1; x += kAhead) {
    float q[kAhead][NV];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float* s = p.part + min(x + j, x1 - 1) * 2 * p.H + c;
#pragma unroll
      for (int i = 0; i < NV; ++i) q[j][i] = s[i];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (x + j < x1)
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] += q[j][i];
  }
  grad_finish<WT, NV>(p, v, c, acc);
}

template <int GT, int WT, int NV>
void launch_grad(const GradParams& p, hipStream_t st) {
  const unsigned ny = (unsigned)cdiv(p.H, (int64_t)kSumThreads * NV);
  const int64_t zero = p.add ? 0 : cdiv(p.V, (int64_t)kZeroRows);
  if (p.chunks + zero > 0)
    hipLaunchKernelGGL((vocab_grad_sum_kernel<GT, WT, NV>), dim3((unsigned)(p.chunks + zero), ny), dim3(kSumThreads), 0, st, p);
  if (p.chunks > 1)
    hipLaunchKernelGGL((vocab_grad_join_kernel<WT, NV>), dim3((unsigned)(p.chunks - 1), ny), dim3(kSumThreads), 0, st, p);
}

// Sorted entries per workgroup: 16 while that gives the CUs work, 64 where the
// partial sums (two rows per chunk) outgrow it (4096 wide: 16384 tokens 209 us by
// 16, 235 by 64; 131072: 448 and 430)
int grad_chunk(int64_t N) { return N <= 65536 ? 16 : 64; }

int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }

// Workspace layout: pos, row, start, partial sums
int64_t grad_layout(int64_t N, int64_t V, int64_t H, int64_t (&off)[4]) {
  int64_t at = 0;
  off[0] = at;
  at += up16(4 * N);
  off[1] = at;
  at += up16(4 * N);
  off[2] = at;
  at += up16(4 * (V + 1));
  off[3] = at;
  at += up16(cdiv(N, (int64_t)grad_chunk(N)) * 2 * H * 4);
  return at;
}

bool vec_ok(const void* p, int64_t ld_bytes, int size) {
  return (reinterpret_cast<uintptr_t>(p) % std::min(16, 8 * size)) == 0 && ld_bytes % std::min(16, 8 * size) == 0;
}

// positions, rows and the grids' thread counts fit 32 bits
constexpr int64_t kMaxIds = ((int64_t)1 << 24) - 1, kMaxRows = (int64_t)1 << 27, kMaxWidth = (int64_t)1 << 20;

}  // namespace

// See include/qmoe.h for the contracts.
extern "C" int qmoe_vocab_lookup(const void* ids, int ids_i64, int64_t N, const void* w, int wtype, int64_t ldw,
                                 const float* row_scale, int64_t V, int64_t H, float scale, void* out, int otype,
                                 int64_t ldo, hipStream_t stream) {
  if (N < 0 || N > kMaxIds || V <= 0 || V > kMaxRows || H <= 0 || H > kMaxWidth || ldw < H || ldo < H) return QMOE_ERR_ARG;
  if (wtype < VT_BF16 || wtype > VT_E5M2 || wtype == VT_F16 || otype < VT_BF16 || otype > VT_F16) return QMOE_ERR_ARG;
  if (N == 0) return QMOE_OK;
  const bool coded = wtype >= VT_E4M3;
  if (!ids || !w || !out || (coded != (row_scale != nullptr))) return QMOE_ERR_ARG;
  LookupParams p{};
  p.ids = ids;
  p.ids_i64 = ids_i64;
  p.N = N, p.V = V, p.H = H;
  p.w = static_cast<const uint8_t*>(w);
  p.ldw = ldw * vt_size(wtype);
  p.row_scale = row_scale;
  p.scale = scale;
  p.out = static_cast<uint8_t*>(out);
  p.ldo = ldo * vt_size(otype);
  const bool vec = H % 8 == 0 && vec_ok(w, p.ldw, vt_size(wtype)) && vec_ok(out, p.ldo, vt_size(otype));
  switch (wtype) {
    case VT_BF16: launch_lookup_out<VT_BF16>(p, otype, vec, stream); break;
    case VT_F32: launch_lookup_out<VT_F32>(p, otype, vec, stream); break;
    case VT_E4M3: launch_lookup_out<VT_E4M3>(p, otype, vec, stream); break;
    case VT_INT8: launch_lookup_out<VT_INT8>(p, otype, vec, stream); break;
    default: launch_lookup_out<VT_E5M2>(p, otype, vec, stream); break;
  }
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_vocab_lookup_grad_workspace_size(int64_t N, int64_t V, int64_t H, int64_t* bytes) {
  if (N < 0 || N > kMaxIds || V <= 0 || V > kMaxRows || H <= 0 || H > kMaxWidth || !bytes) return QMOE_ERR_ARG;
  int64_t off[4];
  *bytes = grad_layout(N, V, H, off);
  return QMOE_OK;
}

extern "C" int qmoe_vocab_lookup_grad(const void* ids, int ids_i64, int64_t N, const void* grad, int gtype, int64_t ldg,
                                      int64_t V, int64_t H, float scale, int64_t padding_idx, void* dw, int wtype,
                                      int64_t lddw, int add, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  int64_t need = 0;
  if (qmoe_vocab_lookup_grad_workspace_size(N, V, H, &need) != QMOE_OK) return QMOE_ERR_ARG;
  if (ldg < H || lddw < H || !dw || (N > 0 && (!ids || !grad))) return QMOE_ERR_ARG;
  if ((gtype != VT_BF16 && gtype != VT_F32) || (wtype != VT_BF16 && wtype != VT_F32)) return QMOE_ERR_ARG;
  if (!workspace || ws_bytes < need) return QMOE_ERR_WORKSPACE;
  int64_t off[4];
  grad_layout(N, V, H, off);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  GradParams p{};
  p.ids = ids;
  p.ids_i64 = ids_i64;
  p.N = N, p.V = V, p.H = H;
  p.padding = padding_idx < 0 ? -1 : padding_idx;
  p.g = static_cast<const uint8_t*>(grad);
  p.ldg = ldg * vt_size(gtype);
  p.scale = scale;
  p.dw = static_cast<uint8_t*>(dw);
  p.lddw = lddw * vt_size(wtype);
  p.add = add;
  p.chunk = grad_chunk(N);
  p.chunks = cdiv(N, (int64_t)p.chunk);
  p.pos = reinterpret_cast<int32_t*>(ws + off[0]);
  p.row = reinterpret_cast<int32_t*>(ws + off[1]);
  p.start = reinterpret_cast<int32_t*>(ws + off[2]);
  p.part = reinterpret_cast<float*>(ws + off[3]);
  // one workgroup per CU, or as many as hold kSortRows rows each
  p.rpw = (int)std::min<int64_t>(std::max<int64_t>(cdiv(V, (int64_t)256), 1), kSortRows);
  const size_t lds = (size_t)(kSortWaves * p.rpw + kSortThreads + kSortWaves * kSortKept) * 4 + kSortWaves * kSortKept * 2;
  hipLaunchKernelGGL(vocab_sort_kernel, dim3((unsigned)cdiv(V, (int64_t)p.rpw)), dim3(kSortThreads), lds, stream, p);
  const bool vec = H % 8 == 0 && vec_ok(grad, p.ldg, vt_size(gtype)) && vec_ok(dw, p.lddw, vt_size(wtype));
#define QMOE_GRAD(G, W) (vec ? launch_grad<G, W, 8>(p, stream) : launch_grad<G, W, 1>(p, stream))
  if (gtype == VT_BF16) wtype == VT_BF16 ? QMOE_GRAD(VT_BF16, VT_BF16) : QMOE_GRAD(VT_BF16, VT_F32);
  else wtype == VT_BF16 ? QMOE_GRAD(VT_F32, VT_BF16) : QMOE_GRAD(VT_F32, VT_F32);
#undef QMOE_GRAD
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
