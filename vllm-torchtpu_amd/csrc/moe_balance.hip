// Routing with its balance loss, per-expert counts and the logits' gradient.
//
//   s[t]    = scores of token t, ids / w as qmoe_moe_route (float32 weights; 0 for a token outside the mask)
//   p[t, e] = s[t, e] / max(sum_e s[t, e], 1e-20)   (softmax: s itself)
//   c[e]    = counted tokens that chose e, N = counted tokens
//   loss    = E / (k N^2) sum_e c[e] sum_t p[t, e],  0 where N = 0
//
// and, with gw and gl the gradients of w and loss, A_j = s[t, ids_j], D = max(sum_j A_j, 1e-20),
//
//   g[t, e]  = gl E c[e] / (k N^2)  as the gradient of p, put through p's quotient to s (a floor is a constant), plus
//              rsf (gw_j - sum_i gw_i A_i / D) / D  at e = ids_j     (renormalized; else rsf gw_j)
//   dlogits  = s (g - sum_e g s)                  softmax
//              g s (1 - s)                        sigmoid
//              g sigmoid(x) / (2 s)               sqrtsoftplus
//
// What bounds it: T E logits read once (forward) and read and written once
// (backward); in fact the router's dependent chain of k row maxima per token
// hides the forward's traffic. So the statistics ride on the router: a wavefront
// keeps its tokens' sums of p in registers, one slot per expert, and counts go
// to integer atomics in LDS (any order, same result); one more launch adds the
// workgroups' parts in a fixed order, and none at all where one workgroup holds
// every token. The gradient reads logits again rather than keeping T E scores.
//
// 16384 tokens, 256 experts in f32, 8 from the best 4 of 8 groups by sigmoids: routes 34 us (84 % of
// the vector ALUs' cycles, four wavefronts a SIMD), sums 5.5, gradient 15 (34 MB, 2.3
// TB/s); 777 tokens, 128 experts, softmax 4.5, 6.5 and 4.5; 8 tokens 3.9 in one launch.

#include "../../include/qmoe.h"
#include "moe_route.h"

namespace {

using namespace qmoe_route;

constexpr int kOneGroup = 32;   // tokens that one workgroup routes alone, two per wavefront
constexpr int kMaxGroups = 256;
constexpr float kTiny = 1e-20f;

struct BalanceParams {
  const void* logits;
  int logits_f32;
  int64_t T;
  int E, topk;
  const float* bias;
  int renormalize;
  float rsf;
  int num_group, topk_group;
  const uint8_t* mask;
  float* weights;
  int32_t* ids;
  float* loss;
  int32_t* counts;
  float* part_p;    // [workgroups][E]
  int32_t* part_c;  // [workgroups][E]
  float* sum_p;     // [E]
  uint32_t* ticket;
};

// loss from sums of p and counts (in LDS or global memory), by one wavefront
__device__ __forceinline__ void balance_loss(const float* sum_p, const int32_t* counts, int E, int topk, float* loss) {
  const int lane = threadIdx.x & 63;
  double dot = 0.0, n = 0.0;
  for (int e = lane; e < E; e += 64) {
    dot += (double)counts[e] * (double)sum_p[e];
    n += (double)counts[e];
  }
  dot = wave_sum_du(dot);
  n = wave_sum_du(n) / topk;
  if (lane == 0) *loss = n > 0.0 ? (float)(dot * E / (topk * n * n)) : 0.0f;
}

template <int S, int SCORING, bool GROUPED>
__global__ __launch_bounds__(1024) void balance_route_kernel(const BalanceParams p) {
  __shared__ float scratch[16][kChoiceLds];  // grouped selection; then the wavefronts' sums of p
  __shared__ int32_t cnt[kMaxSlots * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6, E = p.E;
  for (int e = tid; e < E; e += blockDim.x) cnt[e] = 0;
  if (p.ticket && blockIdx.x == 0 && tid == 0) *p.ticket = 0;  // (for the launch behind this one)
  __syncthreads();
  float acc[S];
#pragma unroll
  for (int j = 0; j < S; ++j) acc[j] = 0.0f;
  float bv[kMaxSlots];
  load_bias<S>(p.bias, E, bv);
  for (int64_t t = (int64_t)blockIdx.x * waves + wave; t < p.T; t += (int64_t)gridDim.x * waves) {
    const bool live = p.mask ? p.mask[t] != 0 : true;
    float s[kMaxSlots];
    row_scores<S, SCORING>(p.logits, p.logits_f32, t, E, s);
    const int id = route_scored<S, GROUPED>(s, bv, t, E, p.topk, p.bias, p.renormalize, p.rsf, p.num_group,
                                            p.topk_group, p.weights, 1, p.ids, scratch[wave], nullptr, nullptr, live);
    if (GROUPED) wave_lds_sync();  // the scratch is read before the next token's scores come
    if (!live) continue;
    if (lane < p.topk) atomicAdd(&cnt[id], 1);
    float q = 1.0f;
    if constexpr (SCORING != 0) {
      float row = 0.0f;
#pragma unroll
      for (int j = 0; j < S; ++j) row += j * 64 + lane < E ? s[j] : 0.0f;
      row = wave_sum_u(row);
      q = 1.0f / (row != row ? row : fmaxf(row, kTiny));
    }
#pragma unroll
    for (int j = 0; j < S; ++j) acc[j] += j * 64 + lane < E ? s[j] * q : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < S; ++j) scratch[wave][j * 64 + lane] = acc[j];
  __syncthreads();
  const bool alone = gridDim.x == 1;
  for (int e = tid; e < E; e += blockDim.x) {
    float v = 0.0f;
    for (int w = 0; w < waves; ++w) v += scratch[w][e];
    if (alone) {
      scratch[0][e] = v;  // (only this thread reads column e)
      p.counts[e] = cnt[e];
    } else {
      p.part_p[(int64_t)blockIdx.x * E + e] = v;
      p.part_c[(int64_t)blockIdx.x * E + e] = cnt[e];
    }
  }
  if (!alone) return;
  __syncthreads();
  if (wave == 0) balance_loss(scratch[0], cnt, E, p.topk, p.loss);
}

// Workgroup x adds the parts of experts 8 x .. + 7 (32 workgroups' parts at a time,
// then across them), and the last to finish the loss.
__global__ __launch_bounds__(256) void balance_join_kernel(const BalanceParams p, int groups) {
  __shared__ float sp[32][9];
  __shared__ int32_t sc[32][9];
  __shared__ bool last;
  const int tid = threadIdx.x, c = tid & 7, r = tid >> 3, e = blockIdx.x * 8 + c;
  float v = 0.0f;
  int32_t n = 0;
  if (e < p.E) {
#pragma unroll 8
    for (int g = r; g < groups; g += 32) {
      v += p.part_p[(int64_t)g * p.E + e];
      n += p.part_c[(int64_t)g * p.E + e];
    }
  }
  sp[r][c] = v;
  sc[r][c] = n;
  __syncthreads();
  if (r == 0 && e < p.E) {
#pragma unroll
    for (int i = 1; i < 32; ++i) {
      v += sp[i][c];
      n += sc[i][c];
    }
    p.sum_p[e] = v;
    p.counts[e] = n;
    __threadfence();
  }
  __syncthreads();
  if (tid == 0) last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (tid < 64) balance_loss(p.sum_p, p.counts, p.E, p.topk, p.loss);
}

struct BalanceGradParams {
  const void* logits;
  int logits_f32;
  int64_t T;
  int E, topk;
  int renormalize;
  float rsf;
  const uint8_t* mask;
  const int32_t* ids;
  const int32_t* counts;
  const float* g_weights;  // [T][topk] or nullptr
  const float* g_loss;     // one value or nullptr
  void* d_logits;          // the logits' type
};

// 1 / x by one correction of the hardware's reciprocal: within 2^-23, in half the
// instructions of the division (an infinite or NaN x keeps the first)
__device__ __forceinline__ float recip(float x) {
  const float r = __builtin_amdgcn_rcpf(x), f = fmaf(fmaf(-x, r, 1.0f), r, r);
  return fabsf(x) < __builtin_inff() ? f : r;
}

// One wavefront per token (scores in float32, from an accurate exponential);
// expert e in lane e % 64, slot e / 64.
template <int S, int SCORING>
__global__ __launch_bounds__(256) void balance_grad_kernel(const BalanceGradParams p) {
  __shared__ float at_expert[4][S * 64];  // the weights' part of a token's scores
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = p.E, k = p.topk;
  // gradient of the loss by p[t, e] of a counted token
  float coef[S];
  {
    double n = 0.0;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int e = j * 64 + lane;
      const int32_t c = e < E ? p.counts[e] : 0;
      coef[j] = (float)c;
      n += (double)c;
    }
    n = wave_sum_du(n);  // k N
    const float unit = p.g_loss && n > 0.0 ? (float)((double)*p.g_loss * E * k / (n * n)) : 0.0f;
#pragma unroll
    for (int j = 0; j < S; ++j) coef[j] = p.g_loss ? coef[j] * unit : 0.0f;
  }
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < p.T; t += (int64_t)gridDim.x * 4) {
    const bool live = p.mask ? p.mask[t] != 0 : true;
    float x[S], d[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int e = j * 64 + lane < E ? j * 64 + lane : E - 1;
      x[j] = p.logits_f32 ? static_cast<const float*>(p.logits)[t * E + e]
                          : bf16_to_f32(static_cast<const uint16_t*>(p.logits)[t * E + e]);
      d[j] = 0.0f;
    }
    const int id = lane < k ? p.ids[t * k + lane] : 0;
    const float gw = lane < k && p.g_weights ? p.g_weights[t * k + lane] : 0.0f;
    if (live) {
      // scores and their derivatives
      float s[S], ds[S];
      if constexpr (SCORING == 0) {
        float mx = -__builtin_inff();
        bool nan = false;
#pragma unroll
        for (int j = 0; j < S; ++j)
          if (j * 64 + lane < E) {
            nan |= x[j] != x[j];
            mx = fmaxf(mx, x[j]);
          }
        mx = wave_max_u(mx);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
          s[j] = j * 64 + lane < E ? expf(x[j] - mx) : 0.0f;
          sum += s[j];
        }
        sum = wave_sum_u(sum);
        const float q = __any(nan) ? __builtin_nanf("") : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < S; ++j) {
          s[j] *= q;
          ds[j] = s[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < S; ++j) {
          const float e = expf(-fabsf(x[j])), r = recip(1.0f + e);
          const float sg = x[j] >= 0.0f ? r : e * r;  // (NaN stays one: e is)
          if constexpr (SCORING == 1) {
            s[j] = sg;
            ds[j] = e * r * r;
          } else {
            s[j] = sqrtf(fmaxf(x[j], 0.0f) + log1pf(e));
            if (x[j] != x[j]) s[j] = x[j];
            // below -16 both the score and its double derivative are e^(x / 2), to 2^-24
            if (x[j] < -16.0f) s[j] = expf(0.5f * x[j]);
            ds[j] = x[j] < -16.0f ? 0.5f * s[j] : sg / (2.0f * s[j]);
          }
          if (j * 64 + lane >= E) s[j] = ds[j] = 0.0f;
        }
      }
      // the gradient by the scores: of the loss through p ...
      float g[S];
      if constexpr (SCORING == 0) {
#pragma unroll
        for (int j = 0; j < S; ++j) g[j] = coef[j];
      } else {
        float row = 0.0f, gp = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
          row += s[j];
          gp += coef[j] * s[j];
        }
        row = wave_sum_u(row);
        gp = wave_sum_u(gp);
        const float q = 1.0f / (row != row ? row : fmaxf(row, kTiny));
        const float off = row < kTiny ? 0.0f : gp * q;
#pragma unroll
        for (int j = 0; j < S; ++j) g[j] = (coef[j] - off) * q;
      }
      // ... and of the weights, at the chosen experts
      float a = 0.0f;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const float v = __shfl(s[j], id & 63, 64);
        a = (id >> 6) == j ? v : a;
      }
      float v = gw * p.rsf;
      if (p.renormalize) {
        // gw counts only by its differences: taken from that of the choice with the largest
        // score (the first may have a small one: the correction bias is not in it), so that
        // one weight, or one that is nearly all, gives no rounding error of gw's own size
        const float top = wave_max_u(lane < k ? a : -__builtin_inff());
        const uint64_t at = __ballot(lane < k && a == top);  // (none: a NaN, as is the sum)
        const float u = gw - lane_f(gw, at ? (int)__builtin_ctzll(at) : 0);
        const float sum = wave_sum_u(lane < k ? a : 0.0f), dot = wave_sum_u(lane < k ? u * a : 0.0f);
        const float q = 1.0f / (sum != sum ? sum : fmaxf(sum, kTiny));
        v = p.rsf * (sum < kTiny ? gw : u - dot * q) * q;
      }
      if (p.g_weights) {
#pragma unroll
        for (int j = 0; j < S; ++j) at_expert[wave][j * 64 + lane] = 0.0f;
        wave_lds_sync();
        if (lane < k && (unsigned)id < (unsigned)E) atomicAdd(&at_expert[wave][id], v);  // (an expert is chosen once)
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < S; ++j) g[j] += at_expert[wave][j * 64 + lane];
        wave_lds_sync();  // read before the next token's zeros
      }
      if constexpr (SCORING == 0) {
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) dot += g[j] * s[j];
        dot = wave_sum_u(dot);
#pragma unroll
        for (int j = 0; j < S; ++j) d[j] = s[j] * (g[j] - dot);
      } else {
#pragma unroll
        for (int j = 0; j < S; ++j) d[j] = g[j] * ds[j];
      }
    }
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int e = j * 64 + lane;
      if (e >= E) continue;
      if (p.logits_f32) static_cast<float*>(p.d_logits)[t * E + e] = d[j];
      else static_cast<uint16_t*>(p.d_logits)[t * E + e] = f32_to_bf16(d[j]);
    }
  }
}

// workgroups and wavefronts of the forward launch. Up to 32 tokens one workgroup, two tokens
// per wavefront, and no second launch: 17 tokens x 128, softmax 5.5 us (two launches 7.8), 32
// tokens 7.5 (8.0), 48 tokens 10.1 (8.0); of 256 experts in groups, whose choice takes
// longer, 17 tokens 11.6 (11.7), but 24 tokens 12.7 (12.0) and 32 tokens 17.4 (11.7). Then one
// token per wavefront while there are fewer than four wavefronts per CU, in workgroups
// of four (of sixteen: 300 x 128 8.7 -> 9.6, 1024 x 256 in groups 12.7 -> 16.5), above that of
// sixteen, so that the parts stay few (of four: 1025 x 128 10.2 -> 9.4, 4096 x 128 10.5 -> 12.8, 16384
// x 256 36.8 -> 69.4). 256 workgroups at most: 16384 x 256 by 128 63.7, by 512 41.4.
int balance_groups(int64_t T, int* waves) {
  if (T <= kOneGroup) {
    *waves = (int)(T < 16 ? T : 16);
    return 1;
  }
  *waves = T <= 1024 ? 4 : 16;
  const int64_t g = cdiv<int64_t>(T, *waves);
  return (int)(g < kMaxGroups ? g : kMaxGroups);
}

template <int S>
void launch_balance(int scoring, bool grouped, int groups, int waves, const BalanceParams& p, hipStream_t st) {
  const dim3 grid(groups), block(64 * waves);
#define QMOE_BALANCE(SC, G) hipLaunchKernelGGL((balance_route_kernel<S, SC, G>), grid, block, 0, st, p)
  switch (scoring * 2 + (grouped ? 1 : 0)) {
    case 0: QMOE_BALANCE(0, false); break;
    case 1: QMOE_BALANCE(0, true); break;
    case 2: QMOE_BALANCE(1, false); break;
    case 3: QMOE_BALANCE(1, true); break;
    case 4: QMOE_BALANCE(2, false); break;
    default: QMOE_BALANCE(2, true); break;
  }
#undef QMOE_BALANCE
}

template <int S>
void launch_balance_grad(int scoring, const BalanceGradParams& p, hipStream_t st) {
  // (65536 tokens x 128 / x 256: 28.7 / 37.7 us, by 1024 workgroups 33.4 / 43.7, by 16384 32.5 / 40.3;
  // no difference up to 16384 tokens)
  const int64_t g = cdiv<int64_t>(p.T, 4);
  const dim3 grid((unsigned)(g < 4096 ? g : 4096)), block(256);
  if (scoring == 0) hipLaunchKernelGGL((balance_grad_kernel<S, 0>), grid, block, 0, st, p);
  else if (scoring == 1) hipLaunchKernelGGL((balance_grad_kernel<S, 1>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((balance_grad_kernel<S, 2>), grid, block, 0, st, p);
}

constexpr int64_t kMaxTokens = 1 << 24;

int64_t balance_bytes(int64_t T, int E) {
  int waves;
  const int g = balance_groups(T, &waves);
  return g == 1 ? 0 : 256 + 4 * (int64_t)E * (2 * g + 1);
}

}  // namespace

// See include/qmoe.h for the contract.
extern "C" int qmoe_moe_balance_workspace_size(int64_t T, int E, int64_t* bytes) {
  if (T < 0 || T > kMaxTokens || E <= 0 || E > kMaxSlots * 64 || !bytes) return QMOE_ERR_ARG;
  *bytes = T == 0 ? 0 : balance_bytes(T, E);
  return QMOE_OK;
}

extern "C" int qmoe_moe_balance(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring,
                                const float* bias, int renormalize, float routed_scaling_factor, int num_group,
                                int topk_group, const uint8_t* token_mask, float* topk_weights, int32_t* topk_ids,
                                float* loss, int32_t* counts, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  if (!route_args_ok(T, E, topk, scoring, num_group, topk_group) || scoring > 2 || T < 1 || T > kMaxTokens)
    return QMOE_ERR_ARG;
  if (!logits || !topk_weights || !topk_ids || !loss || !counts) return QMOE_ERR_ARG;
  int waves;
  const int groups = balance_groups(T, &waves);
  BalanceParams p{logits, logits_f32, T, E, topk, bias, renormalize, routed_scaling_factor, num_group, topk_group,
                  token_mask, topk_weights, topk_ids, loss, counts, nullptr, nullptr, nullptr, nullptr};
  if (groups > 1) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || ws_bytes < balance_bytes(T, E)) return QMOE_ERR_WORKSPACE;
    p.ticket = static_cast<uint32_t*>(workspace);
    p.sum_p = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
    p.part_p = p.sum_p + E;
    p.part_c = reinterpret_cast<int32_t*>(p.part_p + (int64_t)groups * E);
  }
  const bool grouped = num_group > 1 && topk_group < num_group;
  switch (route_slots(E)) {
    case 1: launch_balance<1>(scoring, grouped, groups, waves, p, stream); break;
    case 2: launch_balance<2>(scoring, grouped, groups, waves, p, stream); break;
    case 4: launch_balance<4>(scoring, grouped, groups, waves, p, stream); break;
    default: launch_balance<8>(scoring, grouped, groups, waves, p, stream); break;
  }
  if (groups > 1) hipLaunchKernelGGL(balance_join_kernel, dim3(cdiv(E, 8)), dim3(256), 0, stream, p, groups);
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}

extern "C" int qmoe_moe_balance_grad(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring,
                                     int renormalize, float routed_scaling_factor, const uint8_t* token_mask,
                                     const int32_t* topk_ids, const int32_t* counts, const float* g_weights,
                                     const float* g_loss, void* d_logits, hipStream_t stream) {
  if (!route_args_ok(T, E, topk, scoring, 1, 1) || scoring > 2 || T < 1 || T > kMaxTokens) return QMOE_ERR_ARG;
  if (!logits || !topk_ids || !counts || !d_logits) return QMOE_ERR_ARG;
  const BalanceGradParams p{logits, logits_f32, T, E, topk, renormalize, routed_scaling_factor, token_mask, topk_ids,
                            counts, g_weights, g_loss, d_logits};
  switch (route_slots(E)) {
    case 1: launch_balance_grad<1>(scoring, p, stream); break;
    case 2: launch_balance_grad<2>(scoring, p, stream); break;
    case 4: launch_balance_grad<4>(scoring, p, stream); break;
    default: launch_balance_grad<8>(scoring, p, stream); break;
  }
  return hipGetLastError() == hipSuccess ? QMOE_OK : QMOE_ERR_LAUNCH;
}
