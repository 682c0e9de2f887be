/*
 * qmoe — C ABI of the MI355X (gfx950) quantized-GEMM / fused-MoE library.
 *
 * Every entry point takes raw device pointers, sizes and a hipStream_t, is
 * asynchronous on that stream, allocates nothing, and returns a status:
 *   0 QMOE_OK, 1 QMOE_ERR_ARG (bad shape / unsupported combination),
 *   2 QMOE_ERR_WORKSPACE (workspace too small), 3 QMOE_ERR_LAUNCH,
 *   4 QMOE_ERR_SCRATCH (qmoe_gemm_static: partial sums exceed its scratch).
 * Layouts (all row-major):
 *   activations  [rows, K]            bf16 (uint16 bit patterns) or 1-byte codes
 *   weights      [G][N][K]            N-major: each output channel's K contiguous
 *                                     (e2m1: [G][N][K/2], low nibble = even k)
 *   scales       per-channel f32 [G][N]; block f32 [G][N/bn][K/128];
 *                MX e8m0 bytes [G][N][K/32]; NVFP4 bf16 [G][N][K/16];
 *                INT4 bf16 [G][N][K/wq_group]
 * Reference paths below are relative to the reference plugin's
 * src/vllm_torchtpu/.
 */
#ifndef QMOE_H_
#define QMOE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* qmoe_stream_t; /* == hipStream_t */

/* GEMM kinds (qmoe_gemm_desc.kind) */
enum {
  QMOE_W8A8_PC = 0,  /* A e4m3|int8|e5m2 (wfmt) + per-row f32 scale; W same dtype + per-channel
                        f32 scale */
  QMOE_W8A8_BLK = 1, /* A e4m3 + per-(row,128) scale; W e4m3 + per-(n/bn, 128) scale */
  QMOE_W8A16_PC = 2, /* A bf16; W e4m3 + per-channel scale */
  QMOE_W4A16_MX = 3, /* A bf16; W e2m1 + e8m0 scale per 32 k */
  QMOE_W16A16 = 4,   /* A bf16; W bf16 */
  QMOE_W4A16_NV = 5, /* A bf16; W e2m1 + bf16 scale per 16 k (NVFP4: the checkpoint's e4m3
                        block scale times its f32 global scale, rounded to bf16 as the
                        reference's `kernels/megablox/gmm_v2.py:452-462` dequantization
                        does; each weight is bf16(code * scale)) */
  QMOE_W8A8_GMM = 7, /* A e4m3|int8 codes + f32 scale per (row, 512 columns, the last
                        block partial) from qmoe_row_quant mode 2; W e4m3|int8|e5m2 (wfmt; A is
                        int8 for int8 W, e4m3 for float W) + per-channel f32
                        scale [G][N] (ldws <= 1) or one per (row, B columns) [G][N][K/B] with
                        ldws = K/B, B a power-of-two multiple of 512. The quantized-lhs regime
                        of the reference's grouped
                        matmul, `kernels/megablox/gmm_v2.py:500-548, 1198-1237` (weights with
                        quant blocks of 256 or more columns: per-channel experts) */
  QMOE_W8A16_BLK = 8, /* A bf16; W e4m3 + f32 scale per (n / ws_bn, 128 k) [G][N/bn][K/128];
                        each weight is bf16(code * bf16(scale)) before the product: the
                        dequantize-before-matmul regime of `kernels/megablox/gmm_v2.py:452-462`
                        (quant blocks below 256 columns) */
  QMOE_W4A16_I4 = 6, /* A bf16; W symmetric 4-bit integers in the compressed-tensors
                        encoding (nibble = value + 8, two per byte, even k in the low
                        nibble: the int32 carriers of `compressed_tensors_moe_w4a16.py`
                        read as bytes) + bf16 scale per wq_group k; each weight is
                        bf16(value * scale), `kernels/megablox/gmm_v2.py:452-462` */
  QMOE_W4A4_MX = 9,  /* A e2m1 codes packed as W (lda in bytes >= K/2) + e8m0 bytes per
                        (row, 32 k) in a_scale [M, lds_a >= K/32] (qmoe_mx_quant); W as
                        QMOE_W4A16_MX. Both scales go to the MFMA. Opt-in MX activations
                        (no counterpart in the reference, whose W4A4 method runs W4A16,
                        `compressed_tensors_moe_w4an_mxfp4.py:49-55`). Dense: bias only;
                        grouped: fused activation, bias, row maps and routing weight as
                        the other kinds (a_rows also gathers the scale rows); no K split;
                        K % 512 == 0 and K >= 1024 (pad with zero codes) */
  QMOE_W8A8_PC_DYN = 10 /* A bf16 rows (lda in elements, a multiple of 8), quantized per row
                        inside the call with the runtime recipe of
                        `kernels/quantized_matmul/util.py:294-318` (quantize_block: scale =
                        absmax / qmax, e4m3 / e5m2 in f32 or int8 in bf16 arithmetic per wfmt;
                        qmoe_row_quant mode 0 computes the same codes); W and w_scale as
                        QMOE_W8A8_PC; a_scale unused. The whole xla_quantized_matmul of
                        `:80-124` in one call. Dense only (no group_offs). Decode-size
                        problems quantize inside the weight-streaming kernel (one launch: each
                        workgroup reads its rows' absmax from L2 while its first weight loads
                        are in flight); the rest quantize into the workspace first. The
                        workspace also holds the row scales, so it is needed whatever the
                        plan (qmoe_gemm_workspace_size) */
};

/* Fused gate/up activations (qmoe_gemm_desc.act) */
enum {
  QMOE_ACT_NONE = 0,
  QMOE_ACT_SILU = 1,
  QMOE_ACT_SWIGLUOAI = 2, /* p0 = alpha (1.702), p1 = limit (7.0) */
  QMOE_ACT_GELU_TANH = 3,
  QMOE_ACT_SILU_CLAMP = 4, /* p0 = limit (10.0) */
  QMOE_ACT_SITU = 5        /* p0 = beta, p1 = linear_beta (<= 0: none) */
};

/*
 * Grouped GEMM problem. For each group g (one group when group_offs is NULL)
 * and compact row R in [group_offs[g], group_offs[g+1]):
 *   acc[R, n] = sum_k A[a_rows ? a_rows[R] : R, k] * W[g, n, k]
 *   v = scales(acc) (+ bias[g, n]); with act: out[n] = act(v[n], v[n + N/2])
 *   out *= row_weight[R] (bf16, optional)
 *   Y[y_rows ? y_rows[R] : R, n] = bf16(out)
 */
typedef struct qmoe_gemm_desc {
  int32_t kind;           /* QMOE_W8A8_PC ... */
  int32_t wfmt;           /* QMOE_W8A8_PC, _GMM, _PC_DYN: 0 e4m3, 1 int8, 2 e5m2; other kinds 0 */
  const void* a;          /* activation codes or bf16 */
  int64_t lda;            /* elements (W4A4_MX: bytes of packed codes) */
  const float* a_scale;   /* W8A8: [rows] or [rows, lds_a]; W4A4_MX: e8m0 bytes [rows, lds_a] */
  int64_t lds_a;
  const int32_t* a_rows;  /* optional gather map [M] */
  const void* w;
  int64_t ldw;            /* bytes per weight row */
  int64_t w_gstride;      /* bytes per group */
  const void* w_scale;
  int64_t ldws;           /* elements per scale row */
  int64_t ws_gstride;     /* elements per group */
  int32_t ws_bn;          /* W8A8_BLK: weight rows per scale row (1 or 128) */
  const float* bias;      /* optional [G, N] */
  int64_t bias_gstride;
  const int32_t* group_offs; /* optional [G+1] */
  const int32_t* active;     /* optional slot -> group list (non-empty groups) */
  const int32_t* num_active; /* device scalar, valid slots in `active` */
  int32_t slots;          /* number of groups (or capacity of `active`) */
  int32_t max_rows;       /* host bound on rows of any one group */
  int32_t M;              /* total compact rows */
  int32_t N;              /* weight rows (2*I with a fused activation) */
  int32_t K;
  int32_t act;
  float act_p0, act_p1;
  const uint16_t* row_weight; /* optional bf16 [M] */
  void* y;                /* bf16 output */
  int64_t ldy;
  const int32_t* y_rows;  /* optional scatter map [M] */
  int32_t wq_group;       /* QMOE_W4A16_I4: k values per scale (32, 64 or 128) */
} qmoe_gemm_desc;

/* ABI revision of this header (bumped on any layout change). */
int qmoe_abi_version(void);

/*
 * Row quantizer: rows of x (bf16, or f32 when in_f32) -> 1-byte codes q and
 * f32 scales (one per row, or per (row, 128 columns) when block == 128).
 *   qdtype 0 e4m3fn, 1 int8, 2 e5m2 (per-row scales only; not mode 2, whose codes are
 *   e4m3 for any float weight: `kernels/megablox/gmm_v2.py:1198-1218`).
 *   mode 0: runtime activation quant, replaces the reference's
 *           `kernels/quantized_matmul/util.py:47-64` quantize_tensor /
 *           `:294-318` quantize_block (fp8 in f32, int8 in bf16 arithmetic);
 *   mode 1: load-time weight quant, replaces
 *           `layers/core/quantization.py:232-318` quantize_tensor
 *           (reciprocal-multiply scale, zero rows keep scale 0).
 */
int qmoe_row_quant(const void* x, int64_t ldx, int in_f32, int64_t M, int64_t K, int qdtype,
                   int mode, int block, void* q, int64_t ldq, float* scales, int64_t lds,
                   qmoe_stream_t stream);

/*
 * MX activation quantizer: bf16 rows x [M, K] (K % 32 == 0) -> e2m1 codes
 * packed two per byte (low nibble = even column) q [M, ldq >= Kp/2] and e8m0
 * bytes scales [M, lds >= Kp/32], columns K..Kp-1 (Kp % 32 == 0) as zero
 * blocks (codes 0, byte 0); and/or (xq != NULL) the dequantized values as
 * bf16 [M, ldxq >= K], exact. Per 32-column block: the reference's ue8m0
 * block rule, `layers/core/quantization.py:232-318` (`quantize_tensor` with
 * use_ue8m0, scale = amax * f32(1/6) snapped up to a power of two) and its
 * e2m1 encoder `compressed_tensors_moe/utils.py:167-183`
 * (`quantize_to_fp4_e2m1_nibbles`). The reference's W4A4 MXFP4 method runs
 * its activations unquantized; this is the activation side of the opt-in
 * QMOE_W4A4_MX GEMM. At least one of q, xq. A block holding an inf or NaN
 * (the reference's rule has no answer for it) gets codes 0 and byte 255,
 * the e8m0 NaN encoding: it reads back as NaN (xq: bf16 NaN) and the row's
 * other blocks keep their own codes.
 */
int qmoe_mx_quant(const void* x, int64_t ldx, int64_t M, int64_t K, int64_t Kp, void* q, int64_t ldq,
                  void* scales, int64_t lds, void* xq, int64_t ldxq, qmoe_stream_t stream);

/* Workspace bytes qmoe_gemm needs for this problem (split-K partials). */
int qmoe_gemm_workspace_size(const qmoe_gemm_desc* d, int64_t* bytes);

/*
 * The kernel choice qmoe_gemm makes for this problem, computed on the host
 * from the descriptor alone (no device memory is read): path 0 weight
 * streaming, 1 1-byte x 1-byte tiles, 2 bf16 x 4-bit tiles, 3 generic
 * tiles, 4 weight streaming in 64-row passes, 5 1-byte x 1-byte tiles of
 * 256 tokens x 256 or 224 weight rows, or 128 tokens x 224 rows, on
 * persistent workgroups (at most one per CU of the current device), 6 MX
 * 256 x 256 persistent tiles, 7 MX grouped tiles, 8 weight streaming with
 * the per-row activation quantization inside (QMOE_W8A8_PC_DYN; for the
 * kind's other problems the path of the GEMM after its separate
 * quantization), 9 1-byte x 1-byte tiles of 128 weight rows, 10 weight
 * streaming in slices of tile_m rows of a dense problem (one slice per
 * grid.z index, each streaming the whole weight matrix), 11 eight-wavefront
 * tiles (block-scaled e4m3, dense bf16 x bf16); tile_m = token rows per tile
 * (or per streaming pass or slice); ksplit = K slices. No counterpart in the
 * reference (its tiling is chosen inside the Pallas call,
 * `kernels/megablox/gmm_v2.py:922-1055`); it lets tests assert which kernel
 * instances they exercise. Any output pointer may be NULL.
 */
int qmoe_gemm_plan(const qmoe_gemm_desc* d, int32_t* path, int32_t* tile_m, int32_t* ksplit);

/*
 * Quantized (grouped) GEMM. One group replaces the dense runtime matmul of
 * `layers/adapter/linear_common.py:69-128` (_quantized_matmul_jax ->
 * `kernels/quantized_matmul/util.py:80-124` xla_quantized_matmul, and the
 * single-group gmm_v2 call for rank-4 scales) and `:188-209`
 * (_quantized_matmul_fp4_jax). Several groups replace the grouped matmul
 * `kernels/megablox/gmm_v2.py:1280-1443` (gmm_v2, incl. its fused
 * activation epilogue `:84-122`). The workspace holds split-K partial sums
 * of the small-M path; every call writes before it reads, so it needs no
 * initialisation, and calls that share one workspace must be ordered on one
 * stream.
 */
int qmoe_gemm(const qmoe_gemm_desc* d, void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * qmoe_gemm for callers that cannot allocate device memory (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc). No
 * counterpart in the reference. Same kernels and results as qmoe_gemm; the
 * split-K partial sums go to a static device array of the library
 * (qmoe_gemm_static_scratch_bytes(), 64 MiB, held per GPU until the process
 * ends) instead of a caller workspace, and no call allocates or frees
 * anything. A problem whose partials exceed it returns QMOE_ERR_SCRATCH
 * before any launch. Every call on one GPU shares that GPU's array: calls
 * that overlap on one GPU (other streams, other threads) race.
 */
int qmoe_gemm_static(const qmoe_gemm_desc* d, qmoe_stream_t stream);
int64_t qmoe_gemm_static_scratch_bytes(void);

/*
 * MoE routing for T tokens over E experts: scores, top-k, renormalize and
 * scale; weights written as bf16 (or f32 with weights_f32), ids int32 [T, k].
 * Replaces `layers/adapter/moe_routing.py:232-323` (select_experts) with the
 * sort-free top-k of `layers/core/rowmax_topk.py:28-61` (ties -> lowest id;
 * a row with no score above -3e38 gets NaN weights and ids 0..k-1).
 *   logits   : bf16 [T, E] (logits_f32 = 0) or f32 [T, E] (logits_f32 = 1)
 *   scoring  : 0 softmax, 1 sigmoid, 2 sqrtsoftplus, 3 none (logits are the
 *              scores: the reference's `layers/adapter/router_topk.py:42-50`
 *              rowmax_select)
 *   bias     : optional f32 [E] (choice = score + bias, weight = score)
 *   num_group/topk_group > 1: grouped selection (sum of top-2 per group with
 *   a bias, max without), the DeepSeek-V3 rule; upstream vLLM grouped_topk,
 *   called at `moe_routing.py:276-299`.
 */
int qmoe_moe_route(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring,
                   const float* bias, int renormalize, float routed_scaling_factor, int num_group,
                   int topk_group, void* topk_weights, int weights_f32, int32_t* topk_ids,
                   qmoe_stream_t stream);

/*
 * DeepSeek-V4 hash routing, replaces `layers/adapter/moe_routing.py:204-229`
 * (_hash_moe_select, taken by select_experts when the layer has a
 * hash_indices_table and input ids are given, `:259-274`): ids =
 * hash_table[input_ids[t]] (int32 [table_rows, topk]; input ids int32, or
 * int64 with ids_i64), weights = the row's scores (scoring as in
 * qmoe_moe_route, no bias) at those ids, renormalized, scaled, as bf16. An
 * input id outside the table or a table entry outside [0, E) gives id -1
 * and a NaN weight.
 */
int qmoe_moe_route_hash(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring,
                        const int32_t* hash_table, int64_t table_rows, const void* input_ids, int ids_i64,
                        int renormalize, float routed_scaling_factor, uint16_t* topk_weights, int32_t* topk_ids,
                        qmoe_stream_t stream);

/*
 * Token permutation by expert, replaces `layers/core/fused_moe_gmm.py:288-408`
 * (prepare_routed_gmm_inputs, non-EP): stable order by (expert, flat route
 * index t*k + slot); invalid routes (id < 0, or weight == 0 with
 * skip_padded) sort last. Outputs (int32):
 *   sorted_idx [T*k]  flat route index of each sorted row
 *   revert     [T*k]  sorted position of each flat route (inverse permutation)
 *   token_sorted [T*k] token of each sorted row (sorted_idx / k)
 *   group_offs [E+1]  row offsets per expert (group_sizes = diff)
 *   active     [min(E, T*k)] ids of experts with rows, ascending; num_active [1]
 *   sorted_weight [T*k] bf16 routing weight of each sorted row
 * One workgroup; histogram + exclusive scan + stable scatter in LDS.
 */
int qmoe_moe_dispatch(const int32_t* topk_ids, const uint16_t* topk_weights, int64_t T, int topk,
                      int E, int skip_padded, int32_t* sorted_idx, int32_t* revert,
                      int32_t* token_sorted, int32_t* group_offs, int32_t* active,
                      int32_t* num_active, uint16_t* sorted_weight, qmoe_stream_t stream);

/*
 * Routing and dispatch of a decode step in one launch (1 <= T <= 16 tokens,
 * T * topk <= 64 routes, E <= 512): the outputs of qmoe_moe_route (bf16
 * weights) followed by those of qmoe_moe_dispatch on its routes, written by
 * one workgroup. Replaces `layers/adapter/moe_routing.py:232-323`
 * (select_experts) followed by `layers/core/fused_moe_gmm.py:288-408`
 * (prepare_routed_gmm_inputs), which the reference runs back to back in
 * its MoE entry (`layers/adapter/quantization/fp8.py:1108-1222`). Returns
 * QMOE_ERR_ARG outside those bounds (the caller then makes the two calls).
 */
int qmoe_moe_route_dispatch(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring,
                            const float* bias, int renormalize, float routed_scaling_factor, int num_group,
                            int topk_group, uint16_t* topk_weights, int32_t* topk_ids, int skip_padded,
                            int32_t* sorted_idx, int32_t* revert, int32_t* token_sorted,
                            int32_t* group_offs, int32_t* active, int32_t* num_active,
                            uint16_t* sorted_weight, qmoe_stream_t stream);

/*
 * Weighted unpermute, replaces `layers/core/fused_moe_gmm.py:572-577`:
 * out[t] = bf16( sum over valid slots j of rows[t*k + j] ), where `rows`
 * holds the already weighted down-projection rows in flat route order
 * (written by qmoe_gemm with row_weight and y_rows = sorted_idx). A slot is
 * valid under the dispatch rule: 0 <= id < E (and weight != 0 with
 * skip_padded); the rows of other slots were never written and are skipped.
 */
int qmoe_moe_combine(const uint16_t* rows, const int32_t* topk_ids, const uint16_t* topk_weights,
                     int64_t T, int topk, int E, int64_t H, int skip_padded, uint16_t* out, int64_t ldo,
                     qmoe_stream_t stream);

/*
 * Fused decode MoE layer: the shared expert plus the routed experts of a
 * decode step, one call. Replaces the kernel call of
 * `layers/adapter/fused_moe_decode.py:249-339` (`_build_op` -> `_layer`),
 * i.e. `kernels/experimental/fused_moe_decode/fused_moe_decode_kernel.py:
 * 552-740` (`fused_moe_decode`) on one rank: n_ranks = 1 (the all-reduce is
 * the identity), expert_start = None, scatter_rows = False; the caller's
 * router supplies topk_ids / topk_weights.
 *
 * Numerics (all float32, output bf16): hidden states quantized to e4m3 per
 * (row, 512 columns) as scale = max|x| / 448, codes e4m3(x * (1 / scale));
 * each block's code dot times its row scale, summed, times the per-channel
 * w1 scale; mid = silu(gate) * up * coeff, coeff = bf16(route weight) *
 * routed_scale summed over the token's routes to that expert, or for the
 * shared expert sigmoid(x . shared_gate) (1 when shared_gate is NULL);
 * mid quantized per (row, 512 columns) the same way; second dot per block
 * times its row scale, summed, times the per-channel w2 scale; the shared
 * expert and the active routed experts added into one float32 sum per
 * token.
 *
 * weight_blocks = 128 (this build's variant, no reference counterpart):
 * 128x128 weight tiles kept as checkpointed, activations quantized per
 * (row, 128 columns), each block's dot times the activation block scale
 * times the tile scale.
 */
typedef struct qmoe_moe_decode_desc {
  const void* x;           /* bf16 [T][H] hidden states */
  int64_t T;               /* tokens, 1..64 */
  int64_t H;               /* hidden size, a multiple of 512 */
  int64_t I;               /* routed intermediate size, a multiple of 128 */
  int64_t I_shared;        /* shared intermediate size, a multiple of 128, <= I */
  int E;                   /* routed experts, 1..512 */
  int topk;                /* routes per token, 1..64 */
  const int32_t* topk_ids; /* [T][topk]; ids outside [0, E) select nothing */
  const void* topk_weights;/* [T][topk] bf16 (weights_f32 = 0) or f32 */
  int weights_f32;
  float routed_scale;      /* multiplies the routed experts only */
  int weight_blocks;       /* 0: per-channel scales; 128: 128x128 tile scales */
  const void* w1;          /* e4m3 [E][2I][H]: gate rows then up rows */
  const void* w2;          /* e4m3 [E][H][I] */
  const float* w1_scale;   /* [E][2I] | [E][2I/128][H/128] */
  const float* w2_scale;   /* [E][H]  | [E][H/128][I/128] */
  const void* shared_w1;   /* e4m3 [2 I_shared][H] */
  const void* shared_w2;   /* e4m3 [H][I_shared] */
  const float* shared_w1_scale; /* [2 I_shared] | [2 I_shared/128][H/128] */
  const float* shared_w2_scale; /* [H] | [H/128][I_shared/128] */
  const uint16_t* shared_gate;  /* bf16 [H], or NULL for an ungated shared expert */
  uint16_t* out;           /* bf16 [T][ldo] */
  int64_t ldo;
  /* Routing by the call (optional; no counterpart in the reference, whose
   * router runs before the decode kernel). With router_logits not NULL the
   * call first routes the tokens -- qmoe_moe_route's rule and results for
   * these arguments, bf16 weights -- and writes topk_ids / topk_weights,
   * which are then outputs (weights_f32 must be 0). Up to 8 tokens are
   * routed inside the first launch, more by a routing launch before it. */
  const void* router_logits;     /* [T][E] bf16 (logits_f32 = 0) or f32 */
  int logits_f32;
  int scoring;                   /* as qmoe_moe_route */
  const float* correction_bias;  /* [E] or NULL */
  int renormalize;
  float routed_scaling_factor;
  int num_group;
  int topk_group;
} qmoe_moe_decode_desc;

/* Workspace bytes of qmoe_moe_decode for this descriptor. */
int qmoe_moe_decode_workspace_size(const qmoe_moe_decode_desc* d, int64_t* bytes);

/* Four launches on `stream` (five when more than 8 tokens are routed by the
 * call); QMOE_ERR_ARG outside the envelope above, QMOE_ERR_WORKSPACE when
 * ws_bytes is below qmoe_moe_decode_workspace_size. */
int qmoe_moe_decode(const qmoe_moe_decode_desc* d, void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * A whole MoE layer for a few tokens (a decode step) in two launches: routing
 * (qmoe_moe_route's rule, float32 weights), then for every route j of token t
 *   h[t, j] = bf16(act(W13[e] x[t] + b13[e])),
 *   out[t] = bf16(sum over j of w[t, j] (W2[e] h[t, j] + b2[e])),
 * float32 sums in a fixed order, each weight bf16(code * scale) (FP8:
 * bf16(code * bf16(scale)), as QMOE_W8A16_BLK) and bf16 activations (the
 * dequantize-before-matmul regime of
 * `kernels/megablox/gmm_v2.py:452-462`). Replaces `layers/adapter/
 * moe_routing.py:232-323` followed by `layers/core/fused_moe_gmm.py:592-728`
 * for 1..16 tokens; against qmoe_moe_route_dispatch + qmoe_gemm (twice) +
 * qmoe_moe_combine neither the routing weights nor the route outputs are
 * rounded to bf16 before their sum.
 */
enum {
  QMOE_FEW_MXFP4 = 0, /* e2m1 + e8m0 per 32 k */
  QMOE_FEW_NVFP4 = 1, /* e2m1 + bf16 per 16 k */
  QMOE_FEW_INT4 = 2,  /* offset-binary nibbles + bf16 per `group` k */
  QMOE_FEW_FP8 = 3,   /* e4m3 + f32 per (row, 128 k), rounded to bf16 */
  QMOE_FEW_BF16 = 4
};
typedef struct qmoe_moe_few_desc {
  int32_t format;          /* QMOE_FEW_... */
  int32_t group;           /* QMOE_FEW_INT4: k per scale (32, 64 or 128) */
  const void* x;           /* bf16 [T][ldx] */
  int64_t ldx;             /* a multiple of 8 */
  int32_t T;               /* tokens, 1..16 */
  int32_t H;               /* hidden size, a multiple of 32 (FP8: 128; INT4: group) */
  int32_t I;               /* intermediate size, likewise */
  int32_t E;               /* experts, 1..512 */
  int32_t topk;            /* routes per token, T * topk <= 128 */
  const void* router_logits; /* [T][E] bf16, or f32 with logits_f32 */
  int32_t logits_f32;
  int32_t scoring;         /* as qmoe_moe_route */
  const float* correction_bias; /* [E] or NULL */
  int32_t renormalize;
  float routed_scaling_factor;
  int32_t num_group;
  int32_t topk_group;
  int32_t skip_padded;     /* routes whose weight is 0 in bf16 are padding */
  const void* w1;          /* [E][2I][H]: gate rows then up rows */
  const void* w2;          /* [E][H][I] */
  const void* w1_scale;    /* [E][2I][..]; NULL for QMOE_FEW_BF16 */
  const void* w2_scale;    /* [E][H][..] */
  const float* w1_bias;    /* [E][2I] or NULL */
  const float* w2_bias;    /* [E][H] or NULL */
  int32_t act;             /* QMOE_ACT_SILU ... */
  float act_p0, act_p1;
  void* out;               /* bf16 [T][ldo] */
  int64_t ldo;             /* a multiple of 4 */
} qmoe_moe_few_desc;
int qmoe_moe_few_workspace_size(const qmoe_moe_few_desc* d, int64_t* bytes);
int qmoe_moe_few(const qmoe_moe_few_desc* d, void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * Rows of the vocabulary table: out[n] = round(scale * s[id] * w[id]), id =
 * ids[n]. Replaces the gather + dequantize of `layers/adapter/quantization/
 * fp8.py:1692-1698` (VllmFp8LinearMethodTPU.embedding) with one launch, and the
 * plain gather of an unquantized table.
 *   ids     : int32, or int64 with ids_i64 [N]; an id outside [0, V) gives a
 *             row of NaN
 *   w       : [V, ldw >= H] of `wtype`: 0 bf16, 1 f32, 3 e4m3fn, 4 int8, 5 e5m2
 *   row_scale: f32 [V] for the 1-byte types (rounded to the output type before
 *             the product, as the reference does), else NULL
 *   out     : [N, ldo >= H] of `otype`: 0 bf16, 1 f32, 2 f16
 * N < 2^24, V <= 2^27, H <= 2^20.
 */
int qmoe_vocab_lookup(const void* ids, int ids_i64, int64_t N, const void* w, int wtype, int64_t ldw,
                      const float* row_scale, int64_t V, int64_t H, float scale, void* out, int otype, int64_t ldo,
                      qmoe_stream_t stream);

/*
 * Gradient of the lookup with respect to the table (no counterpart in the
 * reference, which serves only): dw[v] = round(scale * sum of grad[n] over
 * ids[n] == v), in float32 and in a fixed order: the valid ids are sorted by
 * (row, n), partial sums are taken per 16 of them (64 above N = 65536), and a
 * row's are joined in order. The same ids and gradients give the same bits on
 * every call; how a row's terms are grouped depends on the other ids. Ids outside [0, V) and `padding_idx`
 * (-1: none) add nothing. add = 0: every row of dw is written (zeros without a
 * token); add = 1: the sums are added to the rows that have a token, the
 * others are neither read nor written. grad [N, ldg >= H], dw [V, lddw >= H] of
 * types 0 bf16 or 1 f32. The workspace needs no initialisation.
 */
int qmoe_vocab_lookup_grad_workspace_size(int64_t N, int64_t V, int64_t H, int64_t* bytes);
int qmoe_vocab_lookup_grad(const void* ids, int ids_i64, int64_t N, const void* grad, int gtype, int64_t ldg, int64_t V,
                           int64_t H, float scale, int64_t padding_idx, void* dw, int wtype, int64_t lddw, int add,
                           void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * Softmax cross entropy of a projection onto the vocabulary table, without
 * the [T, V] logits in memory (no counterpart in the reference, whose head is
 * the full product of `layers/adapter/quantization/fp8.py:1679-1681`):
 *   l[t, v] = s[v] x[t] . w[v],  lse[t] = log sum_v exp l[t, v],
 *   loss[t] = lse[t] - l[t, target[t]]
 *   x         : bf16 [T, ldx >= H]; w [V, ldw >= H] of `wtype`: 0 bf16, 3 e4m3fn,
 *               4 int8, 5 e5m2; row_scale f32 [V] for the 1-byte types, else
 *               NULL. H, ldx and ldw multiples of 8, x and bf16 w 16-byte
 *               aligned, codes 8-byte aligned
 *   targets   : int32, or int64 with targets_i64 [T]; ignore_index gives loss 0
 *               (lse is computed all the same), any other target outside [0, V)
 *               a NaN loss
 *   loss, lse : f32 [T]
 * T <= 2^20, V <= 2^24, H <= 2^16, ceil(V / 256) * ceil(T / 128) <= 2^22. The
 * workspace needs no initialisation.
 */
int qmoe_vocab_loss_workspace_size(int64_t T, int64_t V, int64_t H, int wtype, int64_t* bytes);
int qmoe_vocab_loss(const void* x, int64_t ldx, int64_t T, const void* w, int wtype, int64_t ldw,
                    const float* row_scale, int64_t V, int64_t H, const void* targets, int targets_i64,
                    int64_t ignore_index, float* loss, float* lse, void* workspace, int64_t ws_bytes,
                    qmoe_stream_t stream);

/*
 * The tiles of qmoe_vocab_loss and of the first vocabulary piece of
 * qmoe_vocab_loss_grad for operands of these sizes with contiguous, 16-byte
 * aligned rows: token rows of a tile (dw: table rows), 64 and 128 by eight
 * wavefronts, 192 and 256 by four, 1 for 128 rows without a stage ring. Reads
 * no memory.
 */
typedef struct qmoe_vocab_loss_tiles {
  int32_t logits;      /* of the forward pass */
  int32_t loss_pieces; /* vocabulary pieces of the forward pass (codes expanded first) */
  int32_t probs, dx, dx_slices, dw, grad_pieces;
} qmoe_vocab_loss_tiles;
int qmoe_vocab_loss_plan(int64_t T, int64_t V, int64_t H, int wtype, qmoe_vocab_loss_tiles* plan);

/*
 * Its gradients. g_loss, g_lse (optional): f32 [T] gradients of loss and lse;
 * lse as qmoe_vocab_loss wrote it. With c[t] = (g_loss[t] where the target
 * counts) + g_lse[t]: P[t, v] = exp(l - lse[t]) c[t] - [v == target[t]]
 * g_loss[t], rounded to bf16; dx = P (s w) bf16 [T, lddx >= H], dw = P^T x bf16
 * [V, lddw >= H] (bf16 tables only). Either may be NULL. A token with neither
 * gradient leaves zeros in dx and nothing in dw, whatever its x and its target
 * are. P and the logits exist for one piece of the vocabulary at a time. lddx, lddw multiples
 * of 8, dx and dw 16-byte aligned. Every row of dx and dw is written; the sums'
 * order is fixed.
 */
int qmoe_vocab_loss_grad_workspace_size(int64_t T, int64_t V, int64_t H, int wtype, int need_dx, int need_dw,
                                        int64_t* bytes);
int qmoe_vocab_loss_grad(const void* x, int64_t ldx, int64_t T, const void* w, int wtype, int64_t ldw,
                         const float* row_scale, int64_t V, int64_t H, const void* targets, int targets_i64,
                         int64_t ignore_index, const float* lse, const float* g_loss, const float* g_lse, void* dx,
                         int64_t lddx, void* dw, int64_t lddw, void* workspace, int64_t ws_bytes,
                         qmoe_stream_t stream);

/*
 * Routing with its balance loss and per-expert counts (no counterpart in the
 * reference, which serves only): routes as qmoe_moe_route with float32 weights,
 * then over the counted tokens (token_mask[t] != 0, or all without a mask), N of
 * them, with p[t, e] = s[t, e] / max(sum over e of s[t, e], 1e-20) and counts[e] the
 * counted tokens that chose e,
 *   loss = E / (topk N^2) sum over e of counts[e] sum over t of p[t, e]    (0 for N = 0)
 *   logits      : [T][E] bf16, or f32 with logits_f32; scoring 0..2, bias,
 *                 renormalize, groups as qmoe_moe_route
 *   token_mask  : one byte per token, or NULL. A token outside it is routed, with
 *                 weights 0
 *   topk_weights: f32 [T][topk]; topk_ids i32 [T][topk]; loss f32 [1]; counts i32 [E]
 * 1 <= T <= 2^24, E <= 512. The sums' order is fixed. The workspace is 16-byte
 * aligned and needs no initialisation.
 */
int qmoe_moe_balance_workspace_size(int64_t T, int E, int64_t* bytes);
int qmoe_moe_balance(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring, const float* bias,
                     int renormalize, float routed_scaling_factor, int num_group, int topk_group,
                     const uint8_t* token_mask, float* topk_weights, int32_t* topk_ids, float* loss, int32_t* counts,
                     void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * Its gradient: d_logits [T][E] (the logits' type) for the gradients of
 * topk_weights (f32 [T][topk] or NULL) and of loss (f32 [1] or NULL); topk_ids and
 * counts as qmoe_moe_balance wrote them. A sum below 1e-20 (of the row's scores, or of
 * the weights that are renormalized) counts as a constant. A token outside the mask
 * gets zeros, whatever its logits are.
 */
int qmoe_moe_balance_grad(const void* logits, int logits_f32, int64_t T, int E, int topk, int scoring, int renormalize,
                          float routed_scaling_factor, const uint8_t* token_mask, const int32_t* topk_ids,
                          const int32_t* counts, const float* g_weights, const float* g_loss, void* d_logits,
                          qmoe_stream_t stream);

/*
 * The norms before and after a block, its gate and the residual (no counterpart
 * in the reference, whose models bring their own norms):
 *   n(a; w) = a (mean a^2 + eps)^(-1/2) (weight_offset + w)
 *   b = n(y; post_weight) or y,  h = residual_scale residual + scale gate b,  z = n(h; next_weight)
 * y NULL: h is the residual itself (the norm before a block alone). Types: 0
 * bf16, 1 f32, 2 f16; residual and h of y_type or f32; z and a gate per element
 * of y_type. h is rounded as it is stored before its norm. Rows may be strided. The
 * mean square is float32: a row whose squares add up to infinity (values beyond
 * 1.8e19 / sqrt(H) in size) gives zeros behind its norm.
 */
typedef struct qmoe_block_desc {
  int64_t T, H;            /* rows, 1..2^24; row length, 1..16384 */
  const void* y;           /* [T][ldy] or NULL */
  int64_t ldy;
  const void* residual;    /* [T][ldr] (not read by the gradient) */
  int64_t ldr;
  const void* gate;        /* by gate_kind: NULL, [H], [T], [T][ldg] */
  int64_t ldg;
  const void* post_weight; /* [H] or NULL */
  const void* next_weight; /* [H] or NULL */
  void* h;                 /* [T][ldh]; the gradient reads it (without y: the residual) */
  int64_t ldh;
  void* z;                 /* [T][ldz], with next_weight */
  int64_t ldz;
  float* rstd_y;           /* [T] or NULL: the row factors of the two norms, for the gradient */
  float* rstd_h;
  int32_t y_type, residual_type, weight_type, gate_type;
  int32_t gate_kind;       /* 0 none, 1 per channel, 2 per token, 3 per element */
  float scale, residual_scale, weight_offset, eps;
} qmoe_block_desc;
int qmoe_block_residual(const qmoe_block_desc* d, qmoe_stream_t stream);

/*
 * Its gradients, for those of h and z (either may be NULL). Outputs that are NULL
 * are not computed, and one whose operand is not there (d_next_weight: without
 * g_z) is refused; d_y, d_residual and a per-element d_gate have contiguous rows,
 * and each output its operand's type. The sums over tokens are float32 in a
 * fixed order; the workspace (for weights and a gate per channel) is 16-byte
 * aligned and needs no initialisation.
 */
typedef struct qmoe_block_grads {
  const void* g_h; /* [T][ldgh] of residual_type */
  int64_t ldgh;
  const void* g_z; /* [T][ldgz] of y_type */
  int64_t ldgz;
  void* d_y;
  void* d_residual;
  void* d_gate;
  void* d_post_weight;
  void* d_next_weight;
} qmoe_block_grads;
int qmoe_block_residual_grad_workspace_size(int64_t T, int64_t H, int64_t* bytes);
int qmoe_block_residual_grad(const qmoe_block_desc* d, const qmoe_block_grads* grads, void* workspace, int64_t ws_bytes,
                             qmoe_stream_t stream);

/*
 * 8 bits of a row: for every 32 columns (the last ones may be fewer) e4m3fn codes
 * and a byte s, the value being code * 2^(s - 127); s is the least byte with the
 * finite values' absolute maximum <= 448 * 2^(s - 127). Infinities and NaN
 * become NaN codes and count for no scale.
 *
 * Gated activation whose operands wait for the backward pass in 8 bits (no
 * counterpart in the reference): gate = x[t][0..I), up = x[t][I..2I),
 *   h[t] = act(gate, up)
 * as the fused activations of qmoe_gemm; with codes also the 8 bits of gate and up.
 *   x      : [T][ldx >= 2I] of `type`: 0 bf16, 2 f16; act QMOE_ACT_SILU ...
 *   h      : [T][ldh >= I]
 *   codes  : [T][2I] or NULL; scales [T][2][ceil(I / 32)]
 * The gradient evaluates the derivatives at the 8-bit values: dx [T][2I]. A
 * clamp passes the gradient at its limits.
 */
int qmoe_act_checkpoint(const void* x, int64_t ldx, int type, int64_t T, int64_t I, int act, float act_p0,
                        float act_p1, void* h, int64_t ldh, uint8_t* codes, uint8_t* scales, qmoe_stream_t stream);
int qmoe_act_checkpoint_grad(const uint8_t* codes, const uint8_t* scales, int64_t T, int64_t I, int act, float act_p0,
                             float act_p1, const void* dh, int64_t lddh, int type, void* dx, qmoe_stream_t stream);

/*
 * The 8 bits of bf16 rows x [T][ldx >= K]: codes [T][K], scales [T][ceil(K / 32)].
 * K and ldx multiples of 8, x 16-byte aligned, codes 8-byte aligned.
 */
int qmoe_pack_8bit(const void* x, int64_t ldx, int64_t T, int64_t K, uint8_t* codes, uint8_t* scales,
                   qmoe_stream_t stream);

/*
 * A linear layer: y = x w^T + bias, bf16 [T][N], float32 sums and one rounding. x bf16
 * [T][ldx], w bf16 [N][ldw], bias f32 [N] or NULL; sizes and alignment as
 * qmoe_linear_grad. With codes (NULL: without) also the 8 bits of x, as
 * qmoe_pack_8bit.
 */
int qmoe_linear_workspace_size(int64_t T, int64_t N, int64_t K, int64_t* bytes);
int qmoe_linear(const void* x, int64_t ldx, int64_t T, int64_t N, int64_t K, const void* w, int64_t ldw,
                const float* bias, void* y, uint8_t* codes, uint8_t* scales, void* workspace, int64_t ws_bytes,
                qmoe_stream_t stream);

/*
 * Gradients of a linear layer y = x w^T + bias whose input waited in 8 bits:
 *   dx = dy w,  dw = dy^T x8,  dbias = sum over t of dy     (x8: the codes' values, K % 32 == 0, N % 8 == 0)
 *   dy  : bf16 [T][lddy]; w bf16 [N][ldw] (for dx); codes / scales of qmoe_pack_8bit
 *         (for dw); lddy and ldw multiples of 8 below 2^22
 *   dx  : bf16 [T][K]; dw bf16 [N][K]; dbias [N] bf16, or f32 with dbias_f32;
 *         each may be NULL
 * Matrices, codes and workspace are 16-byte aligned. Sums are float32 in a fixed
 * order. 1 <= T <= 2^20, N <= 2^18, K <= 2^16. The workspace needs no initialisation.
 */
int qmoe_linear_grad_workspace_size(int64_t T, int64_t N, int64_t K, int need_dx, int need_dw, int need_dbias,
                                    int64_t* bytes);
int qmoe_linear_grad(const void* dy, int64_t lddy, int64_t T, int64_t N, int64_t K, const void* w, int64_t ldw,
                     const uint8_t* codes, const uint8_t* scales, void* dx, void* dw, void* dbias, int dbias_f32,
                     void* workspace, int64_t ws_bytes, qmoe_stream_t stream);

/*
 * The tiles of qmoe_linear (y) and qmoe_linear_grad (dx, dw) for these sizes: rows
 * of a tile (of x, dy and w's gradient), 64 and 128 by eight wavefronts, 192 and 256
 * by four, 1 for 128 rows without a stage ring; the slices that each product's summed
 * axis (K, N, T) is cut into; and whether dw takes the codes as they are. Reads no memory.
 */
typedef struct qmoe_linear_tiles {
  int32_t y, y_slices, dx, dx_slices, dw, dw_slices, dw_codes;
} qmoe_linear_tiles;
int qmoe_linear_plan(int64_t T, int64_t N, int64_t K, qmoe_linear_tiles* plan);

/*
 * Plain read of `bytes` (a multiple of 16, 16-byte aligned) at `src` by at
 * most `workgroups` 256-thread workgroups; `sink` receives at most one dword
 * per workgroup ([workgroups] uint32, normally untouched). No counterpart in
 * the reference: a measurement helper giving the HBM read floor (time vs
 * size, launch included) that the weight-streaming GEMMs are compared with.
 */
int qmoe_stream_read(const void* src, int64_t bytes, int32_t workgroups, void* sink, qmoe_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* QMOE_H_ */
