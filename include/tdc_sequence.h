/*
 * tdc_sequence.h — C ABI of the sequence operators of libtdc_sm100.so: the
 * causal depthwise convolution over [B, T, C], the norms of queries and keys
 * with the position rotation, and the gated delta rule, chunked and recurrent.
 *
 * Conventions are those of tdc_dwconv.h (status codes, tdc_strerror,
 * tdc_last_cuda_error): plain pointers and 64-bit sizes, `stream` is a
 * cudaStream_t, the caller owns every buffer (all on the CUDA device that is
 * current for the calling thread), the library allocates nothing, never
 * synchronises and keeps nothing between calls.  Argument errors come back
 * before any CUDA call is made.  Calls may run at the same time on several
 * streams as long as they do not share output buffers or workspaces.
 *
 * Element types: TDC_F16 (IEEE binary16) or TDC_BF16; sums, norms,
 * states and decays are fp32.  Strides are in elements; the last dimension of
 * every tensor is contiguous.  Vectorised tensors (x, q, k, v, o and their
 * gradients) need 16-byte aligned base pointers and strides that are multiples
 * of 8 elements.
 *
 * Packed batches: cu_seqlens, if not NULL, is a device array of num_seqs + 1
 * int32 (or int64, cu_is_64 != 0) row offsets that do not decrease; B is then
 * 1 and sequence n owns rows cu_seqlens[n] .. cu_seqlens[n+1] - 1.  Rows that
 * no sequence owns get zeros in every output row of theirs.  The offsets must
 * not decrease and must lie in [0, T]; they are not read on the host, and no
 * value of theirs leads to an access out of range.
 */
#ifndef TDC_SEQUENCE_H_
#define TDC_SEQUENCE_H_

#include "tdc_dwconv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TDC_F16  0
#define TDC_BF16 1

/* ---- causal depthwise convolution -----------------------------------------
 *   z[b,t,c] = bias[c] + sum_{j<K} w[j,c] * x[b, t-(K-1)+j, c]
 *   y = z (TDC_ACT_NONE) or z / (1 + exp(-z)) (TDC_ACT_SILU), rounded once.
 * Inputs before a sequence's start are rows of initial_state [N, K-1, C] (its
 * row K-2 is the input just before t = 0), or zeros if it is NULL.
 * final_state [N, K-1, C] receives the last K-1 inputs of each sequence
 * (counting those of initial_state).  N = num_seqs, or B without cu_seqlens.
 * C % 8 == 0, 2 <= K <= 8; w [K, C], bias [C] (or NULL), states and y
 * contiguous, all of x's type. */
typedef struct tdc_conv1d_args {
  const void* x;
  const void* w;
  const void* bias;
  const void* initial_state;
  void* final_state;
  const void* cu_seqlens;
  void* y;
  int64_t B, T, C, K;
  int64_t x_sb, x_st;
  int64_t num_seqs, cu_is_64;
  int64_t dtype, act;
} tdc_conv1d_args;

TDC_API int tdc_conv1d_fwd(const tdc_conv1d_args* a, void* stream);

/* Gradients of the above from dy (strides dy_sb, dy_st) and, if final_state
 * had a gradient, dfinal [N, K-1, C]: dx [B, T, C] contiguous, dw [K, C],
 * dbias [C] (NULL without a bias) and dinitial [N, K-1, C] (NULL if not
 * wanted).  Of `a`, y and final_state are not read; the weight gradients are
 * summed in a fixed order (same bits every run).  workspace: at least
 * tdc_conv1d_bwd_workspace(a) bytes, 16-byte aligned. */
TDC_API int64_t tdc_conv1d_bwd_workspace(const tdc_conv1d_args* a);
TDC_API int tdc_conv1d_bwd(const tdc_conv1d_args* a, const void* dy, int64_t dy_sb, int64_t dy_st,
                           const void* dfinal, void* dx, void* dw, void* dbias, void* dinitial,
                           void* workspace, int64_t workspace_bytes, void* stream);

/* The same convolution for the next T tokens (usually 1) of B running
 * sequences: request b continues the slot state_indices[b] (int32, or int64
 * with indices_are_64; NULL: slot b) of state [slots, K-1, C], which is
 * updated in place.  A negative index marks padding: its output rows are zero
 * and no state is touched.  An index >= slots, and one that an earlier request
 * of the call has already, touches no state and gives NaN rows. */
typedef struct tdc_conv1d_step_args {
  const void* x;
  const void* w;
  const void* bias;
  void* state;
  const void* state_indices;
  void* y;
  int64_t B, T, C, K;
  int64_t x_sb, x_st;
  int64_t slots, indices_are_64;
  int64_t dtype, act;
} tdc_conv1d_step_args;

TDC_API int tdc_conv1d_step(const tdc_conv1d_step_args* a, void* stream);

/* ---- norms of queries and keys with the position rotation ------------------
 * For each head row x of q [B, T, Hq, D] and k [B, T, Hk, D]:
 *   n = x * rsqrt(mean(x^2) + eps)   (TDC_NORM_RMS)
 *   n = x * rsqrt(sum(x^2) + eps)    (TDC_NORM_L2)
 *   n = x                            (TDC_NORM_NONE)
 * times the weight [D] (or 1 if NULL), then with cos, sin [positions_in_table,
 * R/2] (fp32) the first R values of the row are rotated in pairs by the
 * angle of the row's position: pairs (i, i + R/2), or (2i, 2i+1) if
 * interleaved.  positions: int32 (or int64) [B, T] with strides p_sb, p_st, or
 * NULL for t itself; a position outside the table gives NaN in the rotated
 * values.  One rounding at the end.  D % 8 == 0, 8 <= D <= 256, R % 16 == 0,
 * R <= D.  Either of q and k may have 0 heads. */
#define TDC_NORM_NONE 0
#define TDC_NORM_RMS  1
#define TDC_NORM_L2   2

typedef struct tdc_qk_args {
  const void* q;
  const void* k;
  const void* q_weight;
  const void* k_weight;
  const float* cos;
  const float* sin;
  const void* positions;
  void* q_out;              /* [B, T, Hq, D] contiguous */
  void* k_out;              /* [B, T, Hk, D] contiguous */
  int64_t B, T, Hq, Hk, D, R;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, p_sb, p_st;
  int64_t table_rows, positions_are_64;
  int64_t norm, interleaved, dtype;
  double eps;
} tdc_qk_args;

TDC_API int tdc_qk_norm_rope(const tdc_qk_args* a, void* stream);

/* Gradients: dq, dk (contiguous, of q's and k's shapes) from dq_out, dk_out
 * (strides in go_*), and the weights' gradients dq_weight, dk_weight [D] in
 * the element type (NULL where there is no weight), summed in a fixed order. */
typedef struct tdc_qk_grad_args {
  const void* dq_out;
  const void* dk_out;
  void* dq;
  void* dk;
  void* dq_weight;
  void* dk_weight;
  int64_t gq_sb, gq_st, gq_sh, gk_sb, gk_st, gk_sh;
} tdc_qk_grad_args;

TDC_API int64_t tdc_qk_norm_rope_bwd_workspace(const tdc_qk_args* a);
TDC_API int tdc_qk_norm_rope_bwd(const tdc_qk_args* a, const tdc_qk_grad_args* g, void* workspace,
                                 int64_t workspace_bytes, void* stream);

/* ---- gated delta rule -------------------------------------------------------
 * Each value head keeps a state S [K, V] (fp32) and for each token
 *   S~ = exp(g) S;  u = v - S~^T k;  S = S~ + beta k u^T;  o = scale S^T q.
 * q, k [B, T, H, K], v [B, T, HV, V], g (fp32, the logarithm of the decay) and
 * beta [B, T, HV]; value head i uses query and key head i / (HV / H).
 * K is 64 or 128, V is 64, 128 or 256, HV a multiple of H.  Keys are expected
 * to have a norm of about 1 and beta to lie in [0, 2): then the chunked form's
 * triangular systems are well conditioned, as the recurrence itself is.
 * g below -200 acts as -200 (a decay of 0 in fp32).  A value that is not finite
 * reaches no token before its own, in the chunked form as in the recurrence. */
typedef struct tdc_delta_args {
  const void* q;
  const void* k;
  const void* v;
  const float* g;
  const void* beta;
  const float* initial_state;  /* [N, HV, K, V] or NULL for zeros */
  float* final_state;          /* [N, HV, K, V] or NULL */
  const void* cu_seqlens;
  void* o;                     /* [B, T, HV, V] contiguous */
  int64_t B, T, H, HV, K, V;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t g_sb, g_st, b_sb, b_st;       /* g, beta: heads contiguous */
  int64_t num_seqs, cu_is_64;
  int64_t dtype, beta_is_f32;
  double scale;
} tdc_delta_args;

/* Forward over whole sequences in chunks of 64 tokens.  workspace: at least
 * tdc_delta_fwd_workspace(a) bytes, 256-byte aligned. */
TDC_API int64_t tdc_delta_fwd_workspace(const tdc_delta_args* a);
TDC_API int tdc_delta_fwd(const tdc_delta_args* a, void* workspace, int64_t workspace_bytes,
                          void* stream);

/* The chunked kernels wait for their copies and products on barriers with the
 * limit of tdc_set_wait_timeout_ns; a wait that gives up ends its block, leaves
 * the output incomplete and is reported as for the depthwise kernels (see
 * "pipeline-wait failure detection" in tdc_dwconv.h).  This is the forward in
 * which no copy of chunk `withhold_chunk` (of each sequence) and later ones ever
 * comes, so that the wait for it runs out after timeout_ns: it exists to test
 * that path. */
TDC_API int tdc_delta_fwd_withhold(const tdc_delta_args* a, void* workspace,
                                   int64_t workspace_bytes, int64_t withhold_chunk,
                                   int64_t timeout_ns, void* stream);

/* All gradients of the forward from d_o (strides do_sb, do_st, do_sh) and
 * dfinal [N, HV, K, V] (fp32, or NULL).  Of `a`, o and final_state are not
 * used.  dq, dk, dv are contiguous in the element type (the key heads' sums
 * over their value heads included), dg fp32, dbeta of beta's type, both
 * [B, T, HV]; dinitial [N, HV, K, V] fp32 or NULL.  Same bits every run. */
typedef struct tdc_delta_grad_args {
  const void* d_o;
  const float* dfinal;
  void* dq;
  void* dk;
  void* dv;
  float* dg;
  void* dbeta;
  float* dinitial;
  int64_t do_sb, do_st, do_sh;
} tdc_delta_grad_args;

TDC_API int64_t tdc_delta_bwd_workspace(const tdc_delta_args* a);
TDC_API int tdc_delta_bwd(const tdc_delta_args* a, const tdc_delta_grad_args* g, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* The recurrence for the next T tokens (usually 1) of B running sequences:
 * request b updates slot state_indices[b] of state [slots, HV, K, V] in place
 * (indices as for tdc_conv1d_step).  Of `a`, initial_state, final_state,
 * cu_seqlens and num_seqs are not used. */
TDC_API int tdc_delta_step(const tdc_delta_args* a, float* state, int64_t slots,
                           const void* state_indices, int64_t indices_are_64, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* TDC_SEQUENCE_H_ */
