/*
 * qrb200_nn.h -- C ABI of libqrb200's sequence and projection operators, beside the QR of
 * qrb200.h and with its conventions: device pointers, all work enqueued on `stream`, nothing
 * allocated, scratch from the caller's 256-byte aligned workspace (one per call in flight),
 * a qrb_status returned, and the per-thread message in qrb_last_error().
 *
 * The gated delta rule carries a state S (dk x dv) per head through scaled Householder-like
 * transforms, in the chunked compact-WY form that blocked QR uses for its reflectors:
 *     S~_t = exp(g_t) S_{t-1},  u_t = beta_t (v_t - S~_t^T k_t),  S_t = S~_t + k_t u_t^T,
 *     o_t = scale S_t^T q_t.
 */
#ifndef QRB200_NN_H
#define QRB200_NN_H

#include "qrb200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum qrb_dtype { QRB_F32 = 0, QRB_BF16 = 1, QRB_F16 = 2 };
enum qrb_activation { QRB_ACT_NONE = 0, QRB_ACT_RELU = 1, QRB_ACT_SILU = 2, QRB_ACT_GELU = 3 };

#define QRB_DELTA_MAX_DK 128
#define QRB_DELTA_MAX_DV 256

/* Strides in elements of a (batch, time, heads, d) tensor whose last dimension is dense. */
typedef struct {
  int64_t batch, time, head;
} qrb_strides;

/* One call of the gated delta rule over whole sequences.  q, k have hk heads, v, g, beta, o hv
 * heads (a multiple of hk; value head h uses q/k head h / (hv / hk)).
 * Layout: seq_offsets NULL: `batch` sequences of `time` tokens each, nseq == batch.  Otherwise
 * batch == 1 and sequence i is tokens [seq_offsets[i], seq_offsets[i+1]) of the `time` tokens;
 * offsets lie on the device, start at 0 and do not decrease (others are clamped to the tensors:
 * no access leaves them, but results are unspecified).  Empty sequences are allowed.  Rows behind
 * the last sequence are not read; outputs there stay as they are, or with zero_tail become 0.
 * g may be positive as long as its sum over any stretch of a sequence stays below 88 (exp of it must be
 * finite); -inf (and all below -120) empties the state.
 * Forward:  q, k, v, g, beta, initial_state (NULL: zeros) -> o, final_state (NULL: not stored).
 * Backward: also d_o and dfinal_state (NULL: zeros) -> dq, dk_, dv_, dg, dbeta (dense, shaped like
 * q, k, v, g, beta) and dinitial_state (NULL: not stored); dg is good to about 1e-6 of the sums of
 * o do and v dv over a chunk, which it is the difference of.  States are dense fp32 (nseq, hv, dk, dv);
 * final_state may be initial_state.  Else no output may overlap a state, seq_offsets or another
 * output, and no gradient an input.  A value that is not finite (a state, u or an fp32 input above
 * 3.38e38 counts as one) may spoil every output of its sequence from the start of its 64-token chunk,
 * and every gradient of its sequence. */
typedef struct {
  int dtype;                       /* qrb_dtype of q, k, v, o and their gradients */
  int hk, hv, dk, dv;
  int64_t batch, time, nseq;
  const int32_t* seq_offsets;
  float scale;
  int zero_tail;
  const void *q, *k, *v;
  qrb_strides q_strides, k_strides, v_strides;
  const float *g, *beta;
  qrb_strides g_strides, beta_strides;
  const float* initial_state;
  void* o;
  qrb_strides o_strides;
  float* final_state;
  const void* d_o;
  qrb_strides do_strides;
  const float* dfinal_state;
  void *dq, *dk_, *dv_;
  float *dg, *dbeta, *dinitial_state;
} qrb_delta_args;

/* Bytes of workspace for a call of these sizes; 0 for invalid ones. */
QRB_API size_t qrb_delta_workspace_size(const qrb_delta_args* a, int backward);
QRB_API int qrb_delta_forward(const qrb_delta_args* a, void* workspace, size_t workspace_bytes, void* stream);
QRB_API int qrb_delta_backward(const qrb_delta_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* One token per row, for generation: row i reads state slots[i] (slots NULL: i) of `state`
 * (num_slots x hv x dk x dv, fp32, the last three dense, slot_stride elements apart), writes the
 * advanced state to the same slot of state_out (which may be `state`) and o.  A row whose slot is
 * negative is padding: its o is 0 and no state is touched.  A row whose slot is num_slots or more,
 * or is held by an earlier row, gets o = NaN and no state is touched.  o may be v; else neither output may overlap
 * an input or the other.  No workspace. */
typedef struct {
  int dtype;
  int hk, hv, dk, dv;
  int64_t batch, num_slots;
  float scale;
  const void *q, *k, *v;           /* strides: batch and head are used */
  qrb_strides q_strides, k_strides, v_strides;
  const float *g, *beta;
  qrb_strides g_strides, beta_strides;
  const int32_t* slots;
  const float* state;
  float* state_out;
  int64_t slot_stride, slot_stride_out;
  void* o;                         /* dense (batch, hv, dv) */
} qrb_delta_step_args;
QRB_API int qrb_delta_step(const qrb_delta_step_args* a, void* stream);

/* The linear layer y = act(x w^T + bias) + residual: x (m x k), w (n x k), y (m x n), row-major with
 * row strides ldx, ldw, ... in elements, all of one dtype; fp32 accumulation, rounded once.  bias (n),
 * residual and pre (m x n) may be NULL; pre receives x w^T + bias, rounded, for the backward pass.
 * fp32 products carry fp32 accuracy (three bf16 planes per operand; below 2^-109 the last ones underflow).  Results repeat.  y may be
 * residual (same rows); it must not alias x, w or bias.  The workspace size depends on the pointers'
 * alignment as well as on the sizes. */
typedef struct {
  int dtype, activation;           /* qrb_dtype, qrb_activation (GELU: the exact, erf form) */
  int64_t m, k, n;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* y;
  int64_t ldy;
  void* pre;
  int64_t ldpre;
} qrb_linear_args;
QRB_API size_t qrb_linear_workspace_size(const qrb_linear_args* a);
QRB_API int qrb_linear_forward(const qrb_linear_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Its backward pass: dp = dy act'(pre), dx = dp w, dw = dp^T x, dbias = column sums of dp (the
 * residual's gradient is dy).  pre is what the forward call stored (not read without an activation);
 * dx (m x k), dw (n x k) and dbias (n) are dense and each may be NULL; x is read for dw, w for dx.  dp
 * of the 16-bit types is rounded to the type once before its two products; dbias is summed before. */
typedef struct {
  int dtype, activation;
  int64_t m, k, n;
  const void* dy;
  int64_t lddy;
  const void* pre;
  int64_t ldpre;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  void *dx, *dw, *dbias;
} qrb_linear_backward_args;
QRB_API size_t qrb_linear_backward_workspace_size(const qrb_linear_backward_args* a);
QRB_API int qrb_linear_backward(const qrb_linear_backward_args* a, void* workspace, size_t workspace_bytes,
                                void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QRB200_NN_H */
