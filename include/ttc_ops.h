/* ttc_ops.h -- C ABI of libttc_lqr.so's sequence operators, for models that hold the test-time control
 * layer: rotary positions, group norm with an activation or a gate, causal convolution, linear attention with a
 * decay for each head, the gated delta rule (status codes: ttc_lqr.h).
 *
 * Each call takes one argument block on the host (every field 8 bytes: numbers, device pointers, strides in
 * elements).  The calls read it before they return, allocate nothing, enqueue their work on `stream` (a
 * hipStream_t) and never synchronise.  Work sizes that do not fit their limits and null pointers return
 * TTC_LQR_EINVAL, types that have no kernel TTC_LQR_EUNSUPPORTED, both before anything is enqueued. */
#ifndef TTC_OPS_H
#define TTC_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TTC_DTYPE_F32 0
#define TTC_DTYPE_BF16 1

/* ---- Rotary positions ----
 * Pairs (x_a, x_b) of a head's first `rot` components become (x_a c - x_b s, x_a s + x_b c) with (c, s) the
 * table's entry of the token's position and the pair (the backward: s negated); the rest of the head is copied.
 * Pair i is (i, i + rot / 2), or (2 i, 2 i + 1) with `interleaved`.  Both arrays x[0] (queries) and x[1] (keys;
 * heads[1] = 0: none) are [batch, tokens, heads, dim] with unit stride along dim; y contiguous, not
 * overlapping x.  table: [length, rot / 2, 2] fp32 contiguous.  positions: NULL (token t has position
 * first + t) or indices of 4 or 8 bytes; a position outside the table gives a row of NaN in the rotated part. */
typedef struct {
  int64_t dtype, batch, tokens, dim, rot, interleaved, backward;
  int64_t heads[2];
  const void* x[2];
  int64_t stride[2][3]; /* batch, token, head */
  void* y[2];
  const float* table;
  int64_t length;
  const void* positions;
  int64_t position_bytes, position_stride[2]; /* batch, token */
  int64_t first;
} ttc_rotary_args;

int ttc_rotary(const ttc_rotary_args* args, void* stream);

/* Positions with several axes (time, height and width of a picture's or video's token): pair i takes its position from the
 * axis in whose section it lies, the first section[0] pairs from axis 0 and so on, and (c, s) from the table's entry of that
 * position and pair i; a position outside the table gives NaN in its axis's pairs.  rot / 2 is the sections' sum (at most
 * dim / 2), the table [length, rot / 2, 2]; axes: 1 to TTC_ROTARY_MAX_AXES; everything else as above. */
#define TTC_ROTARY_MAX_AXES 4
typedef struct {
  int64_t dtype, batch, tokens, dim, interleaved, backward, axes;
  int64_t section[TTC_ROTARY_MAX_AXES];
  int64_t heads[2];
  const void* x[2];
  int64_t stride[2][3]; /* batch, token, head */
  void* y[2];
  const float* table;
  int64_t length;
  const void* positions;
  int64_t position_bytes, position_stride[3]; /* batch, token, axis */
} ttc_rotary_axes_args;

int ttc_rotary_axes(const ttc_rotary_axes_args* args, void* stream);

/* ---- Causal convolution of each channel, channels last ----
 * y_t = act(bias + sum_j weight[c, j] w_{t + j}) with w the initial state's taps - 1 rows (NULL: zeros) followed by x, so that
 * tap taps - 1 meets x_t itself.  activation 0: none, 1: silu.  x [batch, tokens, channels] with unit stride along the
 * channels; weight [channels, taps] and bias [channels] (NULL: none) of type weight_dtype (fp32, or dtype); taps: 1 to
 * TTC_CAUSAL_CONV_MAX_TAPS.  y contiguous; final_state (NULL: not wanted): the last taps - 1 rows of w, contiguous
 * [batch, taps - 1, channels] as initial_state, both of x's type.
 * The backward takes d_y (unit stride along the channels) and d_final_state (NULL: zero) and writes dx, d_initial_state
 * (contiguous, x's type), dweight and dbias (weight_dtype; zero where there are no sequences or no tokens); NULL: not wanted.
 * workspace: ttc_causal_conv_workspace_bytes() of the same block (0: none needed). */
#define TTC_CAUSAL_CONV_MAX_TAPS 8
typedef struct {
  int64_t dtype, weight_dtype, batch, tokens, channels, taps, activation, backward;
  const void* x;
  int64_t x_stride[2]; /* batch, token */
  const void *weight, *bias, *initial_state;
  void *y, *final_state;
  const void* d_y;
  int64_t d_y_stride[2];
  const void* d_final_state;
  void *dx, *dweight, *dbias, *d_initial_state;
  void* workspace;
  int64_t workspace_bytes;
} ttc_causal_conv_args;

size_t ttc_causal_conv_workspace_bytes(const ttc_causal_conv_args* args);
int ttc_causal_conv(const ttc_causal_conv_args* args, void* stream);

/* One token of each sequence, its state updated in place: x [batch, channels] with unit stride along the channels, y
 * contiguous.  state [slots, taps - 1, channels] of x's type, contiguous; slot_index as in ttc_linear_attention_step. */
typedef struct {
  int64_t dtype, weight_dtype, batch, channels, taps, activation, slots;
  const void* x;
  int64_t x_stride;
  const void *weight, *bias;
  void* state;
  const int32_t* slot_index;
  void* y;
} ttc_causal_conv_step_args;

int ttc_causal_conv_step(const ttc_causal_conv_step_args* args, void* stream);

/* ---- Group norm with an activation or a gate, channels last ----
 * x [n, l, c] contiguous; statistics over the l positions and the c / groups channels of a group, biased
 * variance.  y0 = (x - mean) rstd weight + bias; y = act(y0), or y0 act(gate) where gate is not NULL.
 * activation 0: none, 1: silu (z sigmoid(z)).  weight and bias (both or neither, type weight_dtype): [c].
 * mean, rstd [n, groups] fp32: written by the forward (NULL: not kept), read by the backward.  The backward
 * writes dx, dgate (with a gate), dweight and dbias (zero where n or l is 0); NULL: not wanted.
 * workspace: ttc_group_norm_workspace_bytes() of the same block (0: none needed). */
typedef struct {
  int64_t dtype, weight_dtype, n, l, c, groups, activation, backward;
  double eps;
  const void *x, *gate, *weight, *bias;
  float *mean, *rstd;
  void* y;
  const void* dy;
  void *dx, *dgate, *dweight, *dbias;
  void* workspace;
  int64_t workspace_bytes;
} ttc_group_norm_args;

size_t ttc_group_norm_workspace_bytes(const ttc_group_norm_args* args);
int ttc_group_norm(const ttc_group_norm_args* args, void* stream);

/* ---- Linear attention with a decay for each head ----
 * For each sequence and head, with a state S [dk, dv] held in fp32 and g = log_gamma of the token and head,
 *   S_t = e^{g_t} S_{t-1} + k_t v_t',   o_t = scale S_t' q_t.
 * A log_gamma below TTC_RESET_LOG_GAMMA (e^g is 0 in fp32; -inf included) drops the state: what came before has no
 * effect on what follows, whatever it held.  Tokens after t have no effect on o_t, whatever they hold.
 * q, k [batch, tokens, q_heads / k_heads, dk], v [batch, tokens, v_heads, dv]: unit stride along the last dimension;
 * each head count divides `heads`, and head h reads head h / (heads / q_heads) of q.  log_gamma: any strides over
 * batch, tokens and heads (0 for batch and tokens: one decay for each head), of type gamma_dtype (fp32, or dtype).
 * dk, dv: 1 to TTC_LINEAR_ATTENTION_MAX_DIM.  initial_state (NULL: zero), final_state (NULL: not wanted)
 * [batch, heads, dk, dv] fp32 contiguous; o [batch, tokens, heads, dv] contiguous.
 * The backward takes d_o (unit stride along dv) and d_final_state (NULL: zero) and writes dq, dk_out, dv_out (contiguous,
 * of q's, k's and v's shapes), d_log_gamma (contiguous [batch, tokens, heads], or [heads] with gamma_per_head) and
 * d_initial_state; NULL: not wanted.
 * saved: NULL, or ttc_linear_attention_saved_bytes() that the forward fills (states between the parts that long inputs are
 * swept in) and the backward of the same inputs reads instead of computing them again.
 * workspace: ttc_linear_attention_workspace_bytes() of the same block (the backward's where `backward` is set). */
#define TTC_LINEAR_ATTENTION_MAX_DIM 128
#define TTC_RESET_LOG_GAMMA -104.0f
typedef struct {
  int64_t dtype, gamma_dtype, gamma_per_head, backward;
  int64_t batch, tokens, heads, q_heads, k_heads, v_heads, dk, dv;
  double scale;
  const void *q, *k, *v, *log_gamma;
  int64_t q_stride[3], k_stride[3], v_stride[3], gamma_stride[3]; /* batch, token, head */
  const float* initial_state;
  void* o;
  float* final_state;
  const void* d_o;
  int64_t d_o_stride[3];
  const float* d_final_state;
  void *dq, *dk_out, *dv_out, *d_log_gamma;
  float* d_initial_state;
  float* saved;
  int64_t saved_bytes;
  void* workspace;
  int64_t workspace_bytes;
} ttc_linear_attention_args;

size_t ttc_linear_attention_workspace_bytes(const ttc_linear_attention_args* args);
size_t ttc_linear_attention_saved_bytes(const ttc_linear_attention_args* args);
int ttc_linear_attention(const ttc_linear_attention_args* args, void* stream);

/* One token of each sequence, its state updated in place: q, k, v, log_gamma as above without the token dimension,
 * o [batch, heads, dv] contiguous.  state [slots, heads, dk, dv] fp32 contiguous; row b's state is slot slot_index[b]
 * (int32; NULL: slot b, and slots = batch).  A row whose index lies outside [0, slots) is skipped: its output is 0 and
 * no state changes.  Rows must not share a slot. */
typedef struct {
  int64_t dtype, gamma_dtype, batch, heads, q_heads, k_heads, v_heads, dk, dv, slots;
  double scale;
  const void *q, *k, *v, *log_gamma;
  int64_t q_stride[2], k_stride[2], v_stride[2], gamma_stride[2]; /* batch, head */
  float* state;
  const int32_t* slot_index;
  void* o;
} ttc_linear_attention_step_args;

int ttc_linear_attention_step(const ttc_linear_attention_step_args* args, void* stream);

/* ---- The gated delta rule ----
 * Linear attention whose state forgets, before it takes up v_t at k_t, what it holds there: with strengths b = beta,
 *   S_t = e^{g_t} (I - b_t k_t k_t') S_{t-1} + b_t k_t v_t',   o_t = scale S_t' q_t.
 * normalize: q and k stand for q / sqrt(|q|^2 + eps) and k / sqrt(|k|^2 + eps).  Keys longer than sqrt(2 / b) make the state
 * grow.  beta [batch, tokens, heads]: any strides, of type beta_dtype (fp32, or dtype), like log_gamma (which has all three
 * dimensions here).  Everything else as in ttc_linear_attention; resets (TTC_RESET_LOG_GAMMA) too.
 * saved: NULL, or ttc_delta_rule_saved_bytes() that the forward fills and the backward of the same inputs needs.
 * workspace: ttc_delta_rule_workspace_bytes() of the same block (whether `saved` is there counts).  Both at addresses of 16
 * bytes. */
typedef struct {
  int64_t dtype, gamma_dtype, beta_dtype, normalize, backward;
  int64_t batch, tokens, heads, q_heads, k_heads, v_heads, dk, dv;
  double scale, eps;
  const void *q, *k, *v, *log_gamma, *beta;
  int64_t q_stride[3], k_stride[3], v_stride[3], gamma_stride[3], beta_stride[3]; /* batch, token, head */
  const float* initial_state;
  void* o;
  float* final_state;
  const void* d_o;
  int64_t d_o_stride[3];
  const float* d_final_state;
  void *dq, *dk_out, *dv_out, *d_log_gamma, *d_beta;
  float* d_initial_state;
  void* saved;
  int64_t saved_bytes;
  void* workspace;
  int64_t workspace_bytes;
} ttc_delta_rule_args;

size_t ttc_delta_rule_workspace_bytes(const ttc_delta_rule_args* args);
size_t ttc_delta_rule_saved_bytes(const ttc_delta_rule_args* args);
int ttc_delta_rule(const ttc_delta_rule_args* args, void* stream);

/* One token of each sequence, its state updated in place: as ttc_linear_attention_step. */
typedef struct {
  int64_t dtype, gamma_dtype, beta_dtype, normalize, batch, heads, q_heads, k_heads, v_heads, dk, dv, slots;
  double scale, eps;
  const void *q, *k, *v, *log_gamma, *beta;
  int64_t q_stride[2], k_stride[2], v_stride[2], gamma_stride[2], beta_stride[2]; /* batch, head */
  float* state;
  const int32_t* slot_index;
  void* o;
} ttc_delta_rule_step_args;

int ttc_delta_rule_step(const ttc_delta_rule_step_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TTC_OPS_H */
