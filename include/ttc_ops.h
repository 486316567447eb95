/* ttc_ops.h -- C ABI of libttc_lqr.so's sequence operators, for models that hold the test-time control
 * layer: rotary positions, group norm with an activation or a gate, linear attention with a decay for
 * each head (status codes: ttc_lqr.h).
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

/* ---- Group norm with an activation or a gate, channels last ----
 * x [n, l, c] contiguous; statistics over the l positions and the c / groups channels of a group, biased
 * variance.  y0 = (x - mean) rstd weight + bias; y = act(y0), or y0 act(gate) where gate is not NULL.
 * activation 0: none, 1: silu (z sigmoid(z)).  weight and bias (both or neither, type weight_dtype): [c].
 * mean, rstd [n, groups] fp32: written by the forward (NULL: not kept), read by the backward.  The backward
 * writes dx, dgate (with a gate), dweight and dbias (NULL: not wanted).
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

#ifdef __cplusplus
}
#endif

#endif /* TTC_OPS_H */
