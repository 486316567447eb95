// ttc_ops_delta.hpp -- the gated delta rule: what its kernels share.
//
//   S_t = e^{g_t} (I - b_t k_t k_t') S_{t-1} + b_t k_t v_t',   o_t = scale S_t' q_t
// With e_t = v_t - e^{g_t} S_{t-1}' k_t, what the state does not yet hold at k_t, this is linear attention with the values
// b_t e_t.  In a chunk of C tokens behind the state S, with G_t the sum of its decays up to token t,
//   N_ts = e^{G_t - G_s} k_t . k_s (s < t),   P_ts = scale e^{G_t - G_s} q_t . k_s (s <= t),
//   (I + N b) E = V - e^G K S,   O = scale e^G Q S + P b E,   S <- e^{G_C} S + (e^{G_C - G} K)' b E,
// where the triangle's inverse needs no state: all chunks' at once (prepare), then the states from chunk to chunk (sweep).
// Backward, with R the gradient of the state behind a chunk and dO given,
//   Z = b (P' dO + e^{G_C - G} K R),   dV = (I + N b)^-T Z,   R <- e^{G_C} R + (scale e^G Q)' dO - (e^G K)' dV
// is such a sweep from the end; what remains needs S, R, E and dV of a chunk alone, all chunks at once (gradients).
#pragma once
#include "ttc_ops_linear.hpp"

namespace ttc {

// What prepare leaves for each chunk of each head
enum { IN, UP, BETA, RK, RQ, DEC, HI, LO, PART, WK, WU, WQ, ROWS };  // C values each:
// IN    e^{G_t}, 0 behind a reset                  UP    e^{G_C - G_t}, 0 in front of one
// RK    1 / |k_t| (1 unless keys are normalised)   RQ    1 / |q_t|
// DEC   e^{g_t}, -1 at a reset                     PART  resets so far
// WK    IN RK      WU  UP RK b      WQ  IN RQ scale
// HI, LO  the two parts of log2(e) G_t, whose sum starts anew at a reset; infinite where it is lost (a NaN, growth beyond e^128)

struct Delta {
  Side q, k, v, d_o;
  const void *gamma, *beta;
  int64_t gb, gt, gh, bb, bt, bh;
  bool gamma_bf16, beta_bf16, normalize;
  bool wide_q, wide_k, wide_v, wide_d, wide_o;  // 16-byte loads; stores of 4 elements at once
  int kd, vd, vdp, H, colblocks;                // vdp: columns of the arrays below, 32, 64 or 128
  int64_t B, T, chunks, first;                  // first: head (or chunk) of all that this launch begins with
  float scale, eps;
  const float* state_in;  // [B, H, kd, vd]
  float* state_out;
  void* o;
  // [B, H, chunks, ...]
  void *inverse, *scores;   // lower triangles of 16 x 16 tiles (the diagonal ones whole), each in its parts: (I + N b)^-1, P b
  float* rows;              // [ROWS, C]
  int* odd;                 // keys or inverse not finite
  float *S, *R;             // [KD, vdp]: states in front of the chunks, gradients behind them (NULL: not kept)
  // Where heads are few their chunks are split into `segs` segments of seg_chunks (1: not split), [B, H, segs, ...]:
  float* seg_state;         // [KD, vdp]: a segment's own part of the state behind it, then the state in front of it
  float* seg_matrix;        // [KD, KD]: what becomes of the state in front of it (its transpose: of the gradient behind it)
  int* seg_dead;            // nothing does, whatever it holds: a reset lies between
  int segs;
  int64_t seg_chunks;
  float *E, *dV;            // [C, vdp]
  // outputs of the gradients' kernel; fp32 for heads that share
  void *dq, *dk, *dv, *dgamma, *dbeta;
  bool dq_f32, dk_f32, wide_dqk, wide_dv;  // stores of 4 elements, of 8
};

// a decay or a strength
__device__ __forceinline__ float gate_value(const void* p, bool bf16, int64_t i) {
  return bf16 ? to_f(static_cast<const __bf16*>(p)[i]) : static_cast<const float*>(p)[i];
}

template <class T>
int launch_delta_kd32(const Delta& A, int what, hipStream_t s);
template <class T>
int launch_delta_kd64(const Delta& A, int what, hipStream_t s);
template <class T>
int launch_delta_kd128(const Delta& A, int what, hipStream_t s);
enum { PREPARE, SWEEP, SWEEP_BACK, GRADIENTS };

// Workgroup numbers go round the 8 XCDs.  Of `blocks` workgroups that read the same data (what they share: `group`), all go to
// one XCD, whose L2 then reads it once.
struct Spread {
  int64_t group;
  int block;
};
__device__ __forceinline__ Spread spread(int64_t first, int blocks) {
  const unsigned round = blockIdx.x / (8 * blocks), at = blockIdx.x % (8 * blocks);
  if (round < gridDim.x / (8 * blocks)) return {first + round * 8 + at % 8, (int)(at / 8)};
  return {first + round * 8 + at / blocks, (int)(at % blocks)};  // fewer than 8 are left
}

int launch_delta_join(const Delta& A, bool back, hipStream_t s);

}  // namespace ttc
