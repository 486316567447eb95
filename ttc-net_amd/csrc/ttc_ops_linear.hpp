// ttc_ops_linear.hpp -- linear attention with a decay for each head: the one sweep that all its passes are.
//
//   S_t = e^{g_t} S_{t-1} + k_t v_t',   o_t = scale S_t' q_t
// and with R_t the gradient of S_t,
//   dq_t = scale S_t do_t,   R_t = scale q_t do_t' + e^{g_{t+1}} R_{t+1},   dk_t = R_t v_t,   dv_t = R_t' k_t,
// so that, written sweep(query, key, value) -> out,
//   o = sweep(q, k, v),  dq = sweep(do, v, k),  dv = reverse sweep(k, q, do),  dk = reverse sweep(v, do, q):
// one kernel, in four roles (the state transposed where the roles of dk and dv swap).  In reverse order the decay that
// is applied before token t is that of token t + 1 (none before the last token), and that of token 0 after the end.
// The decays' gradient needs no state either: with the dots r_t = q_t.dq_t and c_t = k_t.dk_t,
//   dg_t = sum_{u >= t} (r_u - c_u) + <S_T, dS_T>,
// and, so that the rounding of a long sum of cancelling terms does not add up, dg_t = e^{g_t} <S_{t-1}, R_t> itself at a
// boundary every 16 chunks, where the two sweeps' states meet.
#pragma once
#include "ttc_ops_common.hpp"

namespace ttc {

constexpr float RESET = TTC_RESET_LOG_GAMMA;
constexpr int MAX_DIM = TTC_LINEAR_ATTENTION_MAX_DIM;
constexpr int MAX_WAVES = 4;  // of a chunked sweep's workgroup
constexpr int sweep_waves(int vd) { return vd <= 32 ? 2 : MAX_WAVES; }

struct Side {  // one of the sweep's inputs: [batch, token, head, dim], heads shared by `div` heads of the sweep
  const void* p;
  int64_t sb, st, sh;
  int div;
  template <class T>
  __device__ __forceinline__ const T* at(int64_t b, int h) const {
    return static_cast<const T*>(p) + b * sb + (h / div) * sh;
  }
};

struct Sweep {
  Side q, k, v;            // query and key of kd elements, value of vd
  Side x;                  // x.p: the dots out_t . x_t are wanted (vd elements)
  const void* gamma;
  int64_t gb, gt, gh;
  bool gamma_bf16, reverse, out_f32;
  int kd, vd, H;
  int64_t B, T;
  int64_t first;               // head, of all sequences' heads in a row, that this launch begins with
  float key_scale, out_scale;  // of the state's products; of the output
  const float* state_in;       // [slot, head, ...]: element (i, j) at i * sr + j * sc
  float* state_out;
  int sr, sc;
  const int32_t* slots;        // NULL: slot b
  int64_t nslots;
  void* out;                   // [B, T, H, vd] contiguous, of the inputs' type or fp32
  float* dots;                 // [B, H, T], with one more such array for each further tile of columns
  // Boundaries every mark_tokens tokens of a chunked sweep (NULL: none), marks of them with the one before token 0.
  // The sweep of dq leaves the state in front of each, [B, H, marks, kd, vd]; the sweep of dk joins its own state there to
  // the decay's gradient, [B, H, marks + 1, MAX_WAVES] in parts, the last from `last`, the state behind all tokens (laid out
  // as state_out; NULL: none).
  float *states, *joins;
  const float* last;
  int64_t mark_tokens, marks;
};

__device__ __forceinline__ float gamma_at(const Sweep& A, int64_t i) {
  return A.gamma_bf16 ? to_f(static_cast<const __bf16*>(A.gamma)[i]) : static_cast<const float*>(A.gamma)[i];
}

// ---- segments: where heads are few, their tokens are split -----------------------------------------------------

struct Segments {
  int count;          // segments a head
  int64_t chunks;     // chunks a segment
  float* state;       // [batch, head, segment, dk, dv]: a segment's own contribution, then the state in front of it
  int sr, sc;         // the sweep's element (i, j) of it at i * sr + j * sc
  float* decay;       // [batch, head, segment]: its whole decay
};

// Where 16-byte loads of all inputs, and stores of 4 elements at once, are possible
struct Wides {
  bool in, out;
};

enum { STATE_ONLY = 0, FAST = 1, EXACT = 2 };  // what a chunked sweep gives: ttc_ops_linear_chunk.hpp

template <class T>
int launch_chunk_kd32(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s);
template <class T>
int launch_chunk_kd64(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s);
template <class T>
int launch_chunk_kd128(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s);

// Tokens of a chunk: in bf16 64, so that the state's own work is spread over more of them (2,048 tokens of 512 heads of
// 128: 372 us, with 32 tokens 397); in fp32, whose tiles are twice as large, 32
constexpr int chunk_tokens(bool bf16) { return bf16 ? 64 : 32; }

}  // namespace ttc
