// ttc_ops_linear.hip -- linear attention with a decay for each head: the token-by-token sweep (single tokens of a serving
// batch, short inputs), the joining kernels of the backward, and the C entries (the roles: ttc_ops_linear.hpp).
#include "ttc_ops_linear.hpp"

namespace ttc {

// Token by token with the state in registers: a workgroup holds 32 columns of one head's state, a thread 4 of them for RPT
// rows.  For one token it reads and writes the state once (8 bytes an element against 5 flops): bound by memory.  192
// sequences x 16 states of 128 x 128 in a pool: 87 us for 406 MB, 4.7 TB/s where a copy of 1 GiB reaches 5.2; one sequence of
// 8 states of 64 x 64: 4.6 us, of which the loads' latency is most.  Whole rows of 128 columns a workgroup take the same
// (61.8 us against 61.1 for states in a row), and leave too few workgroups for few sequences (6.7 us against 4.7).
template <class T, int RPT>
__global__ __launch_bounds__(256) void token_sweep_kernel(Sweep A, int tiles, bool wide) {
  constexpr int COLS = 32, STEP = 32;  // columns of a workgroup, rows between a thread's
  __shared__ float part[2][4][COLS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = (int)(blockIdx.x % tiles);
  const int64_t bh = A.first + blockIdx.x / tiles, b = bh / A.H;
  const int h = (int)(bh % A.H);
  const int e0 = tile * COLS + (lane & 7) * 4, r0 = wave * 8 + (lane >> 3);
  const int64_t slot = A.slots ? A.slots[b] : b;
  T* out = static_cast<T*>(A.out) + (b * A.T * A.H + h) * (int64_t)A.vd;
  float* outf = static_cast<float*>(A.out) + (b * A.T * A.H + h) * (int64_t)A.vd;
  if (slot < 0 || slot >= A.nslots) {  // a row without a state
    for (int64_t t = 0; t < A.T; ++t)
      for (int j = threadIdx.x; j < COLS && tile * COLS + j < A.vd; j += 256) {
        const int64_t at = t * A.H * (int64_t)A.vd + tile * COLS + j;
        if (A.out_f32) outf[at] = 0.0f; else out[at] = from_f<T>(0.0f);
      }
    return;
  }
  const int64_t base = (slot * A.H + h) * (int64_t)A.kd * A.vd;
  // Loads come from the nearest place that exists and are dropped afterwards: in branches, each would wait for the last
  float S[RPT][4];
  const bool held[4] = {e0 < A.vd, e0 + 1 < A.vd, e0 + 2 < A.vd, e0 + 3 < A.vd};
  auto row_at = [&](int i) { return r0 + STEP * i < A.kd ? r0 + STEP * i : A.kd - 1; };
  auto col_at = [&](int j) { return held[j] ? e0 + j : A.vd - 1; };
  if (A.state_in == nullptr) {
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = 0.0f;
  } else if (wide) {
    float4 f[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
      f[i] = *reinterpret_cast<const float4*>(A.state_in + base + row_at(i) * A.sr + (held[0] ? e0 : 0));
#pragma unroll
    for (int i = 0; i < RPT; ++i) S[i][0] = f[i].x, S[i][1] = f[i].y, S[i][2] = f[i].z, S[i][3] = f[i].w;
  } else {
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = A.state_in[base + row_at(i) * A.sr + col_at(j) * A.sc];
  }
  const T *q = A.q.at<T>(b, h), *k = A.k.at<T>(b, h), *v = A.v.at<T>(b, h);
  const T* x = A.x.p ? A.x.at<T>(b, h) : nullptr;
  const int64_t g = b * A.gb + h * A.gh;
  for (int64_t n = 0; n < A.T; ++n) {
    const int64_t t = A.reverse ? A.T - 1 - n : n;
    const float lg = !A.reverse ? gamma_at(A, g + t * A.gt) : n == 0 ? 0.0f : gamma_at(A, g + (t + 1) * A.gt);
    float vv[4], kk[RPT], qq[RPT], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = to_f(v[t * A.v.st + col_at(j)]);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      kk[i] = to_f(k[t * A.k.st + row_at(i)]);
      qq[i] = to_f(q[t * A.q.st + row_at(i)]);
    }
    const float decay = expf(lg);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const bool row = r0 + STEP * i < A.kd;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float add = kk[i] * A.key_scale * vv[j];
        S[i][j] = lg < RESET ? add : fmaf(S[i][j], decay, add);
        acc[j] = row ? fmaf(qq[i], S[i][j], acc[j]) : acc[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int m = 8; m <= 32; m <<= 1) acc[j] += __shfl_xor(acc[j], m, 64);
      if (lane < 8) part[n & 1][wave][lane * 4 + j] = acc[j];
    }
    __syncthreads();  // the next token writes the other buffer, and meets this barrier before it comes back to this one
    if (threadIdx.x < COLS) {
      const int j = threadIdx.x, e = tile * COLS + j;
      float o = (part[n & 1][0][j] + part[n & 1][1][j] + part[n & 1][2][j] + part[n & 1][3][j]) * A.out_scale;
      const int64_t at = t * A.H * (int64_t)A.vd + e;
      if (e < A.vd && A.out) {
        if (A.out_f32) outf[at] = o; else out[at] = from_f<T>(o);
      }
      if (x) {
        const float d = lane_sum(e < A.vd ? o * to_f(x[t * A.x.st + e]) : 0.0f, 32);
        if (j == 0) A.dots[(tile * A.B * A.H + bh) * A.T + t] = d;
      }
    }
  }
  if (A.state_out == nullptr) return;
  const float lg = A.reverse && A.T > 0 ? gamma_at(A, g) : 0.0f;
  const float last = expf(lg);
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + STEP * i;
    if (r >= A.kd) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) S[i][j] = !A.reverse ? S[i][j] : lg < RESET ? 0.0f : S[i][j] * last;
    if (wide) {
      if (e0 < A.vd)
        *reinterpret_cast<float4*>(A.state_out + base + r * A.sr + e0) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e0 + j < A.vd) A.state_out[base + r * A.sr + (e0 + j) * A.sc] = S[i][j];
    }
  }
}

inline int token_tiles(int vd) { return (vd + 31) / 32; }

int launch_token_sweep(const Sweep& A, bool bf16, hipStream_t s) {
  const int tiles = token_tiles(A.vd);
  const int64_t blocks = A.B * A.H * tiles;
  const bool wide = A.sc == 1 && A.vd % 4 == 0 && aligned16(A.state_in) && aligned16(A.state_out);
  auto go = [&](auto kernel) {
    return in_launches(blocks, 256, [&](int64_t first, dim3 grid) {
      Sweep part = A;
      part.first = first / tiles;
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, part, tiles, wide);
    }, tiles);
  };
  if (bf16)
    return A.kd <= 32 ? go(token_sweep_kernel<__bf16, 1>) : A.kd <= 64 ? go(token_sweep_kernel<__bf16, 2>)
                                                                       : go(token_sweep_kernel<__bf16, 4>);
  return A.kd <= 32 ? go(token_sweep_kernel<float, 1>) : A.kd <= 64 ? go(token_sweep_kernel<float, 2>)
                                                                    : go(token_sweep_kernel<float, 4>);
}

// Segments' own contributions to the states in front of them: state_in, then decay * state + contribution.  A thread walks
// along one element of the state; 8 loads in flight (32 segments x 16 heads of 128 x 128: 15 us for 67 MB)
__global__ __launch_bounds__(256) void segment_join_kernel(Sweep A, Segments G, int64_t blocks_a_head,
                                                           int64_t first) {
  const int64_t bh = (first + blockIdx.x) / blocks_a_head, elems = (int64_t)A.kd * A.vd;
  const int64_t i = (first + blockIdx.x) % blocks_a_head * 256 + threadIdx.x;
  if (i >= elems) return;
  float run = A.state_in ? A.state_in[bh * elems + i / A.vd * A.sr + i % A.vd * A.sc] : 0.0f;
  float* p = G.state + bh * G.count * elems + i;
  const float* w = G.decay + bh * G.count;
  constexpr int AHEAD = 8;  // contributions in flight
  for (int j = 0; j < G.count; j += AHEAD) {
    float own[AHEAD], decay[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      own[a] = j + a + 1 < G.count ? p[(j + a) * elems] : 0.0f;
      decay[a] = j + a + 1 < G.count ? w[j + a] : 0.0f;
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (j + a < G.count) p[(j + a) * elems] = run;
      run = decay[a] == 0.0f ? own[a] : fmaf(decay[a], run, own[a]);
    }
  }
}

// Gradients of shared heads, one pass over memory (3 x 509 x 12 heads of 48 to 4: 4.8 us, most of it the launch):
// out [rows, heads / share, d] = sums over `share` heads of in [rows, heads, d]
template <class T>
__global__ __launch_bounds__(256) void share_sum_kernel(const float* __restrict__ in, T* __restrict__ out, int64_t first,
                                                        int64_t n, int share, int d) {
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t head = i / d;
  const float* p = in + head * share * d + i % d;
  float a = 0.0f;
  for (int j = 0; j < share; ++j) a += p[(int64_t)j * d];
  out[i] = from_f<T>(a);
}

// dg_t = sum_{u >= t} (r_u - c_u) + what the boundary behind passes on: one wave per sequence, head and stretch between
// boundaries, from its end, 8 tokens a lane at a time, in 64 bits (the sum's terms cancel).  A reset's own gradient is 0,
// and nothing after it reaches tokens before it.  2,048 tokens x 128 heads: 8.6 us, bound by the latency of the loads and
// of the sums across lanes.
constexpr int GATE_TOKENS = 8;
__global__ __launch_bounds__(64) void gate_kernel(Sweep A, const float* __restrict__ r, const float* __restrict__ c,
                                                  int tiles, int waves, const float* __restrict__ last,
                                                  const float* __restrict__ dlast, int64_t elems, void* d_gamma,
                                                  double* __restrict__ per_head, int64_t first) {
  const int lane = threadIdx.x;
  const int64_t stretch = first + blockIdx.x, bh = stretch / A.marks, mark = stretch % A.marks, b = bh / A.H;
  const int64_t BHT = A.B * A.H * A.T;
  const int h = (int)(bh % A.H);
  const int64_t begin = mark * A.mark_tokens, behind = begin + A.mark_tokens < A.T ? begin + A.mark_tokens : A.T;
  double carry = 0.0, total = 0.0;
  if (A.joins) {
    if (mark + 1 < A.marks || dlast)
      for (int w = 0; w < waves; ++w) carry += A.joins[(bh * (A.marks + 1) + mark + 1) * MAX_WAVES + w];
  } else if (dlast) {
    for (int64_t i = lane; i < elems; i += 64) carry += (double)last[bh * elems + i] * dlast[bh * elems + i];
    for (int m = 32; m >= 1; m >>= 1) carry += __shfl_xor(carry, m, 64);
  }
  for (int64_t end = behind; end > begin; end -= 64 * GATE_TOKENS) {
    const int64_t hi = end - lane * GATE_TOKENS;  // this lane: tokens hi - 1 down to hi - 8
    double sum[GATE_TOKENS], run = 0.0;
    bool cut[GATE_TOKENS], cuts = false;
    float rs[GATE_TOKENS], cs[GATE_TOKENS];
#pragma unroll
    for (int i = 0; i < GATE_TOKENS; ++i) {  // all loads at once, from the stretch's first token where there is none
      const int64_t t = hi - 1 - i < begin ? begin : hi - 1 - i;
      rs[i] = r[bh * A.T + t];
      cs[i] = c[bh * A.T + t];
      cut[i] = gamma_at(A, b * A.gb + h * A.gh + t * A.gt) < RESET;
    }
#pragma unroll
    for (int i = 0; i < GATE_TOKENS; ++i) {
      const int64_t t = hi - 1 - i;
      double d = (double)rs[i] - cs[i];
      if (tiles > 1 && t >= begin)
        for (int j = 1; j < tiles; ++j) d += (double)r[j * BHT + bh * A.T + t] - c[j * BHT + bh * A.T + t];
      cut[i] = cut[i] && t >= begin;
      if (t >= begin) run += d;
      if (cut[i]) run = 0.0, cuts = true;
      sum[i] = run;
    }
    // what the lanes before this one pass on: their runs since the last reset among them
    double in = run;
    bool stop = cuts;
    for (int m = 1; m < 64; m <<= 1) {
      const double up = __shfl_up(in, m, 64);
      const bool sup = __shfl_up((int)stop, m, 64);
      if (lane >= m) {
        if (!stop) in += up;
        stop = stop || sup;
      }
    }
    double before = __shfl_up(in, 1, 64);
    const bool sbefore = __shfl_up((int)stop, 1, 64);
    if (lane == 0) before = carry;
    else if (!sbefore) before += carry;
    const double whole = __shfl(in, 63, 64);
    carry = __shfl((int)stop, 63, 64) ? whole : whole + carry;
    bool open = true;
#pragma unroll
    for (int i = 0; i < GATE_TOKENS; ++i) {
      const int64_t t = hi - 1 - i;
      open = open && !cut[i];
      const double d = cut[i] ? 0.0 : open ? sum[i] + before : sum[i];
      if (t < begin) continue;
      total += d;
      if (per_head == nullptr) {
        const int64_t at = (b * A.T + t) * A.H + h;
        if (A.gamma_bf16) static_cast<__bf16*>(d_gamma)[at] = from_f<__bf16>((float)d);
        else static_cast<float*>(d_gamma)[at] = (float)d;
      }
    }
  }
  if (per_head) {
    for (int m = 32; m >= 1; m >>= 1) total += __shfl_xor(total, m, 64);
    if (lane == 0) per_head[stretch] = total;
  }
}

__global__ __launch_bounds__(64) void gate_head_kernel(const double* __restrict__ per_head, int64_t B, int H,
                                                       int64_t marks, bool bf16, void* d_gamma) {
  const int h = blockIdx.x;
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < B * marks; i += 64) a += per_head[(i / marks * H + h) * marks + i % marks];
  for (int m = 32; m >= 1; m >>= 1) a += __shfl_xor(a, m, 64);
  if (threadIdx.x != 0) return;
  if (bf16) static_cast<__bf16*>(d_gamma)[h] = from_f<__bf16>((float)a);
  else static_cast<float*>(d_gamma)[h] = (float)a;
}

// ---- host ----------------------------------------------------------------------------------------------------

// Up to this many tokens are swept one by one; more in chunks.  8 heads of 128: 2, 4, 8 and 16 tokens take 5.8, 7.8, 12.0 and
// 20.6 us one by one, 13.1 us in a chunk; 1,024 heads 25.4, 35.6, 53.5 and 89.9 us against 39
constexpr int64_t TOKEN_SWEEP = 4;

// Segments of a chunked sweep: enough workgroups to fill the GPU's 256 CUs twice, three times up to 64 x 64, four where keys or
// values have up to 32; a segment's keys and values are read once more for the state behind it, so heads that fill the GPU by
// themselves are not split.  Registers let two workgroups of 128 x 128 run beside each other and three of 64 x 64; with 32 on
// one side it is shared memory (128 x 32: two or three of two waves), and the rule is what the table shows.  Head counts that
// do not divide the number leave some of it empty (400 heads of 64 x 64: one segment each).  Workgroups aimed at, us, bf16:
//                                            384      512     768   1,024   1,536
//   8 x 2,048 tokens x 32 heads of 128 x 128 1,373  1,097   1,290   1,138   1,279   (16,381 x 16 forward 177 150 187 171 193)
//   the same, 64 x 128 (128 x 64)              866    714     819     740     834   (887 722 846 723 832)
//   4 x 2,048 tokens x 32 heads of 64 x 64     353    285     276     286     289
//   3 x 4,096 tokens x 32 heads of 64 x 64     498    422     351     427     380
//   8 x 2,048 tokens x 50 heads of 64 x 64     771    770     768     863     710
//   4 x 4,096 tokens x 32 heads of 64 x 32     625    481     390     385     424
//   8 x 4,096 tokens x 32 heads of 32 x 32   1,303    842     615     540     639
//   4 x 4,096 tokens x 32 heads of 32 x 128    784    640     763     645     694   (128 x 32 845 664 797 661 721)
// and in fp32 (8 x 2,048 x 32 of 128 x 128 2,070 2,085 2,231 2,199 2,286)
//   4 x 2,048 tokens x 32 heads of 64 x 64     612    489     456     477     486   (3 x 4,096 x 32 904 753 644 774 679)
//   8 x 4,096 tokens x 32 heads of 32 x 32   1,710  1,327     952     787     733   (32 x 128 1,526 1,214 1,146 1,145 1,077)
inline Segments segments_of(const ttc_linear_attention_args& A) {
  Segments G{};
  const int64_t chunks = ceil_div(A.tokens, chunk_tokens(A.dtype == TTC_DTYPE_BF16)), heads = A.batch * A.heads;
  const int64_t fill = 256 * (A.dk <= 32 || A.dv <= 32 ? 4 : A.dk <= 64 && A.dv <= 64 ? 3 : 2);
  int64_t count = heads > 0 ? fill / heads : 1;
  if (count > chunks / 2) count = chunks / 2;
  if (count < 1) count = 1;
  G.chunks = ceil_div(chunks, count);
  G.count = (int)(chunks > 0 ? ceil_div(chunks, G.chunks) : 1);
  return G;
}

// The states in front of the segments: 0 where the tokens are not split
inline int64_t saved_bytes(const ttc_linear_attention_args& A) {
  const int64_t n = A.tokens > TOKEN_SWEEP ? segments_of(A).count : 1;
  return n > 1 ? A.batch * A.heads * n * A.dk * A.dv * 4 : 0;
}

struct Layout {  // the workspace, in bytes from its start; 0 bytes: not needed
  int64_t seg_state, seg_decay, dq, dk, dv, r, c, last, states, joins, per_head, total;
  int64_t mark_tokens, marks;  // one stretch where the tokens are swept one by one
  int dot_tiles;
  bool gate;
};

inline bool shared_out(int64_t heads, int64_t own) { return heads != own; }

inline Layout layout_of(const ttc_linear_attention_args& A) {
  Layout W{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  if (A.tokens > TOKEN_SWEEP) {
    const int64_t n = segments_of(A).count;
    W.seg_state = take(A.backward || !A.saved ? saved_bytes(A) : 0);
    W.seg_decay = take(n > 1 ? A.batch * A.heads * n * 4 : 0);
  }
  W.dot_tiles = A.tokens > TOKEN_SWEEP ? 1 : token_tiles((int)A.dk);
  W.total = at;
  if (!A.backward) return W;
  const int64_t rows = A.batch * A.tokens * A.heads;
  W.gate = A.d_log_gamma != nullptr;
  W.dq = take(shared_out(A.heads, A.q_heads) && (A.dq || W.gate) ? rows * A.dk * 4 : !A.dq && W.gate ? rows * A.dk * 4 : 0);
  W.dk = take(shared_out(A.heads, A.k_heads) && (A.dk_out || W.gate) ? rows * A.dk * 4
              : !A.dk_out && W.gate                                    ? rows * A.dk * 4
                                                                       : 0);
  W.dv = take(shared_out(A.heads, A.v_heads) && A.dv_out ? rows * A.dv * 4 : 0);
  if (W.gate) {
    W.r = take(rows * W.dot_tiles * 4);
    W.c = take(rows * W.dot_tiles * 4);
    W.last = take(A.d_final_state ? A.batch * A.heads * A.dk * A.dv * 4 : 0);
    const int64_t stretch = 16 * chunk_tokens(A.dtype == TTC_DTYPE_BF16);
    W.mark_tokens = A.tokens > TOKEN_SWEEP ? stretch : TOKEN_SWEEP;
    W.marks = A.tokens > 0 ? ceil_div(A.tokens, W.mark_tokens) : 1;
    if (A.tokens > TOKEN_SWEEP) {
      W.states = take(W.marks > 1 ? A.batch * A.heads * W.marks * A.dk * A.dv * 4 : 0);
      W.joins = take(A.batch * A.heads * (W.marks + 1) * MAX_WAVES * 4);
    }
    W.per_head = take(A.gamma_per_head ? A.batch * A.heads * W.marks * 8 : 0);
  }
  W.total = at;
  return W;
}

inline int linear_check(int64_t dtype, int64_t gamma_dtype, std::initializer_list<int64_t> sizes, int64_t heads,
                        int64_t qh, int64_t kh, int64_t vh, int64_t dk, int64_t dv) {
  for (int64_t v : sizes)
    if (v < 0) return TTC_LQR_EINVAL;
  if (heads < 1 || heads > (1 << 24) || qh < 1 || kh < 1 || vh < 1 || heads % qh || heads % kh || heads % vh || dk < 1 ||
      dk > MAX_DIM || dv < 1 || dv > MAX_DIM || !countable(sizes))
    return TTC_LQR_EINVAL;
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16) return TTC_LQR_EUNSUPPORTED;
  if (gamma_dtype != TTC_DTYPE_F32 && gamma_dtype != dtype) return TTC_LQR_EUNSUPPORTED;
  return TTC_LQR_OK;
}

inline int args_check(const ttc_linear_attention_args& A) {
  return linear_check(A.dtype, A.gamma_dtype, {A.batch, A.tokens, A.heads, MAX_DIM, MAX_DIM}, A.heads, A.q_heads, A.k_heads,
                      A.v_heads, A.dk, A.dv);
}

inline Side side_of(const void* p, const int64_t* st, int64_t heads, int64_t own) {
  return Side{p, st[0], st[1], st[2], (int)(heads / own)};
}

template <class T>
int share_sum(const float* in, void* out, int64_t rows, int64_t own, int64_t heads, int64_t d, hipStream_t s) {
  const int64_t n = rows * own * d;
  return in_launches(ceil_div(n, 256), 256, [&](int64_t first, dim3 grid) {
    hipLaunchKernelGGL(share_sum_kernel<T>, grid, dim3(256), 0, s, in, static_cast<T*>(out), first, n,
                       (int)(heads / own), (int)d);
  });
}

inline Sweep sweep_of(const ttc_linear_attention_args& A) {
  Sweep S{};
  S.gamma = A.log_gamma;
  S.gb = A.gamma_stride[0], S.gt = A.gamma_stride[1], S.gh = A.gamma_stride[2];
  S.gamma_bf16 = A.gamma_dtype == TTC_DTYPE_BF16;
  S.H = (int)A.heads;
  S.B = A.batch;
  S.T = A.tokens;
  S.nslots = A.batch;
  S.key_scale = S.out_scale = 1.0f;
  return S;
}

int launch_chunks(const Sweep& S, const Segments& G, bool bf16, int mode, hipStream_t s) {
  const int vec = bf16 ? 8 : 4;
  auto wide = [&](const Side& x, int dim) {
    return dim % vec == 0 && aligned16(x.p) && x.sb % vec == 0 && x.st % vec == 0 && x.sh % vec == 0 && x.st >= dim &&
           x.st < (1 << 22);  // rows that do not overlap, a chunk's within 2^30 bytes
  };
  const Wides V{(mode == STATE_ONLY || wide(S.q, S.kd)) && wide(S.k, S.kd) && wide(S.v, S.vd) &&
                    (!S.x.p || wide(S.x, S.vd)),
                S.vd % 4 == 0 && aligned16(S.out) && (int64_t)S.H * S.vd < (1 << 22)};
  if (bf16)
    return S.kd <= 32   ? launch_chunk_kd32<__bf16>(S, G, V, mode, s)
           : S.kd <= 64 ? launch_chunk_kd64<__bf16>(S, G, V, mode, s)
                        : launch_chunk_kd128<__bf16>(S, G, V, mode, s);
  return S.kd <= 32   ? launch_chunk_kd32<float>(S, G, V, mode, s)
         : S.kd <= 64 ? launch_chunk_kd64<float>(S, G, V, mode, s)
                      : launch_chunk_kd128<float>(S, G, V, mode, s);
}

// The states in front of the segments of sweep S, whose roles are those of the state [dk, dv] (S.sr = dv, S.sc = 1): read by
// it and by the sweep with the roles of dk and dv swapped
int segment_states(const Sweep& S, Segments& G, bool bf16, hipStream_t s) {
  if (G.count <= 1) return TTC_LQR_OK;
  if (const int rc = launch_chunks(S, G, bf16, STATE_ONLY, s)) return rc;
  const int64_t per = ceil_div((int64_t)S.kd * S.vd, 256), blocks = S.B * S.H * per;
  return in_launches(blocks, 256, [&](int64_t first, dim3 grid) {
    hipLaunchKernelGGL(segment_join_kernel, grid, dim3(256), 0, s, S, G, per, first);
  });
}

}  // namespace ttc

extern "C" size_t ttc_linear_attention_workspace_bytes(const ttc_linear_attention_args* args) {
  using namespace ttc;
  if (!args || args_check(*args) != TTC_LQR_OK) return 0;
  return (size_t)layout_of(*args).total;
}

extern "C" size_t ttc_linear_attention_saved_bytes(const ttc_linear_attention_args* args) {
  using namespace ttc;
  if (!args || args_check(*args) != TTC_LQR_OK) return 0;
  return (size_t)saved_bytes(*args);
}

extern "C" int ttc_linear_attention(const ttc_linear_attention_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_linear_attention_args& A = *args;
  if (const int rc = args_check(A)) return rc;
  const bool some = A.batch > 0 && A.tokens > 0, bf16 = A.dtype == TTC_DTYPE_BF16;
  if (some && (!A.q || !A.k || !A.v || !A.log_gamma)) return TTC_LQR_EINVAL;
  const Layout W = layout_of(A);
  if (W.total > 0 && (!A.workspace || A.workspace_bytes < W.total)) return TTC_LQR_EINVAL;
  if (A.saved && A.saved_bytes < saved_bytes(A)) return TTC_LQR_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Side q = side_of(A.q, A.q_stride, A.heads, A.q_heads), k = side_of(A.k, A.k_stride, A.heads, A.k_heads),
             v = side_of(A.v, A.v_stride, A.heads, A.v_heads), none{};
  char* ws = static_cast<char*>(A.workspace);
  auto space = [&](int64_t at) { return reinterpret_cast<float*>(ws + at); };
  const bool chunked = A.tokens > TOKEN_SWEEP && A.batch > 0;
  Segments G = segments_of(A);
  G.state = A.saved ? A.saved : space(W.seg_state);
  G.decay = space(W.seg_decay);
  int rc = TTC_LQR_OK;
  // exact: the sweep's dots are wanted
  auto sweep = [&](const Sweep& S, bool exact) {
    if (!chunked) return launch_token_sweep(S, bf16, s);
    G.sr = S.sr, G.sc = S.sc;
    return launch_chunks(S, G, bf16, exact ? EXACT : FAST, s);
  };
  const int dk = (int)A.dk, dv = (int)A.dv;
  Sweep S = sweep_of(A);
  S.q = q, S.k = k, S.v = v;
  S.kd = dk, S.vd = dv;
  S.sr = dv, S.sc = 1;
  S.out_scale = (float)A.scale;
  S.state_in = A.initial_state;
  if (!A.backward) {
    if (some && !A.o) return TTC_LQR_EINVAL;
    S.state_out = A.final_state;
    S.out = A.o;
    if (chunked && (rc = segment_states(S, G, bf16, s))) return rc;
    return sweep(S, false);
  }
  if (some && !A.d_o) return TTC_LQR_EINVAL;
  const Side d_o = side_of(A.d_o, A.d_o_stride, A.heads, A.heads);
  const bool gate = W.gate && some;
  if (some && (A.dq || gate)) {  // S transposed: [dv, dk]
    if (chunked && !A.saved && (rc = segment_states(S, G, bf16, s))) return rc;
    S.q = d_o, S.k = v, S.v = k;
    S.x = gate ? q : none;
    S.kd = dv, S.vd = dk;
    S.state_out = gate && A.d_final_state ? space(W.last) : nullptr;
    S.sr = 1, S.sc = dv;
    S.dots = space(W.r);
    S.mark_tokens = W.mark_tokens, S.marks = W.marks;
    S.states = gate && W.marks > 1 ? space(W.states) : nullptr;
    S.out_f32 = shared_out(A.heads, A.q_heads) || !A.dq;
    S.out = S.out_f32 ? space(W.dq) : A.dq;
    if ((rc = sweep(S, gate))) return rc;
  }
  S = sweep_of(A);
  S.reverse = true;
  S.q = k, S.k = q, S.v = d_o;
  S.kd = dk, S.vd = dv;
  S.sr = dv, S.sc = 1;
  S.key_scale = (float)A.scale;
  S.state_in = A.d_final_state;
  const bool want_v = (some && A.dv_out) || A.d_initial_state, want_k = some && (A.dk_out || gate);
  G.state = space(W.seg_state);
  if (chunked && (want_v || want_k) && (rc = segment_states(S, G, bf16, s))) return rc;
  if (want_v) {
    Sweep V = S;
    V.state_out = A.d_initial_state;
    V.out_f32 = shared_out(A.heads, A.v_heads) && A.dv_out;
    V.out = V.out_f32 ? space(W.dv) : A.dv_out;
    if ((rc = sweep(V, false))) return rc;
  }
  if (want_k) {  // R transposed: [dv, dk]
    S.q = v, S.k = d_o, S.v = q;
    S.x = gate ? k : none;
    S.kd = dv, S.vd = dk;
    S.sr = 1, S.sc = dv;
    S.dots = space(W.c);
    S.mark_tokens = W.mark_tokens, S.marks = W.marks;
    S.states = gate && W.marks > 1 ? space(W.states) : nullptr;
    S.joins = gate ? space(W.joins) : nullptr;
    S.last = gate && A.d_final_state ? space(W.last) : nullptr;
    S.out_f32 = shared_out(A.heads, A.k_heads) || !A.dk_out;
    S.out = S.out_f32 ? space(W.dk) : A.dk_out;
    if ((rc = sweep(S, gate))) return rc;
  }
  if (some) {
    const int64_t rows = A.batch * A.tokens;
    auto join = [&](const float* in, void* out, int64_t own, int64_t d) {
      return bf16 ? share_sum<__bf16>(in, out, rows, own, A.heads, d, s) : share_sum<float>(in, out, rows, own, A.heads, d, s);
    };
    if (A.dq && shared_out(A.heads, A.q_heads) && (rc = join(space(W.dq), A.dq, A.q_heads, A.dk))) return rc;
    if (A.dk_out && shared_out(A.heads, A.k_heads) && (rc = join(space(W.dk), A.dk_out, A.k_heads, A.dk))) return rc;
    if (A.dv_out && shared_out(A.heads, A.v_heads) && (rc = join(space(W.dv), A.dv_out, A.v_heads, A.dv))) return rc;
  }
  if (W.gate) {  // of one decay for each head: zero where there are no tokens
    const int64_t stretches = A.batch * A.heads * W.marks;
    S = sweep_of(A);
    S.mark_tokens = W.mark_tokens, S.marks = W.marks;
    S.joins = A.tokens > TOKEN_SWEEP ? space(W.joins) : nullptr;
    const int waves = sweep_waves(dk);  // of the sweep of dk
    double* per_head = A.gamma_per_head ? reinterpret_cast<double*>(space(W.per_head)) : nullptr;
    rc = in_launches(stretches, 64, [&](int64_t first, dim3 grid) {
      hipLaunchKernelGGL(gate_kernel, grid, dim3(64), 0, s, S, space(W.r), space(W.c), W.dot_tiles, waves, space(W.last),
                         some ? A.d_final_state : nullptr, (int64_t)dk * dv, A.d_log_gamma, per_head, first);
    });
    if (rc) return rc;
    if (per_head)
      hipLaunchKernelGGL(gate_head_kernel, dim3((unsigned)A.heads), dim3(64), 0, s, per_head, A.batch, (int)A.heads, W.marks,
                         S.gamma_bf16, A.d_log_gamma);
  }
  return launched();
}

extern "C" int ttc_linear_attention_step(const ttc_linear_attention_step_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_linear_attention_step_args& A = *args;
  if (const int rc = linear_check(A.dtype, A.gamma_dtype, {A.batch, A.heads, MAX_DIM, MAX_DIM}, A.heads, A.q_heads,
                                  A.k_heads, A.v_heads, A.dk, A.dv))
    return rc;
  if (A.slots < 0 || !countable({A.slots, A.heads, MAX_DIM, MAX_DIM}) || (!A.slot_index && A.slots != A.batch))
    return TTC_LQR_EINVAL;
  if (A.batch == 0) return TTC_LQR_OK;
  if (!A.q || !A.k || !A.v || !A.log_gamma || !A.o || (A.slots > 0 && !A.state)) return TTC_LQR_EINVAL;
  auto side = [&](const void* p, const int64_t* st, int64_t own) { return Side{p, st[0], 0, st[1], (int)(A.heads / own)}; };
  Sweep S{};
  S.q = side(A.q, A.q_stride, A.q_heads);
  S.k = side(A.k, A.k_stride, A.k_heads);
  S.v = side(A.v, A.v_stride, A.v_heads);
  S.gamma = A.log_gamma;
  S.gb = A.gamma_stride[0], S.gh = A.gamma_stride[1];
  S.gamma_bf16 = A.gamma_dtype == TTC_DTYPE_BF16;
  S.kd = (int)A.dk, S.vd = (int)A.dv, S.H = (int)A.heads;
  S.B = A.batch, S.T = 1;
  S.key_scale = 1.0f, S.out_scale = (float)A.scale;
  S.state_in = S.state_out = A.state;
  S.sr = S.vd, S.sc = 1;
  S.slots = A.slot_index;
  S.nslots = A.slots;
  S.out = A.o;
  return launch_token_sweep(S, A.dtype == TTC_DTYPE_BF16, reinterpret_cast<hipStream_t>(stream));
}
