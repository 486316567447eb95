// ttc_ops_conv.hip -- causal convolution of each channel over a few tokens, forward, backward and single tokens.
//
//   w = [state; x] (taps - 1 rows more than x),  p_t = bias + sum_j c_j w_{t + j},  y_t = act(p_t)
// and with e_t = dy_t act'(p_t), zero outside [0, T),
//   dw_i = sum_j c_j e_{i - j} (+ the final state's gradient),  dc_j = sum_t e_t w_{t + j},  dbias = sum_t e_t.
// A thread holds 4 neighbouring channels and walks along a run of tokens with the last `taps` rows in registers,
// so that a row is read from memory once (and once more from the caches at the start of each run).
// Bound: memory.  16,381 tokens x 6,144 channels of 4 taps in bf16: 76 us for 403 MB, 5.4 TB/s; training on 4 x 2,048 x 4,096: 28
// us forward, 58 to 61 us backward for 201 MB (3.4 TB/s: the K - 1 tokens in front of each run, and three waves a SIMD); one token of
// 16 sequences: 3.7 us.
#include "ttc_ops_common.hpp"

namespace ttc {

constexpr int MAX_TAPS = TTC_CAUSAL_CONV_MAX_TAPS;

struct Conv {
  const void *x, *weight, *bias, *state;
  int64_t xb, xt, B, T, C;
  bool weight_bf16, wide_weight;
  void *y, *final_state;
  const void *dy, *dfinal;
  int64_t yb, yt;
  void *dx, *dstate;
  float* part;  // [row of workgroups, taps + 1, C]: sums of the weights' and the bias's gradients
  int64_t run, runs;  // tokens a thread, such runs a sequence
  int64_t cols;       // vectors of a row
};

template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

// 1 / (1 + e^-z): the reciprocal as one instruction, off by one unit in the last place, as an exact division costs as much as all
// taps (the same: 151 us, so 136)
__device__ __forceinline__ float gate(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

template <class T, int V>
__device__ __forceinline__ void floats(const Vec<T, V>& a, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(a.v[i]);
}

template <class T, int V>
__device__ __forceinline__ void get(const T* p, float (&f)[V]) {
  const Vec<T, V> a = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(a.v[i]);
}

template <class T, int V>
__device__ __forceinline__ void put(T* p, const float (&f)[V]) {
  Vec<T, V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = a;
}

// A thread's V K taps lie one after the other: 16 bytes at a time where they can be (`wide`).  With 8 channels a thread, prompt of
// 16,381 tokens x 6,144 channels: 32 taps one by one for 8 tokens 215 us, together for 16 tokens 151
template <class W, int K, int V>
__device__ __forceinline__ void taps_from(const W* p, bool wide, float (&w)[K][V]) {
  constexpr int E = 16 / sizeof(W);
  if constexpr (V > 1 && K * V % E == 0) {
    if (wide) {
#pragma unroll
      for (int k = 0; k < K * V / E; ++k) {
        const Vec<W, E> a = reinterpret_cast<const Vec<W, E>*>(p)[k];
#pragma unroll
        for (int i = 0; i < E; ++i) w[(k * E + i) % K][(k * E + i) / K] = to_f(a.v[i]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = to_f(p[i * K + j]);
}

template <int K, int V>
__device__ __forceinline__ void weights(const Conv& A, int64_t c, float (&w)[K][V], float (&b)[V]) {
  if (A.weight_bf16) taps_from<__bf16, K, V>(static_cast<const __bf16*>(A.weight) + c * K, A.wide_weight, w);
  else taps_from<float, K, V>(static_cast<const float*>(A.weight) + c * K, A.wide_weight, w);
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = 0.0f;
  if (A.bias == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i)
    b[i] = A.weight_bf16 ? to_f(static_cast<const __bf16*>(A.bias)[c + i]) : static_cast<const float*>(A.bias)[c + i];
}

// row i of w = [state; x], for 0 <= i < T + K - 1
template <class T, int K, int V>
__device__ __forceinline__ Vec<T, V> wide_row(const Conv& A, int64_t b, int64_t i, int64_t c) {
  if (i >= K - 1) return *reinterpret_cast<const Vec<T, V>*>(static_cast<const T*>(A.x) + b * A.xb + (i - (K - 1)) * A.xt + c);
  if (A.state) return *reinterpret_cast<const Vec<T, V>*>(static_cast<const T*>(A.state) + (b * (K - 1) + i) * A.C + c);
  Vec<T, V> none;
#pragma unroll
  for (int j = 0; j < V; ++j) none.v[j] = from_f<T>(0.0f);
  return none;
}

template <int K, int V>
__device__ __forceinline__ void taps_of(const float (&w)[K][V], const float (&b)[V], const float (&row)[K][V], float (&p)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = b[i];
#pragma unroll
    for (int j = 0; j < K; ++j) p[i] = fmaf(w[j][i], row[j][i], p[i]);
  }
}

constexpr int FORWARD_RUN = 16;  // tokens a thread

// All rows of a run are asked for at once, and taken from 16 bits when their turn comes.
template <class T, int K, int V, bool SILU>
__global__ __launch_bounds__(256) void conv_kernel(Conv A, int64_t first, int64_t items) {
  const int64_t item = (first + blockIdx.x) * 256 + threadIdx.x;
  if (item >= items) return;
  const int64_t c = item % A.cols * V, rest = item / A.cols, run = rest % A.runs, b = rest / A.runs;
  const int64_t t0 = run * FORWARD_RUN, last = A.T + K - 2;  // of w's rows
  Vec<T, V> rows[FORWARD_RUN + K - 1];
  float w[K][V], bias[V], now[K][V];
  if (t0 >= K - 1) {
    const T* x = static_cast<const T*>(A.x) + b * A.xb + (t0 - (K - 1)) * A.xt + c;
    const int left = last - t0 < FORWARD_RUN + K - 2 ? (int)(last - t0) : FORWARD_RUN + K - 2;
#pragma unroll
    for (int i = 0; i < FORWARD_RUN + K - 1; ++i) rows[i] = *reinterpret_cast<const Vec<T, V>*>(x + (i < left ? i : left) * A.xt);
  } else {
#pragma unroll
    for (int i = 0; i < FORWARD_RUN + K - 1; ++i) rows[i] = wide_row<T, K, V>(A, b, t0 + i < last ? t0 + i : last, c);
  }
  weights<K, V>(A, c, w, bias);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) floats(rows[j], now[j + 1]);
#pragma unroll
  for (int i = 0; i < FORWARD_RUN; ++i) {
    if (t0 + i >= A.T) break;
    float p[V];
#pragma unroll
    for (int j = 0; j + 1 < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) now[j][k] = now[j + 1][k];
    floats(rows[i + K - 1], now[K - 1]);
    taps_of<K, V>(w, bias, now, p);
    if (SILU) {
#pragma unroll
      for (int k = 0; k < V; ++k) p[k] *= gate(p[k]);
    }
    put<T, V>(static_cast<T*>(A.y) + (b * A.T + t0 + i) * A.C + c, p);
  }
  if (K > 1 && A.final_state && run == A.runs - 1) {
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
      *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(A.final_state) + (b * (K - 1) + i) * A.C + c) =
          wide_row<T, K, V>(A, b, A.T + i, c);
  }
}

// Four runs a workgroup, 64 vectors of channels each: the weights' sums are joined in shared memory.  A run covers `run` of
// the T + K - 1 rows of w and the tokens of the same numbers; the K - 1 tokens in front of it, whose e its rows' gradients
// need, are computed again.
template <class T, int K, int V, bool SILU>
__global__ __launch_bounds__(256) void conv_backward_kernel(Conv A, int64_t first) {
  __shared__ float sums[3][64][V + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tiles = (A.cols + 63) / 64, block = first + blockIdx.x, tile = block % tiles, rest = block / tiles;
  const int64_t quads = (A.runs + 3) / 4, b = rest / quads, run = rest % quads * 4 + wave;
  const int64_t col = tile * 64 + lane, c = col * V, N = A.T + K - 1;
  const bool here = col < A.cols && run < A.runs;
  float dw[K + 1][V];
#pragma unroll
  for (int j = 0; j <= K; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j][i] = 0.0f;
  if (here) {
    float w[K][V], bias[V], rows[K][V], e[K][V];  // rows t .. t + K - 1 of w; e of tokens t - K + 1 .. t
    const int64_t t0 = run * A.run, t1 = t0 + A.run < N ? t0 + A.run : N, lead = t0 - (K - 1) > 0 ? t0 - (K - 1) : 0;
    const T *x = static_cast<const T*>(A.x) + b * A.xb + c, *dy = static_cast<const T*>(A.dy) + b * A.yb + c;
    constexpr int AHEAD = 4;  // tokens that are on their way while as many are worked on
    Vec<T, V> xs[AHEAD], ds[AHEAD];
    auto fetch = [&](int64_t t) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (A.T == 0) break;
        const int64_t at = t + u < A.T ? t + u : A.T - 1;
        xs[u] = *reinterpret_cast<const Vec<T, V>*>(x + at * A.xt);
        ds[u] = *reinterpret_cast<const Vec<T, V>*>(dy + at * A.yt);
      }
    };
    fetch(lead);
    weights<K, V>(A, c, w, bias);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) e[j][i] = rows[j][i] = 0.0f;
#pragma unroll
    for (int j = 1; j < K; ++j)
      if (lead + j - 1 < N) floats(wide_row<T, K, V>(A, b, lead + j - 1, c), rows[j]);
    for (int64_t first_t = lead; first_t < t1; first_t += AHEAD) {
      Vec<T, V> x_now[AHEAD], d_now[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) x_now[u] = xs[u], d_now[u] = ds[u];
      if (first_t + AHEAD < t1) fetch(first_t + AHEAD);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t t = first_t + u;
        if (t >= t1) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int j = 0; j + 1 < K; ++j) rows[j][i] = rows[j + 1][i], e[j][i] = e[j + 1][i];
          e[K - 1][i] = 0.0f;
        }
        if (t < A.T) {
          float p[V], d[V];
          floats(x_now[u], rows[K - 1]);
          floats(d_now[u], d);
          if (SILU) {
            taps_of<K, V>(w, bias, rows, p);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float s = gate(p[i]);
              d[i] *= s * fmaf(p[i], 1.0f - s, 1.0f);
            }
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            e[K - 1][i] = d[i];
            if (t >= t0) {
#pragma unroll
              for (int j = 0; j < K; ++j) dw[j][i] = fmaf(d[i], rows[j][i], dw[j][i]);
              dw[K][i] += d[i];
            }
          }
        }
        if (t < t0) continue;
        float g[V];
        const bool inner = t >= K - 1 && t < A.T;  // all taps meet tokens
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[i] = 0.0f;
#pragma unroll
          for (int j = 0; j < K; ++j)  // of tokens that exist: a tap may be infinite
            g[i] = inner || (t - j >= 0 && t - j < A.T) ? fmaf(w[j][i], e[K - 1 - j][i], g[i]) : g[i];
        }
        if (t >= A.T && A.dfinal) {
          float f[V];
          get<T, V>(static_cast<const T*>(A.dfinal) + (b * (K - 1) + t - A.T) * A.C + c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] += f[i];
        }
        if (t >= K - 1) {
          if (A.dx) put<T, V>(static_cast<T*>(A.dx) + (b * A.T + t - (K - 1)) * A.C + c, g);
        } else if (A.dstate) {
          put<T, V>(static_cast<T*>(A.dstate) + (b * (K - 1) + t) * A.C + c, g);
        }
      }
    }
  }
  if (A.part == nullptr) return;
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) sums[wave - 1][lane][i] = dw[j][i];
    }
    __syncthreads();
    if (wave == 0 && col < A.cols) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a = dw[j][i];
#pragma unroll
        for (int m = 0; m < 3; ++m) a += sums[m][lane][i];
        A.part[(rest * (K + 1) + j) * A.C + c + i] = a;
      }
    }
    __syncthreads();
  }
}

// The workgroups' sums: a workgroup takes 64 neighbouring entries of [taps + 1, C], its waves every fourth row of parts
__global__ __launch_bounds__(256) void conv_join_kernel(const float* __restrict__ part, int64_t parts, int64_t C, int K,
                                                        bool bf16, void* dweight, void* dbias) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = C * (K + 1), i = (int64_t)blockIdx.x * 64 + lane;
  float a = 0.0f;
  if (i < n)
    for (int64_t p = wave; p < parts; p += 4) a += part[p * n + i];
  sums[wave][lane] = a;
  __syncthreads();
  if (wave > 0 || i >= n) return;
  a = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  const int64_t j = i / C, c = i % C;
  void* to = j == K ? dbias : dweight;
  const int64_t at = j == K ? c : c * K + j;
  if (to == nullptr) return;
  if (bf16) static_cast<__bf16*>(to)[at] = from_f<__bf16>(a);
  else static_cast<float*>(to)[at] = a;
}

// One token: a thread's channels of a row's state, moved on by one.  A state's rows are read before any is written.
template <class T, int K, int V, bool SILU>
__global__ __launch_bounds__(256) void conv_step_kernel(Conv A, const int32_t* __restrict__ slots, int64_t nslots,
                                                        int64_t first, int64_t items) {
  const int64_t item = (first + blockIdx.x) * 256 + threadIdx.x;
  if (item >= items) return;
  const int64_t c = item % A.cols * V, b = item / A.cols, slot = slots ? slots[b] : b;
  T* y = static_cast<T*>(A.y) + b * A.C + c;
  float w[K][V], bias[V], rows[K][V], p[V];
  if (slot < 0 || slot >= nslots) {  // a row without a state
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = 0.0f;
    put<T, V>(y, p);
    return;
  }
  T* state = static_cast<T*>(A.final_state) + slot * (K - 1) * A.C + c;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) get<T, V>(state + j * A.C, rows[j]);
  get<T, V>(static_cast<const T*>(A.x) + b * A.xb + c, rows[K - 1]);
  weights<K, V>(A, c, w, bias);
  taps_of<K, V>(w, bias, rows, p);
  if (SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] *= gate(p[i]);
  }
  put<T, V>(y, p);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) put<T, V>(state + j * A.C, rows[j + 1]);
}

// ---- host ----------------------------------------------------------------------------------------------------

// f(tap count as a constant)
template <class F>
int with_taps(int64_t taps, F f) {
  switch (taps) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}

inline int conv_check(int64_t dtype, int64_t weight_dtype, std::initializer_list<int64_t> sizes, int64_t taps,
                      int64_t activation) {
  for (int64_t v : sizes)
    if (v < 0) return TTC_LQR_EINVAL;
  if (taps < 1 || taps > MAX_TAPS || activation < 0 || activation > 1 || !countable(sizes)) return TTC_LQR_EINVAL;
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16) return TTC_LQR_EUNSUPPORTED;
  if (weight_dtype != TTC_DTYPE_F32 && weight_dtype != dtype) return TTC_LQR_EUNSUPPORTED;
  return TTC_LQR_OK;
}

constexpr int64_t MAX_CHANNELS = 1 << 26;  // the sums' join is one launch

inline int conv_check(const ttc_causal_conv_args& A) {
  if (A.tokens < 0 || A.tokens > ((int64_t)1 << 58) || A.channels > MAX_CHANNELS) return TTC_LQR_EINVAL;
  return conv_check(A.dtype, A.weight_dtype, {A.batch, A.tokens + MAX_TAPS, A.channels, MAX_TAPS + 1}, A.taps, A.activation);
}

// Rows of w a thread walks along backwards: as many as let all workgroups run at once (three a CU, of four runs each), since the
// K - 1 tokens in front of a run are computed again; 8 at least, 128 at most.  us by run:
//                                               8     12     16     24     32     48     64     96    128
//   4 x 2,048 tokens x 4,096 channels, bf16    84     74     70     68     73     63     78     91    115
//   16,384 x 2,048                             82     74     69     68     69     63     68     91    103
//   2,048 x 1,024                              14     16     19     24     29     40     51     73     95
//   8 x 4,096 x 4,096, fp32                   495    457    430    399    393    386    360    372    354
inline int64_t backward_run(const ttc_causal_conv_args& A, int64_t cols) {
  const int64_t tiles = ceil_div(cols, 64) * (A.batch > 0 ? A.batch : 1), N = A.tokens + A.taps - 1;
  const int64_t run = ceil_div(N * tiles, 3 * 256 * 4);
  return run < 8 ? 8 : run > 128 ? 128 : run;
}

// Channels a thread, where sizes, strides and addresses allow: 8 bytes in 16 bits, 16 in 32.  With 8 channels taps, rows and
// sums leave two waves a SIMD (prompt of 16,381 tokens x 6,144 channels in bf16: 136 us, with four 75)
constexpr int VECTOR = 4;

template <class T>
bool conv_wide(const ttc_causal_conv_args& A) {
  auto ok = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (VECTOR * sizeof(T)) == 0; };
  bool wide = A.channels % VECTOR == 0 && A.x_stride[0] % VECTOR == 0 && A.x_stride[1] % VECTOR == 0 && ok(A.x) && ok(A.y) &&
              ok(A.initial_state) && ok(A.final_state);
  if (A.backward)
    wide = wide && A.d_y_stride[0] % VECTOR == 0 && A.d_y_stride[1] % VECTOR == 0 && ok(A.d_y) && ok(A.dx) &&
           ok(A.d_final_state) && ok(A.d_initial_state);
  return wide;
}

// Sums of the weights' gradients: one row of them for each four runs of a sequence.  Of the block alone, whatever its
// pointers: with vectors of channels they are fewer.
inline int64_t conv_parts(const ttc_causal_conv_args& A, int64_t cols) {
  return A.batch * ceil_div(ceil_div(A.tokens + A.taps - 1, backward_run(A, cols)), 4);
}

inline int64_t conv_bytes(const ttc_causal_conv_args& A) {
  if (!A.backward || (!A.dweight && !A.dbias)) return 0;
  const int64_t a = conv_parts(A, ceil_div(A.channels, VECTOR)), b = conv_parts(A, A.channels);
  return (a > b ? a : b) * (A.taps + 1) * A.channels * 4;
}

template <class T, int V>
int conv_run(const ttc_causal_conv_args& A, hipStream_t s) {
  Conv P{};
  P.x = A.x, P.weight = A.weight, P.bias = A.bias, P.state = A.initial_state;
  P.xb = A.x_stride[0], P.xt = A.x_stride[1];
  P.B = A.batch, P.T = A.tokens, P.C = A.channels;
  P.weight_bf16 = A.weight_dtype == TTC_DTYPE_BF16, P.wide_weight = aligned16(A.weight);
  P.cols = A.channels / V;
  if (!A.backward) {
    P.y = A.y, P.final_state = A.final_state;
    P.runs = A.tokens > 0 ? ceil_div(A.tokens, FORWARD_RUN) : 1;
    const int64_t items = A.batch * P.runs * P.cols;
    return with_taps(A.taps, [&](auto taps) {
      constexpr int K = decltype(taps)::value;
      return in_launches(ceil_div(items, 256), 256, [&](int64_t first, dim3 grid) {
        if (A.activation) hipLaunchKernelGGL((conv_kernel<T, K, V, true>), grid, dim3(256), 0, s, P, first, items);
        else hipLaunchKernelGGL((conv_kernel<T, K, V, false>), grid, dim3(256), 0, s, P, first, items);
      });
    });
  }
  P.dy = A.d_y, P.dfinal = A.d_final_state;
  P.yb = A.d_y_stride[0], P.yt = A.d_y_stride[1];
  P.dx = A.dx, P.dstate = A.d_initial_state;
  P.part = A.dweight || A.dbias ? static_cast<float*>(A.workspace) : nullptr;
  P.run = backward_run(A, P.cols);
  P.runs = ceil_div(A.tokens + A.taps - 1, P.run);
  const int64_t parts = conv_parts(A, P.cols);
  const int rc = with_taps(A.taps, [&](auto taps) {
    constexpr int K = decltype(taps)::value;
    return in_launches(parts * ceil_div(P.cols, 64), 256, [&](int64_t first, dim3 grid) {
      if (A.activation) hipLaunchKernelGGL((conv_backward_kernel<T, K, V, true>), grid, dim3(256), 0, s, P, first);
      else hipLaunchKernelGGL((conv_backward_kernel<T, K, V, false>), grid, dim3(256), 0, s, P, first);
    });
  });
  if (rc || (!A.dweight && !A.dbias)) return rc;
  // of no parts, where there are no sequences or no rows: sums of nothing
  hipLaunchKernelGGL(conv_join_kernel, dim3((unsigned)ceil_div(A.channels * (A.taps + 1), 64)), dim3(256), 0, s, P.part, parts,
                     A.channels, (int)A.taps, P.weight_bf16, A.dweight, A.dbias);
  return launched();
}

template <class T>
int conv_typed(const ttc_causal_conv_args& A, hipStream_t s) {
  return conv_wide<T>(A) ? conv_run<T, VECTOR>(A, s) : conv_run<T, 1>(A, s);
}

template <class T, int V>
int conv_step_run(const ttc_causal_conv_step_args& A, hipStream_t s) {
  Conv P{};
  P.x = A.x, P.weight = A.weight, P.bias = A.bias;
  P.xb = A.x_stride;
  P.C = A.channels;
  P.weight_bf16 = A.weight_dtype == TTC_DTYPE_BF16, P.wide_weight = aligned16(A.weight);
  P.y = A.y, P.final_state = A.state;
  P.cols = A.channels / V;
  const int64_t items = A.batch * P.cols;
  return with_taps(A.taps, [&](auto taps) {
    constexpr int K = decltype(taps)::value;
    return in_launches(ceil_div(items, 256), 256, [&](int64_t first, dim3 grid) {
      if (A.activation)
        hipLaunchKernelGGL((conv_step_kernel<T, K, V, true>), grid, dim3(256), 0, s, P, A.slot_index, A.slots, first, items);
      else
        hipLaunchKernelGGL((conv_step_kernel<T, K, V, false>), grid, dim3(256), 0, s, P, A.slot_index, A.slots, first, items);
    });
  });
}

template <class T>
int conv_step_typed(const ttc_causal_conv_step_args& A, hipStream_t s) {
  auto ok = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (VECTOR * sizeof(T)) == 0; };
  const bool wide = A.channels % VECTOR == 0 && A.x_stride % VECTOR == 0 && ok(A.x) && ok(A.y) && ok(A.state);
  return wide ? conv_step_run<T, VECTOR>(A, s) : conv_step_run<T, 1>(A, s);
}

}  // namespace ttc

extern "C" size_t ttc_causal_conv_workspace_bytes(const ttc_causal_conv_args* args) {
  using namespace ttc;
  if (!args || conv_check(*args) != TTC_LQR_OK) return 0;
  return (size_t)conv_bytes(*args);
}

extern "C" int ttc_causal_conv(const ttc_causal_conv_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_causal_conv_args& A = *args;
  if (const int rc = conv_check(A)) return rc;
  if (A.channels == 0 || (!A.backward && (A.batch == 0 || A.tokens + A.taps == 1))) return TTC_LQR_OK;
  const bool some = A.batch > 0 && A.tokens > 0;
  if (!A.weight || (some && (!A.x || (A.backward ? !A.d_y : !A.y)))) return TTC_LQR_EINVAL;
  const int64_t bytes = conv_bytes(A);
  if (bytes > 0 && (!A.workspace || A.workspace_bytes < bytes)) return TTC_LQR_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return A.dtype == TTC_DTYPE_F32 ? conv_typed<float>(A, s) : conv_typed<__bf16>(A, s);
}

extern "C" int ttc_causal_conv_step(const ttc_causal_conv_step_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_causal_conv_step_args& A = *args;
  if (const int rc = conv_check(A.dtype, A.weight_dtype, {A.batch, A.channels, MAX_TAPS}, A.taps, A.activation)) return rc;
  if (A.slots < 0 || !countable({A.slots, A.channels, MAX_TAPS}) || (!A.slot_index && A.slots != A.batch))
    return TTC_LQR_EINVAL;
  if (A.batch == 0 || A.channels == 0) return TTC_LQR_OK;
  if (!A.x || !A.weight || !A.y || (A.slots > 0 && A.taps > 1 && !A.state)) return TTC_LQR_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return A.dtype == TTC_DTYPE_F32 ? conv_step_typed<float>(A, s) : conv_step_typed<__bf16>(A, s);
}
