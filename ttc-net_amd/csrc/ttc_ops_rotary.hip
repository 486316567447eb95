// ttc_ops_rotary.hip -- rotary positions of queries and keys in one launch, forward and backward.
//
// A pair (x_a, x_b) of a head turns by its token's angle: (x_a c - x_b s, x_a s + x_b c); the gradient turns
// back (s negated), so both directions are one kernel.  Cosines and sines come from a table in fp32, because an
// angle of 10^5 radians held in fp32 is itself off by 4e-3.
//
// Bound: memory (each element read and written once, 3 flops an element).  16,381 tokens x (16 + 16) heads of 128 in bf16:
// 47 us for 277 MB, 5.9 TB/s (a copy of 1 GiB: 5.2); one token of 16 sequences: 4.0 us.
#include "ttc_ops_common.hpp"

namespace ttc {

struct RotaryShape {
  int64_t T, length, first;
  int64_t pos_b, pos_t, xs[2][3];
  int H0, H1, dim, half, cols, groups;  // cols: vectors of a head, groups: head groups of a token
  float sign;
};

__device__ __forceinline__ int64_t position_of(const void* pos, int bytes, const RotaryShape& S, int64_t b, int64_t t) {
  if (pos == nullptr) return S.first + t;
  const int64_t i = b * S.pos_b + t * S.pos_t;
  return bytes == 8 ? static_cast<const int64_t*>(pos)[i] : static_cast<const int32_t*>(pos)[i];
}

// One thread: one vector column of one token, HEADS heads of it.  V elements a vector (1 where sizes or
// addresses do not allow 16 bytes).  Half layout: columns [0, half / V) are the pairs (column and its partner half
// a rotation on); interleaved: columns [0, 2 half / V) hold whole pairs, or with V = 1 one pair each.  The columns
// after them are copied.
template <class T, int V, bool INTER, int HEADS>
__global__ __launch_bounds__(256) void rotary_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                     T* __restrict__ yq, T* __restrict__ yk,
                                                     const float* __restrict__ table, const void* __restrict__ pos,
                                                     int pos_bytes, RotaryShape S, int64_t first, int64_t items) {
  const int64_t item = (first + blockIdx.x) * 256 + threadIdx.x;
  if (item >= items) return;
  const int col = (int)(item % S.cols);
  const int64_t rest = item / S.cols;
  const int grp = (int)(rest % S.groups);
  const int64_t token = rest / S.groups, b = token / S.T, t = token % S.T;
  const int heads = S.H0 + S.H1, h0 = grp * HEADS;

  constexpr int W = INTER && V == 1 ? 2 : V;             // elements a pair column spans from its start
  const int pair_cols = INTER ? 2 * S.half / W : S.half / V;
  const bool turn = col < pair_cols;
  const int at = turn ? col * W : 2 * S.half + (col - pair_cols) * V;  // its first element
  constexpr int PAIRS = INTER ? W / 2 : V;
  float c[PAIRS], s[PAIRS];
  if (turn) {
    const int64_t p = position_of(pos, pos_bytes, S, b, t);
    const int pair = INTER ? at / 2 : at;
    const bool in = p >= 0 && p < S.length;
    const float* row = table + ((in ? p : 0) * S.half + pair) * 2;
    float cs[2 * PAIRS];
    if constexpr (V == 1) {
      cs[0] = row[0], cs[1] = row[1];
    } else {
#pragma unroll
      for (int i = 0; i < PAIRS / 2; ++i) {
        const float4 two = reinterpret_cast<const float4*>(row)[i];
        cs[4 * i] = two.x, cs[4 * i + 1] = two.y, cs[4 * i + 2] = two.z, cs[4 * i + 3] = two.w;
      }
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      c[i] = in ? cs[2 * i] : __builtin_nanf("");
      s[i] = in ? cs[2 * i + 1] * S.sign : __builtin_nanf("");
    }
  }
  struct alignas(V * sizeof(T)) Vec { T v[V]; };
  Vec a[HEADS], z[HEADS];  // INTER with V = 1: the pair's two elements in a and z
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    const bool key = h >= S.H0;
    const T* x = (key ? k : q) + b * S.xs[key][0] + t * S.xs[key][1] + (key ? h - S.H0 : h) * S.xs[key][2] + at;
    a[i] = *reinterpret_cast<const Vec*>(x);
    if (turn && (!INTER || V == 1)) z[i] = *reinterpret_cast<const Vec*>(x + (INTER ? 1 : S.half));
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    const bool key = h >= S.H0;
    T* y = (key ? yk : yq) + (token * (key ? S.H1 : S.H0) + (key ? h - S.H0 : h)) * S.dim + at;
    if (turn) {
      if constexpr (INTER && V > 1) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
          const float u = to_f(a[i].v[2 * j]), w = to_f(a[i].v[2 * j + 1]);
          a[i].v[2 * j] = from_f<T>(u * c[j] - w * s[j]);
          a[i].v[2 * j + 1] = from_f<T>(u * s[j] + w * c[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float u = to_f(a[i].v[j]), w = to_f(z[i].v[j]);
          a[i].v[j] = from_f<T>(u * c[j] - w * s[j]);
          z[i].v[j] = from_f<T>(u * s[j] + w * c[j]);
        }
        *reinterpret_cast<Vec*>(y + (INTER ? 1 : S.half)) = z[i];
      }
    }
    *reinterpret_cast<Vec*>(y) = a[i];
  }
}

template <class T, int V>
int rotary_launch(const ttc_rotary_args& A, RotaryShape& S, hipStream_t s) {
  const bool inter = A.interleaved != 0;
  const int w = inter && V == 1 ? 2 : V;
  S.cols = (int)((inter ? 2 * S.half / w : S.half / V) + (S.dim - 2 * S.half) / V);
  // heads a thread: 4 share one read of the table (4,096 tokens x 40 heads of 128: 14.4 us, with one 15.7); a call too small
  // to fill the GPU takes one, for the shorter chain (10 heads: 3.5 us, with four 3.7)
  const int64_t tokens = A.batch * A.tokens, heads = S.H0 + S.H1;
  const int per = tokens * heads * S.cols >= (int64_t)4 * 256 * 1024 ? 4 : 1;
  S.groups = (int)ceil_div(heads, per);
  const int64_t items = tokens * S.groups * S.cols;
  auto go = [&](auto kernel) {
    return in_launches(ceil_div(items, 256), 256, [&](int64_t first, dim3 grid) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const T*>(A.x[0]), static_cast<const T*>(A.x[1]),
                         static_cast<T*>(A.y[0]), static_cast<T*>(A.y[1]), A.table, A.positions, (int)A.position_bytes,
                         S, first, items);
    });
  };
  if (inter) return per == 4 ? go(rotary_kernel<T, V, true, 4>) : go(rotary_kernel<T, V, true, 1>);
  return per == 4 ? go(rotary_kernel<T, V, false, 4>) : go(rotary_kernel<T, V, false, 1>);
}

template <class T>
int rotary_typed(const ttc_rotary_args& A, RotaryShape& S, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  bool wide = S.dim % V == 0 && (A.interleaved ? 2 * S.half : S.half) % V == 0 && aligned16(A.table);
  for (int i = 0; i < 2; ++i) {
    if (A.heads[i] == 0) continue;
    wide = wide && aligned16(A.x[i]) && aligned16(A.y[i]);
    for (int j = 0; j < 3; ++j) wide = wide && A.stride[i][j] % V == 0;
  }
  return wide ? rotary_launch<T, V>(A, S, s) : rotary_launch<T, 1>(A, S, s);
}

}  // namespace ttc

extern "C" int ttc_rotary(const ttc_rotary_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_rotary_args& A = *args;
  const int64_t lim = 1 << 24;  // heads and head sizes are held in 32 bits
  if (A.batch < 0 || A.tokens < 0 || A.heads[0] < 0 || A.heads[1] < 0 || A.heads[0] > lim || A.heads[1] > lim ||
      A.dim < 0 || A.dim > lim || A.rot < 0 || A.rot > A.dim || A.rot % 2 || A.length < 0 ||
      !countable({A.batch, A.tokens, A.heads[0] + A.heads[1], A.dim}) || !countable({A.length, A.rot}))
    return TTC_LQR_EINVAL;
  if (A.dtype != TTC_DTYPE_F32 && A.dtype != TTC_DTYPE_BF16) return TTC_LQR_EUNSUPPORTED;
  if (A.batch == 0 || A.tokens == 0 || A.heads[0] + A.heads[1] == 0 || A.dim == 0) return TTC_LQR_OK;
  for (int i = 0; i < 2; ++i)
    if (A.heads[i] > 0 && (!A.x[i] || !A.y[i])) return TTC_LQR_EINVAL;
  if (A.rot > 0 && A.length > 0 && !A.table) return TTC_LQR_EINVAL;
  if (A.rot > 0 && A.length == 0) return TTC_LQR_EINVAL;
  if (A.positions && A.position_bytes != 4 && A.position_bytes != 8) return TTC_LQR_EINVAL;
  RotaryShape S;
  S.T = A.tokens;
  S.length = A.length;
  S.first = A.first;
  S.pos_b = A.position_stride[0];
  S.pos_t = A.position_stride[1];
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) S.xs[i][j] = A.stride[i][j];
  S.H0 = (int)A.heads[0];
  S.H1 = (int)A.heads[1];
  S.dim = (int)A.dim;
  S.half = (int)(A.rot / 2);
  S.sign = A.backward ? -1.0f : 1.0f;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return A.dtype == TTC_DTYPE_F32 ? rotary_typed<float>(A, S, s) : rotary_typed<__bf16>(A, S, s);
}
