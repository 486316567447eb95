// ttc_ops_norm.hip -- group norm with an activation or a gate over channels-last data, forward and backward.
//
//   y0 = (x - mean) rstd w + b over the l positions and the c / G channels of a group;
//   y = act(y0), or y0 act(gate)
//   backward, with dy0 = dy act'(y0) or dy act(gate):  dxhat = dy0 w,
//   dx = rstd (dxhat - mean(dxhat) - xhat mean(dxhat xhat)),  dw = sum dy0 xhat,  db = sum dy0,
//   dgate = dy y0 act'(gate).
//
// Bound: memory.  Three forms:
//  * one position (l = 1: a norm over each head of a token): a group is contiguous, up to 64 lanes hold it in
//    registers (up to 4 vectors of 16 bytes each), so x is read once and the variance is that of the centred values.
//    8,192 x 2,048 in 32 groups, gated, bf16: forward 30 us (100 MB, 3.4 TB/s), backward 39 us (168 MB, 4.3 TB/s) and
//    8 us for the sums of the weights' gradients; 16 x 2,048: 4.2 us;
//  * a group that fits in a workgroup's registers, forward: up to 64 lanes or one workgroup a group, x read once.
//    2 x 1,021 x 192 in 6 groups, bf16: 12 us, most of it latency (slabs 16 in three launches);
//  * any other, and every backward over several positions: slabs of positions, each reduced over whole rows of c
//    channels (coalesced); sums per channel are taken about the slab's first position (a large common mean costs no
//    digits) and joined as (mean, sum of squares) pairs; a second pass reads x again and writes y.  8 x 4,096 x 320 in 32
//    groups, fp32 (42 MB an array): forward 14 + 5 + 17 us (statistics, join, output), backward 18 + 5 + 21 + 5 us; the
//    caches hold x between the passes.  7,269 x 768 in 12 groups, bf16 (11 MB): forward 7 + 6 + 10 us.
#include "ttc_ops_common.hpp"

namespace ttc {

struct Affine {  // weight and bias of type float or bf16, or none
  const void *w, *b;
  bool bf16, wide;  // wide: at 16-byte addresses
  // V of each from channel c (a multiple of V) on, 1 and 0 beyond `end`
  template <int V>
  __device__ __forceinline__ void load(int64_t c, int64_t end, float (&wv)[V], float (&bv)[V]) const {
    if (V > 1 && wide && w != nullptr && c + V <= end) {
      auto vec = [&](const void* p, float (&out)[V]) {
        if (bf16) {
          struct alignas(V * 2) Values { __bf16 v[V]; };
          const Values r = *reinterpret_cast<const Values*>(static_cast<const __bf16*>(p) + c);
#pragma unroll
          for (int j = 0; j < V; ++j) out[j] = to_f(r.v[j]);
        } else {
          struct alignas(V * 4 < 16 ? V * 4 : 16) Values { float v[V]; };
          const Values r = *reinterpret_cast<const Values*>(static_cast<const float*>(p) + c);
#pragma unroll
          for (int j = 0; j < V; ++j) out[j] = r.v[j];
        }
      };
      vec(w, wv);
      vec(b, bv);
      return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wv[j] = c + j < end ? weight(c + j) : 1.0f;
      bv[j] = c + j < end ? bias(c + j) : 0.0f;
    }
  }
  __device__ __forceinline__ float weight(int64_t c) const {
    if (w == nullptr) return 1.0f;
    return bf16 ? to_f(static_cast<const __bf16*>(w)[c]) : static_cast<const float*>(w)[c];
  }
  __device__ __forceinline__ float bias(int64_t c) const {
    if (b == nullptr) return 0.0f;
    return bf16 ? to_f(static_cast<const __bf16*>(b)[c]) : static_cast<const float*>(b)[c];
  }
};

// act(z) and its slope
template <bool SILU>
__device__ __forceinline__ float act(float z) {
  return SILU ? z * sigmoid(z) : z;
}
template <bool SILU>
__device__ __forceinline__ void act_slope(float z, float& on, float& slope) {
  if (SILU) {
    const float s = sigmoid(z);
    on = z * s;
    slope = s * (1.0f + z * (1.0f - s));
  } else {
    on = z;
    slope = 1.0f;
  }
}

template <bool SILU, bool GATE>
__device__ __forceinline__ float out_of(float y0, float gate) {
  return GATE ? y0 * act<SILU>(gate) : act<SILU>(y0);
}
// gradient of y0 and of the gate
template <bool SILU, bool GATE>
__device__ __forceinline__ float back_of(float dy, float y0, float gate, float& dgate) {
  float on, slope;
  act_slope<SILU>(GATE ? gate : y0, on, slope);
  dgate = GATE ? dy * y0 * slope : 0.0f;
  return GATE ? dy * on : dy * slope;
}

template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

// ---- one position: rows of `cg` contiguous channels ---------------------------------------------------------

// How the rows' kernels spread: `lanes` (a power of two) lanes a group, NV vectors of V elements each.  A thread keeps its
// channels (group, lane) and walks down a slab of the n rows, so that weights stay in registers and the backward's sums over
// n do; a workgroup covers 256 / lanes groups of a row of G, or several rows at once where G is smaller.
struct Rows {
  int64_t n;
  int G, cg, lanes, gper, rper, gblocks, slab;  // gper groups and rper rows at once, slab rows in all
};

template <class T, int V, int NV, bool SILU, bool GATE>
__global__ __launch_bounds__(256) void norm_row_kernel(const T* __restrict__ x, const T* __restrict__ gate, Affine aff,
                                                       Rows R, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                                                       float* __restrict__ rstd_out) {
  const int lanes = R.lanes, cg = R.cg, lane = threadIdx.x % lanes, unit = threadIdx.x / lanes;
  const int gb = blockIdx.x % R.gblocks;
  const int64_t sl = blockIdx.x / R.gblocks;
  const int r = unit / R.gper, g = gb * R.gper + unit % R.gper;
  if (r >= R.rper || g >= R.G) return;  // no barrier follows; a group's lanes leave together
  const int64_t n1 = (sl + 1) * R.slab < R.n ? (sl + 1) * R.slab : R.n;
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * lanes + lane) * V;
    aff.load<V>((int64_t)g * cg + c, (int64_t)g * cg + (c < cg ? cg : c), w[i], b[i]);
  }
  const float inv = 1.0f / cg;
  Vec<T, V> xn[NV], gn[NV];  // the next row's, on their way
  auto fetch = [&](int64_t m) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * V;
      if (c < cg) {
        xn[i] = *reinterpret_cast<const Vec<T, V>*>(x + (m * R.G + g) * cg + c);
        if (GATE) gn[i] = *reinterpret_cast<const Vec<T, V>*>(gate + (m * R.G + g) * cg + c);
      }
    }
  };
  const int64_t m0 = sl * R.slab + r;
  if (m0 < n1) fetch(m0);
  for (int64_t m = m0; m < n1; m += R.rper) {
    Vec<T, V> xv[NV], gv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) xv[i] = xn[i], gv[i] = gn[i];
    if (m + R.rper < n1) fetch(m + R.rper);
    const int64_t row = m * R.G + g, base = row * cg;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * lanes + lane) * V < cg) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum += to_f(xv[i].v[j]);
      }
    const float mean = lane_sum(sum, lanes) * inv;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * lanes + lane) * V < cg) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = to_f(xv[i].v[j]) - mean;
          sq = fmaf(d, d, sq);
        }
      }
    const float rstd = 1.0f / sqrtf(lane_sum(sq, lanes) * inv + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * V;
      if (c >= cg) break;
      Vec<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float y0 = fmaf((to_f(xv[i].v[j]) - mean) * rstd, w[i][j], b[i][j]);
        out.v[j] = from_f<T>(out_of<SILU, GATE>(y0, GATE ? to_f(gv[i].v[j]) : 0.0f));
      }
      *reinterpret_cast<Vec<T, V>*>(y + base + c) = out;
    }
    if (lane == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// partial: [parts, 2, c] fp32, the sums over each thread row's part of the n rows
template <class T, int V, int NV, bool SILU, bool GATE>
__global__ __launch_bounds__(256) void norm_row_backward_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                                const T* __restrict__ dy, Affine aff, Rows R,
                                                                const float* __restrict__ mean_in,
                                                                const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                                T* __restrict__ dgate, float* __restrict__ partial) {
  const int lanes = R.lanes, cg = R.cg, G = R.G, rper = R.rper, lane = threadIdx.x % lanes, unit = threadIdx.x / lanes;
  const int gb = blockIdx.x % R.gblocks;
  const int64_t sl = blockIdx.x / R.gblocks;
  const int r = unit / R.gper, g = gb * R.gper + unit % R.gper;
  if (r >= rper || g >= G) return;  // no barrier follows; a group's lanes leave together
  const int64_t n0 = sl * R.slab, n1 = n0 + R.slab < R.n ? n0 + R.slab : R.n;
  float w[NV][V], b[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * lanes + lane) * V;
    aff.load<V>((int64_t)g * cg + c, (int64_t)g * cg + (c < cg ? cg : c), w[i], b[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  Vec<T, V> xn[NV], dn[NV], gn[NV];  // the next row's, on their way
  float mean_n = 0.0f, rstd_n = 0.0f;
  auto fetch = [&](int64_t m) {
    const int64_t row = m * G + g;
    mean_n = mean_in[row];
    rstd_n = rstd_in[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * V;
      if (c < cg) {
        xn[i] = *reinterpret_cast<const Vec<T, V>*>(x + row * cg + c);
        dn[i] = *reinterpret_cast<const Vec<T, V>*>(dy + row * cg + c);
        if (GATE) gn[i] = *reinterpret_cast<const Vec<T, V>*>(gate + row * cg + c);
      }
    }
  };
  if (n0 + r < n1) fetch(n0 + r);
  const float inv = 1.0f / cg;
  for (int64_t m = n0 + r; m < n1; m += rper) {
    const int64_t row = m * G + g, base = row * cg;
    const float mean = mean_n, rstd = rstd_n;
    float xh[NV][V], dh[NV][V], s1 = 0.0f, s2 = 0.0f;
    Vec<T, V> xv[NV], dv[NV], gv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) xv[i] = xn[i], dv[i] = dn[i], gv[i] = gn[i];
    if (m + rper < n1) fetch(m + rper);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * V;
      if (c < cg) {
        Vec<T, V> dg;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          xh[i][j] = (to_f(xv[i].v[j]) - mean) * rstd;
          float dgj;
          const float d0 = back_of<SILU, GATE>(to_f(dv[i].v[j]), fmaf(xh[i][j], w[i][j], b[i][j]),
                                               GATE ? to_f(gv[i].v[j]) : 0.0f, dgj);
          dg.v[j] = from_f<T>(dgj);
          dw[i][j] = fmaf(d0, xh[i][j], dw[i][j]);
          db[i][j] += d0;
          dh[i][j] = d0 * w[i][j];
          s1 += dh[i][j];
          s2 = fmaf(dh[i][j], xh[i][j], s2);
        }
        if (GATE && dgate) *reinterpret_cast<Vec<T, V>*>(dgate + base + c) = dg;
      }
    }
    s1 = lane_sum(s1, lanes) * inv;
    s2 = lane_sum(s2, lanes) * inv;
    if (dx) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + lane) * V;
        if (c < cg) {
          Vec<T, V> out;
#pragma unroll
          for (int j = 0; j < V; ++j) out.v[j] = from_f<T>(rstd * (dh[i][j] - s1 - xh[i][j] * s2));
          *reinterpret_cast<Vec<T, V>*>(dx + base + c) = out;
        }
      }
    }
  }
  if (partial) {
    float* p = partial + (sl * rper + r) * 2 * (int64_t)G * cg + g * cg;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (i * lanes + lane) * V + j;
        if (c < cg) {
          p[c] = dw[i][j];
          p[(int64_t)G * cg + c] = db[i][j];
        }
      }
  }
}

// Sums of [parts, 2, c] over the parts, in 64 bits: 16 channels a workgroup, 64 threads each
template <class W>
__global__ __launch_bounds__(1024) void norm_affine_sum_kernel(const float* __restrict__ partial, int64_t parts, int64_t c,
                                                               W* __restrict__ dw, W* __restrict__ db) {
  __shared__ double sw[64][17], sb[64][17];
  const int cx = threadIdx.x % 16, py = threadIdx.x / 16;
  const int64_t ch = (int64_t)blockIdx.x * 16 + cx;
  double w = 0.0, b = 0.0;
  if (ch < c)
#pragma unroll 4
    for (int64_t p = py; p < parts; p += 64) {
      w += partial[p * 2 * c + ch];
      b += partial[(p * 2 + 1) * c + ch];
    }
  sw[py][cx] = w;
  sb[py][cx] = b;
  for (int m = 32; m >= 1; m >>= 1) {
    __syncthreads();
    if (py < m) {
      sw[py][cx] += sw[py + m][cx];
      sb[py][cx] += sb[py + m][cx];
    }
  }
  if (py == 0 && ch < c) {
    if (dw) dw[ch] = from_f<W>((float)sw[0][cx]);
    if (db) db[ch] = from_f<W>((float)sb[0][cx]);
  }
}

// ---- any number of positions ---------------------------------------------------------------------------------

// Slab kernels: a workgroup reads `slab` positions of one n, all channels in blocks of 256 / rper vectors; thread
// (r, column) walks down positions r, r + rper, ...
struct Slab {
  int64_t L, slab, slabs, first;  // first: workgroup of this launch
  int C, G, cg, cols, rper, cblocks;  // cols: vectors of a row
  int per;  // channels of a forward's partial: a vector's where none reaches into two groups
};

// Groups that fit in registers, forward: x read once, one launch instead of three.  The group's l rows of cg channels are
// counted in vectors; thread t of its `team` holds vectors t, t + team, ...  A team is a workgroup, or up to 64 lanes of a
// workgroup of 256 that holds several groups (NV = 2): 38,176 groups of 5 x 8 in bf16 7 us, a workgroup each 150.
constexpr int WHOLE = 8, SMALL = 2;  // vectors a thread
template <class T, int V, bool SILU, bool GATE, int NV>
__global__ __launch_bounds__(1024) void norm_whole_kernel(const T* __restrict__ x, const T* __restrict__ gate, Affine aff,
                                                          Slab S, int team, int64_t groups, float eps, T* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float part[16];
  const int t = (int)threadIdx.x % team;
  const int64_t mine = (S.first + blockIdx.x) * ((int)blockDim.x / team) + (int)threadIdx.x / team;
  const bool live = mine < groups;  // the others repeat the last group and write nothing
  const int64_t ng = live ? mine : groups - 1, n = ng / S.G;
  const int g = (int)(ng % S.G), cols = S.cg / V;
  const int vecs = (int)S.L * cols;
  const T *xg = x + n * S.L * S.C + g * S.cg, *gg = GATE ? gate + n * S.L * S.C + g * S.cg : nullptr;
  T* yg = y + n * S.L * S.C + g * S.cg;
  auto sum = [&](float v) {
    v = lane_sum(v, NV == SMALL ? team : 64);
    if (NV == SMALL) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = 0.0f;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) r += part[i];
    return r;
  };
  Vec<T, V> xv[NV];
  int64_t at[NV];
  float a = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {  // loads from the last vector where there is none: in branches each would wait
    const int i = t + k * team, j = i < vecs ? i : vecs - 1;
    at[k] = (int64_t)(j / cols) * S.C + j % cols * V;
    xv[k] = *reinterpret_cast<const Vec<T, V>*>(xg + at[k]);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) a += t + k * team < vecs ? to_f(xv[k].v[j]) : 0.0f;
  const float total = (float)S.L * S.cg, mean = sum(a) / total;
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = to_f(xv[k].v[j]) - mean;
      q = t + k * team < vecs ? fmaf(d, d, q) : q;
    }
  const float rstd = 1.0f / sqrtf(sum(q) / total + eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = t + k * team;
    if (i >= vecs || !live) break;
    float w[V], b[V];
    const int64_t c = (int64_t)g * S.cg + i % cols * V;
    aff.load<V>(c, S.C, w, b);
    Vec<T, V> gt, out;
    if (GATE) gt = *reinterpret_cast<const Vec<T, V>*>(gg + at[k]);
#pragma unroll
    for (int j = 0; j < V; ++j)
      out.v[j] = from_f<T>(
          out_of<SILU, GATE>(fmaf((to_f(xv[k].v[j]) - mean) * rstd, w[j], b[j]), GATE ? to_f(gt.v[j]) : 0.0f));
    *reinterpret_cast<Vec<T, V>*>(yg + at[k]) = out;
  }
  if (t == 0 && live && mean_out) {
    mean_out[ng] = mean;
    rstd_out[ng] = rstd;
  }
}

// (mean, M2) of `count` values per (n, slab, channel or vector of a group) -> partial [n, slabs, 2, c / per]
template <class T, int V>
__global__ __launch_bounds__(256) void norm_slab_stats_kernel(const T* __restrict__ x, Slab S,
                                                              float* __restrict__ partial) {
  __shared__ float s1[256 * V], s2[256 * V];
  const int cper = 256 / S.rper;
  const int r = threadIdx.x / cper, cc = threadIdx.x % cper;
  int64_t blk = S.first + blockIdx.x;
  const int cb = (int)(blk % S.cblocks);
  blk /= S.cblocks;
  const int64_t sl = blk % S.slabs, n = blk / S.slabs;
  const int col = cb * cper + cc;
  const bool live = r < S.rper && col < S.cols;
  const int64_t l0 = sl * S.slab, l1 = l0 + S.slab < S.L ? l0 + S.slab : S.L;
  float a[V], q[V], k[V];
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = q[j] = k[j] = 0.0f;
  if (live) {
    const T* p = x + n * S.L * S.C + (int64_t)col * V;
    const Vec<T, V> first = *reinterpret_cast<const Vec<T, V>*>(p + l0 * S.C);
#pragma unroll
    for (int j = 0; j < V; ++j) k[j] = to_f(first.v[j]);
#pragma unroll 4
    for (int64_t l = l0 + r; l < l1; l += S.rper) {
      const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p + l * S.C);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f(v.v[j]) - k[j];
        a[j] += d;
        q[j] = fmaf(d, d, q[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s1[j * 256 + threadIdx.x] = a[j];
    s2[j * 256 + threadIdx.x] = q[j];
  }
  __syncthreads();
  if (r == 0 && col < S.cols) {
    const float cnt = (float)(l1 - l0);
    const int row = S.C / S.per;
    float* out = partial + ((n * S.slabs + sl) * 2) * row + (S.per > 1 ? (int64_t)col : (int64_t)col * V);
    float mean = 0.0f, m2 = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int i = 1; i < S.rper; ++i) {
        a[j] += s1[j * 256 + i * cper + cc];
        q[j] += s2[j * 256 + i * cper + cc];
      }
      q[j] = fmaxf(q[j] - a[j] * (a[j] / cnt), 0.0f);
      a[j] = k[j] + a[j] / cnt;
      mean += (a[j] - a[0]) * (1.0f / V);
    }
    if (S.per > 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = a[j] - a[0] - mean;
        m2 += q[j] + cnt * d * d;
      }
      out[0] = a[0] + mean;
      out[row] = m2;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = a[j], out[row + j] = q[j];
    }
  }
}

// The partials of a group, one workgroup per (n, group) and up to 1,024 threads: f(slab, channel, both values), 4 at a time
// in flight, with no division in the loop
template <class F>
__device__ __forceinline__ void each_partial(const float* partial, const Slab& S, int64_t n, int g, int per, F f) {
  const int row = S.C / per, cg = S.cg / per, NT = blockDim.x, dsl = NT / cg, dc = NT % cg;
  const float* p = partial + n * S.slabs * 2 * row + g * cg;
  int64_t sl = (int)threadIdx.x / cg;
  int c = (int)threadIdx.x % cg;
  while (sl < S.slabs) {
    float u[4], w[4];
    int64_t at[4];
    int ch[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] = sl, ch[i] = c;
      const float* from = p + (sl < S.slabs ? sl : S.slabs - 1) * 2 * row + c;
      u[i] = from[0], w[i] = from[row];
      sl += dsl, c += dc;
      if (c >= cg) c -= cg, ++sl;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at[i] < S.slabs) f(at[i], ch[i], u[i], w[i]);
  }
}
// sums of a and q over the workgroup, in thread 0
__device__ __forceinline__ void block_sum(double& a, double& q) {
  __shared__ double sa[16], sq[16];
  for (int m = 32; m >= 1; m >>= 1) a += __shfl_xor(a, m, 64), q += __shfl_xor(q, m, 64);
  if (threadIdx.x % 64 == 0) sa[threadIdx.x / 64] = a, sq[threadIdx.x / 64] = q;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < (int)blockDim.x / 64; ++i) a += sa[i], q += sq[i];
}

// joins them, about the first one's mean
__global__ __launch_bounds__(1024) void norm_slab_join_kernel(const float* __restrict__ partial, Slab S, float eps,
                                                              float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const int64_t ng = S.first + blockIdx.x, n = ng / S.G;
  const int g = (int)(ng % S.G);
  const double pivot = partial[n * S.slabs * 2 * (S.C / S.per) + g * (S.cg / S.per)];
  const double whole = (double)S.slab * S.per, rest = (double)(S.L - (S.slabs - 1) * S.slab) * S.per;
  double a = 0.0, q = 0.0;
  each_partial(partial, S, n, g, S.per, [&](int64_t sl, int, float m, float m2) {
    const double count = sl + 1 < S.slabs ? whole : rest, d = m - pivot;
    a += count * d;
    q += m2 + count * d * d;
  });
  block_sum(a, q);
  if (threadIdx.x == 0) {
    const double total = (double)S.L * S.cg, off = a / total, var = q / total - off * off;
    mean_out[ng] = (float)(pivot + off);
    rstd_out[ng] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));
  }
}

template <class T, int V, bool SILU, bool GATE>
__global__ __launch_bounds__(256) void norm_slab_apply_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                              Affine aff, Slab S, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, T* __restrict__ y) {
  const int cper = 256 / S.rper;
  const int r = threadIdx.x / cper, cc = threadIdx.x % cper;
  int64_t blk = S.first + blockIdx.x;
  const int cb = (int)(blk % S.cblocks);
  blk /= S.cblocks;
  const int64_t sl = blk % S.slabs, n = blk / S.slabs;
  const int col = cb * cper + cc;
  if (r >= S.rper || col >= S.cols) return;
  const int64_t l0 = sl * S.slab, l1 = l0 + S.slab < S.L ? l0 + S.slab : S.L;
  float m[V], k[V], w[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = col * V + j, g = c / S.cg;
    m[j] = mean[n * S.G + g];
    k[j] = rstd[n * S.G + g];
  }
  aff.load<V>((int64_t)col * V, S.C, w, b);
  const int64_t base = n * S.L * S.C + (int64_t)col * V;
#pragma unroll 4
  for (int64_t l = l0 + r; l < l1; l += S.rper) {
    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + base + l * S.C);
    Vec<T, V> gt, out;
    if (GATE) gt = *reinterpret_cast<const Vec<T, V>*>(gate + base + l * S.C);
#pragma unroll
    for (int j = 0; j < V; ++j)
      out.v[j] = from_f<T>(
          out_of<SILU, GATE>(fmaf((to_f(v.v[j]) - m[j]) * k[j], w[j], b[j]), GATE ? to_f(gt.v[j]) : 0.0f));
    *reinterpret_cast<Vec<T, V>*>(y + base + l * S.C) = out;
  }
}

// sums over a slab of dy0 xhat and dy0 per channel -> partial [n, slabs, 2, c]; writes dgate on the way
template <class T, int V, bool SILU, bool GATE>
__global__ __launch_bounds__(256) void norm_slab_back_stats_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                                   const T* __restrict__ dy, Affine aff, Slab S,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, T* __restrict__ dgate,
                                                                   float* __restrict__ partial) {
  __shared__ float s1[256 * V], s2[256 * V];
  const int cper = 256 / S.rper;
  const int r = threadIdx.x / cper, cc = threadIdx.x % cper;
  int64_t blk = S.first + blockIdx.x;
  const int cb = (int)(blk % S.cblocks);
  blk /= S.cblocks;
  const int64_t sl = blk % S.slabs, n = blk / S.slabs;
  const int col = cb * cper + cc;
  const bool live = r < S.rper && col < S.cols;
  const int64_t l0 = sl * S.slab, l1 = l0 + S.slab < S.L ? l0 + S.slab : S.L;
  float a[V], q[V], m[V], k[V], w[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = q[j] = 0.0f;
  if (live) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = col * V + j, g = c / S.cg;
      m[j] = mean[n * S.G + g];
      k[j] = rstd[n * S.G + g];
    }
    aff.load<V>((int64_t)col * V, S.C, w, b);
    const int64_t base = n * S.L * S.C + (int64_t)col * V;
#pragma unroll 4
    for (int64_t l = l0 + r; l < l1; l += S.rper) {
      const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + base + l * S.C);
      const Vec<T, V> d = *reinterpret_cast<const Vec<T, V>*>(dy + base + l * S.C);
      Vec<T, V> gt, dg;
      if (GATE) gt = *reinterpret_cast<const Vec<T, V>*>(gate + base + l * S.C);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (to_f(v.v[j]) - m[j]) * k[j];
        float dgj;
        const float d0 =
            back_of<SILU, GATE>(to_f(d.v[j]), fmaf(xh, w[j], b[j]), GATE ? to_f(gt.v[j]) : 0.0f, dgj);
        dg.v[j] = from_f<T>(dgj);
        a[j] = fmaf(d0, xh, a[j]);
        q[j] += d0;
      }
      if (GATE && dgate) *reinterpret_cast<Vec<T, V>*>(dgate + base + l * S.C) = dg;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s1[j * 256 + threadIdx.x] = a[j];
    s2[j * 256 + threadIdx.x] = q[j];
  }
  __syncthreads();
  if (r == 0 && col < S.cols) {
    float* out = partial + ((n * S.slabs + sl) * 2) * S.C + (int64_t)col * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int i = 1; i < S.rper; ++i) {
        a[j] += s1[j * 256 + i * cper + cc];
        q[j] += s2[j * 256 + i * cper + cc];
      }
      out[j] = a[j];
      out[S.C + j] = q[j];
    }
  }
}

// means over each group of dxhat xhat and dxhat -> sums [n, g, 2]
__global__ __launch_bounds__(1024) void norm_slab_back_join_kernel(const float* __restrict__ partial, Affine aff, Slab S,
                                                                   float* __restrict__ sums) {
  const int64_t ng = S.first + blockIdx.x, n = ng / S.G;
  const int g = (int)(ng % S.G);
  double a = 0.0, q = 0.0;
  each_partial(partial, S, n, g, 1, [&](int64_t, int c, float u, float v) {
    const double w = aff.weight(g * S.cg + c);
    a += w * u;
    q += w * v;
  });
  block_sum(a, q);
  if (threadIdx.x == 0) {
    const double total = (double)S.L * S.cg;
    sums[2 * ng] = (float)(a / total);
    sums[2 * ng + 1] = (float)(q / total);
  }
}

template <class T, int V, bool SILU, bool GATE>
__global__ __launch_bounds__(256) void norm_slab_back_apply_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                                   const T* __restrict__ dy, Affine aff, Slab S,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd,
                                                                   const float* __restrict__ sums, T* __restrict__ dx) {
  const int cper = 256 / S.rper;
  const int r = threadIdx.x / cper, cc = threadIdx.x % cper;
  int64_t blk = S.first + blockIdx.x;
  const int cb = (int)(blk % S.cblocks);
  blk /= S.cblocks;
  const int64_t sl = blk % S.slabs, n = blk / S.slabs;
  const int col = cb * cper + cc;
  if (r >= S.rper || col >= S.cols) return;
  const int64_t l0 = sl * S.slab, l1 = l0 + S.slab < S.L ? l0 + S.slab : S.L;
  float m[V], k[V], w[V], b[V], c1[V], c2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = col * V + j;
    const int64_t g = n * S.G + c / S.cg;
    m[j] = mean[g];
    k[j] = rstd[g];
    c2[j] = sums[2 * g];
    c1[j] = sums[2 * g + 1];
  }
  aff.load<V>((int64_t)col * V, S.C, w, b);
  const int64_t base = n * S.L * S.C + (int64_t)col * V;
#pragma unroll 4
  for (int64_t l = l0 + r; l < l1; l += S.rper) {
    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + base + l * S.C);
    const Vec<T, V> d = *reinterpret_cast<const Vec<T, V>*>(dy + base + l * S.C);
    Vec<T, V> gt, out;
    if (GATE) gt = *reinterpret_cast<const Vec<T, V>*>(gate + base + l * S.C);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xh = (to_f(v.v[j]) - m[j]) * k[j];
      float dgj;
      const float d0 = back_of<SILU, GATE>(to_f(d.v[j]), fmaf(xh, w[j], b[j]), GATE ? to_f(gt.v[j]) : 0.0f, dgj);
      out.v[j] = from_f<T>(k[j] * (d0 * w[j] - c1[j] - xh * c2[j]));
    }
    *reinterpret_cast<Vec<T, V>*>(dx + base + l * S.C) = out;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------

struct NormPlan {
  bool rows;              // the one-position form
  int V, NV;
  int whole;              // threads a group of the form in registers, up to 64: several groups a workgroup; 0: slabs
  Rows R;
  int64_t slabs;
  Slab S;
  size_t floats;          // workspace
};

inline bool norm_wide(const ttc_group_norm_args& A) {
  const int V = A.dtype == TTC_DTYPE_F32 ? 4 : 8;
  return A.c % V == 0 && aligned16(A.x) && aligned16(A.gate) && aligned16(A.y) && aligned16(A.dy) &&
         aligned16(A.dx) && aligned16(A.dgate);
}

// Everything but the vector width follows from sizes alone, so that the workspace's size does too: it is computed for
// both widths and the larger taken.
inline NormPlan norm_plan(const ttc_group_norm_args& A, bool wide) {
  NormPlan P{};
  const int full = A.dtype == TTC_DTYPE_F32 ? 4 : 8;
  const int64_t cg = A.c / A.groups;
  wide = wide && A.c % full == 0;
  const int Vr = wide && cg % full == 0 ? full : 1;
  const int64_t vecs = ceil_div(cg, Vr);
  P.rows = A.l == 1 && vecs <= 64 * 4;
  if (P.rows) {
    P.V = Vr;
    Rows& R = P.R;
    R.n = A.n;
    R.G = (int)A.groups;
    R.cg = (int)cg;
    R.lanes = 1;
    while (R.lanes < 64 && R.lanes < vecs) R.lanes *= 2;
    const int need = (int)ceil_div(vecs, R.lanes);
    P.NV = need <= 1 ? 1 : need <= 2 ? 2 : 4;
    const int units = 256 / R.lanes;
    R.gper = A.groups < units ? (int)A.groups : units;
    R.rper = units / R.gper;
    R.gblocks = (int)ceil_div(A.groups, R.gper);
    // Workgroups: 2,048 fill the GPU; half as many in the backward, whose partial sums grow with them
    int64_t want = (A.backward ? 1024 : 2048) / R.gblocks;
    if (want < 1) want = 1;
    int64_t slab = ceil_div(A.n, want);
    if (slab < R.rper) slab = R.rper;
    if (slab > (1 << 30)) slab = 1 << 30;
    R.slab = (int)slab;
    P.slabs = ceil_div(A.n, slab);
    if (A.backward && (A.dweight || A.dbias)) P.floats = (size_t)(P.slabs * R.rper * 2 * A.c);
    return P;
  }
  Slab& S = P.S;
  P.V = wide ? full : 1;
  S.L = A.l;
  S.C = (int)A.c;
  S.G = (int)A.groups;
  S.cg = (int)cg;
  S.cols = (int)(A.c / P.V);
  S.per = !A.backward && cg % P.V == 0 ? P.V : 1;
  const int cper = S.cols < 256 ? S.cols : 256;
  S.rper = 256 / cper;
  S.cblocks = (int)ceil_div(S.cols, 256 / S.rper);
  if (!A.backward) {
    const int Vw = wide && cg % full == 0 ? full : 1;
    const int64_t v = ceil_div(cg, Vw) <= 1024 * WHOLE && A.l <= 1024 * WHOLE ? A.l * (cg / Vw) : 1024 * WHOLE + 1;
    // Rows of less than 64 bytes a group are read in halves of what memory gives: large arrays of them take the slabs (1,024 x
    // 512 in 32 groups, bf16, 64 of them: slabs 55 us, whole 85; 32: 33, 37; 16: 24, 25 in one launch; wider rows, 64 x 256 x
    // 1,024 in 8 groups: 32, whole 25)
    const bool narrow = cg * (A.dtype == TTC_DTYPE_F32 ? 4 : 2) < 64;
    if (v <= 64 * SMALL) {  // teams beside each other read whole rows between them
      P.V = Vw;
      P.whole = 1;
      while (P.whole * SMALL < v) P.whole *= 2;
      return P;
    }
    if (v <= 1024 * WHOLE && (!narrow || A.n * A.l * A.c <= 1 << 23)) {
      P.V = Vw;
      P.whole = (int)(ceil_div(ceil_div(v, WHOLE), 64) * 64);
      if (P.whole < 256) P.whole = 256;
      return P;
    }
  }
  const int64_t want = ceil_div(1024, A.n * S.cblocks);
  int64_t slab = ceil_div(A.l, want);
  slab = slab < 4 * S.rper ? 4 * S.rper : slab;
  S.slab = slab < A.l ? slab : A.l;
  S.slabs = ceil_div(A.l, S.slab);
  P.floats = (size_t)(A.n * S.slabs * 2 * A.c) + (size_t)(A.n * A.groups * 2);
  return P;
}

template <class T, int V, bool SILU, bool GATE>
int norm_run(const ttc_group_norm_args& A, const NormPlan& P, hipStream_t s) {
  const T *x = static_cast<const T*>(A.x), *gate = static_cast<const T*>(A.gate), *dy = static_cast<const T*>(A.dy);
  const Affine aff{A.weight, A.bias, A.weight_dtype == TTC_DTYPE_BF16, aligned16(A.weight) && aligned16(A.bias)};
  const float eps = (float)A.eps;
  float* ws = static_cast<float*>(A.workspace);
  const int G = (int)A.groups;
  int64_t parts = 0;
  if (P.rows) {
    auto go = [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      const int64_t blocks = P.slabs * P.R.gblocks;
      if (blocks > max_blocks(256)) return TTC_LQR_EINVAL;
      const dim3 grid((unsigned)blocks);
      if (!A.backward) {
        hipLaunchKernelGGL((norm_row_kernel<T, V, NV, SILU, GATE>), grid, dim3(256), 0, s, x, gate, aff, P.R, eps,
                           static_cast<T*>(A.y), A.mean, A.rstd);
        return launched();
      }
      float* part = A.dweight || A.dbias ? ws : nullptr;
      hipLaunchKernelGGL((norm_row_backward_kernel<T, V, NV, SILU, GATE>), grid, dim3(256), 0, s, x, gate, dy, aff, P.R,
                         A.mean, A.rstd, static_cast<T*>(A.dx), static_cast<T*>(A.dgate), part);
      return launched();
    };
    const int rc = P.NV == 1   ? go(std::integral_constant<int, 1>{})
                   : P.NV == 2 ? go(std::integral_constant<int, 2>{})
                               : go(std::integral_constant<int, 4>{});
    if (rc != TTC_LQR_OK) return rc;
    parts = P.slabs * P.R.rper;
  } else {
    Slab S = P.S;
    const int64_t blocks = A.n * S.slabs * S.cblocks, joins = A.n * G;
    const int64_t parts_a_group = S.slabs * (S.cg / S.per);
    const dim3 block(256), joiners(parts_a_group >= 1024 ? 1024 : (unsigned)(ceil_div(parts_a_group, 64) * 64));
    int rc = TTC_LQR_OK;
    auto each = [&](int64_t n, auto go) {
      if (rc == TTC_LQR_OK)
        rc = in_launches(n, 1024, [&](int64_t first, dim3 grid) {
          S.first = first;
          go(grid);
        });
    };
    if (P.whole) {
      const bool small = P.whole <= 64;
      const int threads = small ? 256 : P.whole;
      rc = in_launches(ceil_div(joins, threads / P.whole), threads, [&](int64_t first, dim3 grid) {
        S.first = first;
        auto go = [&](auto nv) {
          hipLaunchKernelGGL((norm_whole_kernel<T, V, SILU, GATE, decltype(nv)::value>), grid, dim3(threads), 0, s, x, gate,
                             aff, S, P.whole, joins, eps, static_cast<T*>(A.y), A.mean, A.rstd);
        };
        if (small) go(std::integral_constant<int, SMALL>{});
        else go(std::integral_constant<int, WHOLE>{});
      });
      return rc;
    }
    float* extra = ws + A.n * S.slabs * 2 * A.c;
    if (!A.backward) {
      float* mean = A.mean ? A.mean : extra;
      float* rstd = A.mean ? A.rstd : extra + A.n * G;
      each(blocks, [&](dim3 g) { hipLaunchKernelGGL((norm_slab_stats_kernel<T, V>), g, block, 0, s, x, S, ws); });
      each(joins, [&](dim3 g) { hipLaunchKernelGGL(norm_slab_join_kernel, g, joiners, 0, s, ws, S, eps, mean, rstd); });
      each(blocks, [&](dim3 g) {
        hipLaunchKernelGGL((norm_slab_apply_kernel<T, V, SILU, GATE>), g, block, 0, s, x, gate, aff, S, mean, rstd,
                           static_cast<T*>(A.y));
      });
      return rc;
    }
    each(blocks, [&](dim3 g) {
      hipLaunchKernelGGL((norm_slab_back_stats_kernel<T, V, SILU, GATE>), g, block, 0, s, x, gate, dy, aff, S, A.mean, A.rstd,
                         static_cast<T*>(A.dgate), ws);
    });
    if (A.dx) {
      each(joins, [&](dim3 g) { hipLaunchKernelGGL(norm_slab_back_join_kernel, g, joiners, 0, s, ws, aff, S, extra); });
      each(blocks, [&](dim3 g) {
        hipLaunchKernelGGL((norm_slab_back_apply_kernel<T, V, SILU, GATE>), g, block, 0, s, x, gate, dy, aff, S, A.mean,
                           A.rstd, extra, static_cast<T*>(A.dx));
      });
    }
    if (rc != TTC_LQR_OK) return rc;
    parts = A.n * S.slabs;
  }
  if (A.dweight || A.dbias) {
    const dim3 grid((unsigned)ceil_div(A.c, 16));
    if (A.weight_dtype == TTC_DTYPE_BF16)
      hipLaunchKernelGGL(norm_affine_sum_kernel<__bf16>, grid, dim3(1024), 0, s, ws, parts, A.c,
                         static_cast<__bf16*>(A.dweight), static_cast<__bf16*>(A.dbias));
    else
      hipLaunchKernelGGL(norm_affine_sum_kernel<float>, grid, dim3(1024), 0, s, ws, parts, A.c,
                         static_cast<float*>(A.dweight), static_cast<float*>(A.dbias));
  }
  return launched();
}

template <class T, int V>
int norm_dispatch(const ttc_group_norm_args& A, const NormPlan& P, hipStream_t s) {
  if (A.activation == 1) return A.gate ? norm_run<T, V, true, true>(A, P, s) : norm_run<T, V, true, false>(A, P, s);
  return A.gate ? norm_run<T, V, false, true>(A, P, s) : norm_run<T, V, false, false>(A, P, s);
}

// 0, or the status that the block's sizes and types deserve
inline int norm_check(const ttc_group_norm_args& A) {
  const int64_t lim = 1 << 24;
  if (A.n < 0 || A.l < 0 || A.c < 0 || A.c > lim || A.groups <= 0 || A.c % A.groups || A.activation < 0 ||
      A.activation > 1 || !(A.eps >= 0.0) || !countable({A.n, A.l, A.c}))
    return TTC_LQR_EINVAL;
  auto known = [](int64_t t) { return t == TTC_DTYPE_F32 || t == TTC_DTYPE_BF16; };
  if (!known(A.dtype) || !known(A.weight_dtype)) return TTC_LQR_EUNSUPPORTED;
  return TTC_LQR_OK;
}

inline size_t norm_floats(const ttc_group_norm_args& A) {
  const size_t a = norm_plan(A, false).floats, b = norm_plan(A, true).floats;
  return a > b ? a : b;
}

}  // namespace ttc

extern "C" size_t ttc_group_norm_workspace_bytes(const ttc_group_norm_args* args) {
  using namespace ttc;
  if (!args || norm_check(*args) != TTC_LQR_OK || args->n == 0 || args->l == 0 || args->c == 0) return 0;
  return norm_floats(*args) * sizeof(float);
}

extern "C" int ttc_group_norm(const ttc_group_norm_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_group_norm_args& A = *args;
  if (const int rc = norm_check(A)) return rc;
  if (A.n == 0 || A.l == 0 || A.c == 0) return TTC_LQR_OK;
  if (!A.x || !A.weight != !A.bias || !A.mean != !A.rstd) return TTC_LQR_EINVAL;
  if (A.backward ? !A.dy || !A.mean || (A.dgate && !A.gate) : !A.y) return TTC_LQR_EINVAL;
  const size_t need = norm_floats(A) * sizeof(float);
  if (need > 0 && (!A.workspace || A.workspace_bytes < 0 || (size_t)A.workspace_bytes < need)) return TTC_LQR_EINVAL;
  const NormPlan P = norm_plan(A, norm_wide(A));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (A.dtype == TTC_DTYPE_F32)
    return P.V == 4 ? norm_dispatch<float, 4>(A, P, s) : norm_dispatch<float, 1>(A, P, s);
  return P.V == 8 ? norm_dispatch<__bf16, 8>(A, P, s) : norm_dispatch<__bf16, 1>(A, P, s);
}
