// ttc_ops_delta.hip -- the gated delta rule: token by token (single tokens of a serving batch, short inputs), sums over shared
// heads, and the C entries (formulas: ttc_ops_delta.hpp).
#include "ttc_ops_delta.hpp"
#include "ttc_ops_mfma.hpp"

namespace ttc {

struct Tokens {
  Side q, k, v;
  const void *gamma, *beta;
  int64_t gb, gt, gh, bb, bt, bh, B, T, nslots;
  bool gamma_bf16, beta_bf16, normalize;
  int kd, vd, H;
  float scale, eps;
  const float* state_in;  // [slot, head, kd, vd]
  float* state_out;
  const int32_t* slots;
  void* o;
};

// A workgroup holds 32 columns of one head's state in registers, a thread 4 of them for RPT rows.  Both reads of the state meet
// in one sum over the rows, since S_t' q = e^g S' q + (k . q) b e: one exchange a token, and for one token the state is read and
// written once (8 bytes an element against 9 flops): bound by memory.  192 sequences x 16 states of 128 x 128 in a pool: 95 us a
// call for 406 MB, 4.3 TB/s where a copy of 1 GiB reaches 5.1; one sequence of 8 states of 64 x 64: 5.3 us, most of it latency.
template <class T, int RPT>
__global__ __launch_bounds__(256) void delta_tokens_kernel(Tokens A, int tiles, bool wide, int64_t first) {
  constexpr int COLS = 32, STEP = 32;  // columns of a workgroup, rows between a thread's
  __shared__ float part[2][4][2][COLS], dots[2][4][3];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = (int)(blockIdx.x % tiles);
  const int64_t bh = first + blockIdx.x / tiles, b = bh / A.H;
  const int h = (int)(bh % A.H);
  const int e0 = tile * COLS + (lane & 7) * 4, r0 = wave * 8 + (lane >> 3);
  const int64_t slot = A.slots ? A.slots[b] : b;
  T* out = static_cast<T*>(A.o) + (b * A.T * A.H + h) * (int64_t)A.vd;
  if (slot < 0 || slot >= A.nslots) {  // a row without a state
    for (int64_t t = 0; t < A.T; ++t)
      for (int j = threadIdx.x; j < COLS && tile * COLS + j < A.vd; j += 256)
        out[t * A.H * (int64_t)A.vd + tile * COLS + j] = from_f<T>(0.0f);
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
      f[i] = *reinterpret_cast<const float4*>(A.state_in + base + row_at(i) * A.vd + (held[0] ? e0 : 0));
#pragma unroll
    for (int i = 0; i < RPT; ++i) S[i][0] = f[i].x, S[i][1] = f[i].y, S[i][2] = f[i].z, S[i][3] = f[i].w;
  } else {
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = A.state_in[base + row_at(i) * A.vd + col_at(j)];
  }
  const T *q = A.q.at<T>(b, h), *k = A.k.at<T>(b, h), *v = A.v.at<T>(b, h);
  for (int64_t t = 0; t < A.T; ++t) {
    const int buf = t & 1;
    const float lg = gate_value(A.gamma, A.gamma_bf16, b * A.gb + h * A.gh + t * A.gt);
    const float be = gate_value(A.beta, A.beta_bf16, b * A.bb + h * A.bh + t * A.bt);
    float vv[4], kk[RPT], qq[RPT], sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f}, d[3] = {0.f, 0.f, 0.f};
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
        S[i][j] = lg < RESET ? 0.0f : S[i][j] * decay;
        sk[j] = row ? fmaf(kk[i], S[i][j], sk[j]) : sk[j];
        sq[j] = row ? fmaf(qq[i], S[i][j], sq[j]) : sq[j];
      }
      d[0] = row ? fmaf(kk[i], kk[i], d[0]) : d[0];
      d[1] = row ? fmaf(qq[i], qq[i], d[1]) : d[1];
      d[2] = row ? fmaf(kk[i], qq[i], d[2]) : d[2];
    }
#pragma unroll
    for (int m = 8; m <= 32; m <<= 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sk[j] += __shfl_xor(sk[j], m, 64), sq[j] += __shfl_xor(sq[j], m, 64);
#pragma unroll
      for (int j = 0; j < 3; ++j) d[j] += __shfl_xor(d[j], m, 64);
    }
    if (lane < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) part[buf][wave][0][lane * 4 + j] = sk[j], part[buf][wave][1][lane * 4 + j] = sq[j];
      if (lane == 0) dots[buf][wave][0] = d[0], dots[buf][wave][1] = d[1], dots[buf][wave][2] = d[2];
    }
    __syncthreads();  // the next token writes the other buffer, and meets this barrier before it comes back to this one
    auto sum = [&](auto at) { return (at(0) + at(1)) + (at(2) + at(3)); };
    const float rk = A.normalize ? 1.0f / sqrtf(sum([&](int w) { return dots[buf][w][0]; }) + A.eps) : 1.0f;
    const float rq = A.normalize ? 1.0f / sqrtf(sum([&](int w) { return dots[buf][w][1]; }) + A.eps) : 1.0f;
    const float kq = sum([&](int w) { return dots[buf][w][2]; }) * rk;
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = (lane & 7) * 4 + j;
      u[j] = be * (vv[j] - rk * sum([&](int w) { return part[buf][w][0][c]; }));
    }
    if (threadIdx.x < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = sum([&](int w) { return part[buf][w][1][lane * 4 + j]; });
        if (held[j]) out[t * A.H * (int64_t)A.vd + e0 + j] = from_f<T>((rq * A.scale) * fmaf(kq, u[j], s));
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = fmaf(rk * kk[i], u[j], S[i][j]);
  }
  if (A.state_out == nullptr) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + STEP * i;
    if (r >= A.kd) continue;
    if (wide) {
      if (e0 < A.vd)
        *reinterpret_cast<float4*>(A.state_out + base + r * A.vd + e0) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (held[j]) A.state_out[base + r * A.vd + e0 + j] = S[i][j];
    }
  }
}

int launch_tokens(const Tokens& A, bool bf16, hipStream_t s) {
  const int tiles = (A.vd + 31) / 32;
  const bool wide = A.vd % 4 == 0 && aligned16(A.state_in) && aligned16(A.state_out);
  auto go = [&](auto kernel) {
    return in_launches(A.B * A.H * tiles, 256, [&](int64_t first, dim3 grid) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, A, tiles, wide, first / tiles);
    }, tiles);
  };
  if (bf16)
    return A.kd <= 32 ? go(delta_tokens_kernel<__bf16, 1>) : A.kd <= 64 ? go(delta_tokens_kernel<__bf16, 2>)
                                                                        : go(delta_tokens_kernel<__bf16, 4>);
  return A.kd <= 32 ? go(delta_tokens_kernel<float, 1>) : A.kd <= 64 ? go(delta_tokens_kernel<float, 2>)
                                                                     : go(delta_tokens_kernel<float, 4>);
}

// The states in front of the segments: S_{j+1} = M_j S_j + own_j from state_in on, or (BACK) R_{j-1} = M_j' R_j + own_j from the
// last one.  A workgroup has 16 columns, a wave 16 rows of them; what a segment's reset drops has no effect, whatever it holds.
// Bound by the chain: 16 segments x 16 heads of 128 x 128 53 us, 3 us a segment, for 17 MB of matrices that each XCD reads once.
template <int KD, bool BACK>
__global__ __launch_bounds__(KD / 16 * 64) void delta_join_kernel(Delta A) {
  using Op = Operand<__bf16>;
  constexpr int DB = KD / 32, RS = KD + 8, PLANE = 16 * RS;
  __shared__ __attribute__((aligned(16))) __bf16 Now[2][3 * PLANE];  // the state's columns as rows, in their parts
  const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Spread W = spread(A.first, A.vdp / 16);
  const int c = W.block * 16 + n, r0 = wave * 16;
  const int64_t bh = W.group;
  auto segment = [&](int i) { return bh * A.segs + (BACK ? A.segs - 1 - i : i); };
  struct Part {
    float m[DB][8], own[4];
    int dead;
  };
  auto fetch = [&](int i, Part& P) {
    const float* p = A.seg_matrix + segment(i) * KD * KD;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        P.m[d][j] = BACK ? p[(32 * d + 8 * g + j) * KD + r0 + n] : p[(r0 + n) * KD + 32 * d + 8 * g + j];
#pragma unroll
    for (int j = 0; j < 4; ++j) P.own[j] = A.seg_state[(segment(i) * KD + r0 + 4 * g + j) * A.vdp + c];
    P.dead = A.seg_dead[segment(i)];
  };
  f32x4 now;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = r0 + 4 * g + j;
    now[j] = A.state_in && r < A.kd && c < A.vd ? A.state_in[(bh * A.kd + r) * A.vd + c] : 0.0f;
  }
  // segment i, whose part is here, while that of the next one is on its way
  auto pass = [&](int i, const Part& P, Part& ahead, __bf16* to) {
    if (i + 1 < A.segs) fetch(i + 1, ahead);
#pragma unroll
    for (int j = 0; j < 4; ++j) A.seg_state[(segment(i) * KD + r0 + 4 * g + j) * A.vdp + c] = now[j];
    if (i + 1 == A.segs) return;
    Op::put_wide(&to[n * RS + r0 + 4 * g], PLANE, now);
    __syncthreads();  // the next segment writes the other buffer, and meets this barrier before it comes back to this one
    f32x4 sum[2] = {{P.own[0], P.own[1], P.own[2], P.own[3]}, {0.f, 0.f, 0.f, 0.f}};
    if (!P.dead) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const __bf16* x = &to[n * RS + 32 * d + 8 * g];
        sum[d & 1] = Op::mma(Op::wide(P.m[d]), Op::Wide{Op::row(x), Op::row(x + PLANE), Op::row(x + 2 * PLANE)}, sum[d & 1]);
      }
    }
    now = sum[0] + sum[1];
  };
  Part even, odd;
  fetch(0, even);
  for (int i = 0; i < A.segs; i += 2) {
    pass(i, even, odd, Now[0]);
    if (i + 1 < A.segs) pass(i + 1, odd, even, Now[1]);
  }
}

int launch_delta_join(const Delta& A, bool back, hipStream_t s) {
  const int blocks = A.vdp / 16;
  auto go = [&](auto kernel, int threads) {
    return in_launches(A.B * A.H * blocks, threads, [&](int64_t first, dim3 grid) {
      Delta P = A;
      P.first = first / blocks;
      hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, P);
    }, blocks);
  };
  if (A.kd <= 32) return back ? go(delta_join_kernel<32, true>, 128) : go(delta_join_kernel<32, false>, 128);
  if (A.kd <= 64) return back ? go(delta_join_kernel<64, true>, 256) : go(delta_join_kernel<64, false>, 256);
  return back ? go(delta_join_kernel<128, true>, 512) : go(delta_join_kernel<128, false>, 512);
}

// Gradients of shared heads: out [B, T, heads / share, d] = sums over `share` heads of `in`, element (b, t, h, i) at
// b sb + t st + h sh + i
template <class T>
__global__ __launch_bounds__(256) void head_sum_kernel(const float* __restrict__ in, T* __restrict__ out, int64_t first, int64_t n,
                                                       int64_t tokens, int own, int share, int d, int64_t sb, int64_t st,
                                                       int64_t sh) {
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t row = i / d, token = row / own;
  const float* p = in + token / tokens * sb + token % tokens * st + row % own * share * sh + i % d;
  float a = 0.0f;
  for (int j = 0; j < share; ++j) a += p[j * sh];
  out[i] = from_f<T>(a);
}

// ---- host ----------------------------------------------------------------------------------------------------

// Up to this many tokens are taken one by one where nothing is kept for a backward.  The chunk kernels' time (12.8 to 72 us) hardly
// depends on the number of tokens below a chunk's, and meets the other's between 5 and 8.  us on the GPU, states in and out, one by
// one by tokens, and in a chunk:                                     1     2     3     4     5     6     8    chunk
//   1 sequence x 8 heads of 64 x 64, fp32                          4.5   5.9   7.2   8.6   9.9  11.3  14.1     12.8
//   1 x 16 of 128 x 128, bf16                                      5.1   6.5   8.0   9.5  11.0  12.5  15.6     19.2
//   16 x 16 of 128 x 128, bf16                                    11.0  13.1  15.8  18.4  20.9  23.3  28.7     25.5
//   64 x 16 of 128 x 128, bf16                                    29.9  36.2  43.5  51.4  60.1  68.2  84.5     71.6
//   64 x 32 of 64 x 64, bf16                                      17.9  24.0  31.6  39.3  47.5  55.7  70.5     58.2
//   32 x 16 of 64 x 64, fp32                                       7.7  10.6  12.9  15.6  17.9  20.4  25.3     19.1
constexpr int64_t ONE_BY_ONE = 4;

inline int padded(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

inline int delta_check(int64_t dtype, int64_t gamma_dtype, int64_t beta_dtype, std::initializer_list<int64_t> sizes, int64_t heads,
                       int64_t qh, int64_t kh, int64_t vh, int64_t dk, int64_t dv) {
  for (int64_t v : sizes)
    if (v < 0) return TTC_LQR_EINVAL;
  if (heads < 1 || heads > (1 << 24) || qh < 1 || kh < 1 || vh < 1 || heads % qh || heads % kh || heads % vh || dk < 1 ||
      dk > MAX_DIM || dv < 1 || dv > MAX_DIM || !countable(sizes))
    return TTC_LQR_EINVAL;
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16) return TTC_LQR_EUNSUPPORTED;
  for (int64_t t : {gamma_dtype, beta_dtype})
    if (t != TTC_DTYPE_F32 && t != dtype) return TTC_LQR_EUNSUPPORTED;
  return TTC_LQR_OK;
}

inline int delta_check(const ttc_delta_rule_args& A) {  // a token's share of what is kept is below 16 x MAX_DIM values
  return delta_check(A.dtype, A.gamma_dtype, A.beta_dtype, {A.batch, A.tokens, A.heads, MAX_DIM, 16 * MAX_DIM}, A.heads,
                     A.q_heads, A.k_heads, A.v_heads, A.dk, A.dv);
}

struct DeltaLayout {  // bytes from the start of `saved` (inverse to E) and of the workspace; `saved` lies in it where none is given
  int64_t inverse, scores, rows, odd, S, E, seg_matrix, seg_dead, kept;
  int64_t R, dV, dq, dk, seg_state, total;
  int64_t chunks, seg_chunks;
  int vdp, segs;
};

// Segments: enough workgroups to fill the GPU's 256 CUs twice, of at least 4 chunks each.  A split sweep does some three times
// the work (own states, and what becomes of the one in front), so heads that fill the GPU by themselves are not split.  us a
// call by the workgroups aimed at:                          1     128    256    384    512    768  1,024  1,536
//   16,381 tokens x 16 heads of 128 x 128, bf16         1,463    669    433    448    412    449    464    520
//   4 x 2,048 x 32 of 64 x 64, bf16, training             581    581    576    551    536    578    557    558
//   2 x 2,048 x 32 of 128 x 128, bf16, training           714    714    720    710    675    753    735    737
//   3 x 509 x 12 of 48 x 80, fp32, training               174    174    160    157    157    157    157    157
//   4,096 x 16 of 128 x 128, fp32                         735    344    242    256    250    276    296    295
//   4 x 4,096 x 8 of 32 x 32, bf16                        248    124     88     90     80     80     80     80
//   8 x 2,048 x 32 of 128 x 128, bf16                     414    413    414    414    411    405    721    675
inline void segments_of(const ttc_delta_rule_args& A, DeltaLayout& W) {
  const int64_t sweeps = A.batch * A.heads * (A.dv > 64 ? 2 : 1);
  int64_t count = sweeps > 0 ? 512 / sweeps : 1;
  if (count > W.chunks / 4) count = W.chunks / 4;
  if (count < 2) count = 1;
  W.seg_chunks = ceil_div(W.chunks > 0 ? W.chunks : 1, count);
  W.segs = (int)ceil_div(W.chunks > 0 ? W.chunks : 1, W.seg_chunks);
}

inline DeltaLayout delta_layout(const ttc_delta_rule_args& A) {
  DeltaLayout W{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const bool bf16 = A.dtype == TTC_DTYPE_BF16, keep = A.saved != nullptr || A.backward;
  const int64_t C = chunk_tokens(bf16), tiles = C / 16 * (C / 16 + 1) / 2;
  W.chunks = ceil_div(A.tokens, C);
  W.vdp = padded(A.dv);
  segments_of(A, W);
  const int64_t units = A.batch * A.heads * W.chunks, state = (int64_t)padded(A.dk) * W.vdp * 4, values = C * W.vdp * 4;
  const int64_t tile = bf16 ? 3 * 512 : 1024;  // values in three parts of 16 bits
  W.inverse = take(units * tiles * tile);
  W.scores = take(units * tiles * tile);
  W.rows = take(units * ROWS * C * 4);
  W.odd = take(units * 4);
  W.S = take(keep ? units * state : 0);
  W.E = take(keep ? units * values : 0);
  const int64_t parts = W.segs > 1 ? A.batch * A.heads * W.segs : 0;
  W.seg_matrix = take(parts * padded(A.dk) * padded(A.dk) * 4);
  W.seg_dead = take(parts * 4);
  W.kept = at;
  if (A.backward || A.saved) at = 0;
  W.seg_state = take(parts * state);
  if (A.backward) {
    W.R = take(units * state);
    W.dV = take(units * values);
    W.dq = take(A.heads != A.q_heads && A.dq ? A.batch * A.tokens * A.heads * A.dk * 4 : 0);
    W.dk = take(A.heads != A.k_heads && A.dk_out ? A.batch * A.tokens * A.heads * A.dk * 4 : 0);
    W.total = at;
  } else {
    W.total = !A.saved && A.tokens <= ONE_BY_ONE ? 0 : at;
  }
  return W;
}

inline Side side_of(const void* p, const int64_t* st, int64_t heads, int64_t own) {
  return Side{p, st[0], st[1], st[2], (int)(heads / own)};
}

int launch_delta_any(const Delta& A, bool bf16, int what, hipStream_t s) {
  if (bf16)
    return A.kd <= 32   ? launch_delta_kd32<__bf16>(A, what, s)
           : A.kd <= 64 ? launch_delta_kd64<__bf16>(A, what, s)
                        : launch_delta_kd128<__bf16>(A, what, s);
  return A.kd <= 32   ? launch_delta_kd32<float>(A, what, s)
         : A.kd <= 64 ? launch_delta_kd64<float>(A, what, s)
                      : launch_delta_kd128<float>(A, what, s);
}

int head_sum(const float* in, void* out, bool bf16, const ttc_delta_rule_args& A, int64_t own, int64_t d, int64_t sb, int64_t st,
             int64_t sh, hipStream_t s) {
  const int64_t n = A.batch * A.tokens * own * d;
  const int share = (int)(A.heads / own);
  return in_launches(ceil_div(n, 256), 256, [&](int64_t first, dim3 grid) {
    if (bf16)
      hipLaunchKernelGGL(head_sum_kernel<__bf16>, grid, dim3(256), 0, s, in, static_cast<__bf16*>(out), first, n, A.tokens, (int)own,
                         share, (int)d, sb, st, sh);
    else
      hipLaunchKernelGGL(head_sum_kernel<float>, grid, dim3(256), 0, s, in, static_cast<float*>(out), first, n, A.tokens, (int)own,
                         share, (int)d, sb, st, sh);
  });
}

__global__ __launch_bounds__(256) void copy_state_kernel(const float* from, float* to, int64_t first, int64_t n) {
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.0f;
}

}  // namespace ttc

extern "C" size_t ttc_delta_rule_workspace_bytes(const ttc_delta_rule_args* args) {
  using namespace ttc;
  if (!args || delta_check(*args) != TTC_LQR_OK) return 0;
  return (size_t)delta_layout(*args).total;
}

extern "C" size_t ttc_delta_rule_saved_bytes(const ttc_delta_rule_args* args) {
  using namespace ttc;
  if (!args || delta_check(*args) != TTC_LQR_OK) return 0;
  ttc_delta_rule_args A = *args;
  A.backward = 1;
  return (size_t)delta_layout(A).kept;
}

extern "C" int ttc_delta_rule(const ttc_delta_rule_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_delta_rule_args& A = *args;
  if (const int rc = delta_check(A)) return rc;
  if (!(A.eps >= 0)) return TTC_LQR_EINVAL;
  const bool some = A.batch > 0 && A.tokens > 0, bf16 = A.dtype == TTC_DTYPE_BF16;
  if (some && (!A.q || !A.k || !A.v || !A.log_gamma || !A.beta)) return TTC_LQR_EINVAL;
  if (some && (A.backward ? !A.d_o || !A.saved : !A.o)) return TTC_LQR_EINVAL;
  const DeltaLayout W = delta_layout(A);
  if (W.total > 0 && (!A.workspace || !aligned16(A.workspace) || A.workspace_bytes < W.total)) return TTC_LQR_EINVAL;
  if (A.saved && (!aligned16(A.saved) || A.saved_bytes < W.kept)) return TTC_LQR_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!some) {  // no tokens: the state passes
    const float* from = A.backward ? A.d_final_state : A.initial_state;
    float* to = A.backward ? A.d_initial_state : A.final_state;
    const int64_t n = A.batch * A.heads * A.dk * A.dv;
    if (!to) return TTC_LQR_OK;
    return in_launches(ceil_div(n, 256), 256, [&](int64_t first, dim3 grid) {
      hipLaunchKernelGGL(copy_state_kernel, grid, dim3(256), 0, s, from, to, first, n);
    });
  }
  const Side q = side_of(A.q, A.q_stride, A.heads, A.q_heads), k = side_of(A.k, A.k_stride, A.heads, A.k_heads),
             v = side_of(A.v, A.v_stride, A.heads, A.v_heads);
  if (!A.backward && !A.saved && A.tokens <= ONE_BY_ONE) {
    Tokens P{};
    P.q = q, P.k = k, P.v = v;
    P.gamma = A.log_gamma, P.beta = A.beta;
    P.gb = A.gamma_stride[0], P.gt = A.gamma_stride[1], P.gh = A.gamma_stride[2];
    P.bb = A.beta_stride[0], P.bt = A.beta_stride[1], P.bh = A.beta_stride[2];
    P.B = P.nslots = A.batch, P.T = A.tokens, P.H = (int)A.heads;
    P.gamma_bf16 = A.gamma_dtype == TTC_DTYPE_BF16, P.beta_bf16 = A.beta_dtype == TTC_DTYPE_BF16;
    P.normalize = A.normalize != 0;
    P.kd = (int)A.dk, P.vd = (int)A.dv;
    P.scale = (float)A.scale, P.eps = (float)A.eps;
    P.state_in = A.initial_state, P.state_out = A.final_state;
    P.o = A.o;
    return launch_tokens(P, bf16, s);
  }
  Delta P{};
  P.q = q, P.k = k, P.v = v;
  P.gamma = A.log_gamma, P.beta = A.beta;
  P.gb = A.gamma_stride[0], P.gt = A.gamma_stride[1], P.gh = A.gamma_stride[2];
  P.bb = A.beta_stride[0], P.bt = A.beta_stride[1], P.bh = A.beta_stride[2];
  P.gamma_bf16 = A.gamma_dtype == TTC_DTYPE_BF16, P.beta_bf16 = A.beta_dtype == TTC_DTYPE_BF16;
  P.normalize = A.normalize != 0;
  const int vec = bf16 ? 8 : 4;
  auto wide = [&](const Side& x, int64_t dim) {
    return dim % vec == 0 && aligned16(x.p) && x.sb % vec == 0 && x.st % vec == 0 && x.sh % vec == 0 && x.st >= dim &&
           x.st < (1 << 22);  // rows that do not overlap, a chunk's within 2^30 bytes
  };
  P.wide_q = wide(q, A.dk), P.wide_k = wide(k, A.dk), P.wide_v = wide(v, A.dv);
  P.wide_o = A.dv % 4 == 0 && aligned16(A.o) && A.heads * A.dv < (1 << 22);
  P.kd = (int)A.dk, P.vd = (int)A.dv, P.vdp = W.vdp, P.H = (int)A.heads;
  P.B = A.batch, P.T = A.tokens, P.chunks = W.chunks;
  P.scale = (float)A.scale, P.eps = (float)A.eps;
  char *ws = static_cast<char*>(A.workspace), *kept = A.saved ? static_cast<char*>(A.saved) : ws;
  auto floats = [](char* p, int64_t at) { return reinterpret_cast<float*>(p + at); };
  P.inverse = kept + W.inverse, P.scores = kept + W.scores, P.rows = floats(kept, W.rows);
  P.odd = reinterpret_cast<int*>(kept + W.odd);
  P.segs = W.segs, P.seg_chunks = W.seg_chunks;
  P.seg_matrix = floats(kept, W.seg_matrix), P.seg_state = floats(ws, W.seg_state);
  P.seg_dead = reinterpret_cast<int*>(kept + W.seg_dead);
  if (A.saved) P.S = floats(kept, W.S), P.E = floats(kept, W.E);
  int rc = TTC_LQR_OK;
  if (!A.backward) {
    P.state_in = A.initial_state, P.state_out = A.final_state;
    P.o = A.o;
    if ((rc = launch_delta_any(P, bf16, PREPARE, s))) return rc;
    return launch_delta_any(P, bf16, SWEEP, s);
  }
  P.d_o = side_of(A.d_o, A.d_o_stride, A.heads, A.heads);
  P.wide_d = wide(P.d_o, A.dv);
  P.state_in = A.d_final_state, P.state_out = A.d_initial_state;
  P.R = floats(ws, W.R), P.dV = floats(ws, W.dV);
  if ((rc = launch_delta_any(P, bf16, SWEEP_BACK, s))) return rc;
  const bool dq_shared = A.heads != A.q_heads, dk_shared = A.heads != A.k_heads, dv_shared = A.heads != A.v_heads;
  P.dq = !A.dq ? nullptr : dq_shared ? floats(ws, W.dq) : A.dq;
  P.dk = !A.dk_out ? nullptr : dk_shared ? floats(ws, W.dk) : A.dk_out;
  P.dv = dv_shared ? nullptr : A.dv_out;
  P.dq_f32 = dq_shared || !bf16, P.dk_f32 = dk_shared || !bf16;
  P.wide_dqk = A.dk % 4 == 0 && aligned16(P.dq) && aligned16(P.dk), P.wide_dv = A.dv % 8 == 0 && aligned16(P.dv);
  P.dgamma = A.d_log_gamma, P.dbeta = A.d_beta;
  if ((P.dq || P.dk || P.dv || P.dgamma || P.dbeta) && (rc = launch_delta_any(P, bf16, GRADIENTS, s))) return rc;
  const int64_t all = A.heads * A.dk, C = chunk_tokens(bf16), rows = W.chunks * C;
  if (A.dq && dq_shared && (rc = head_sum(floats(ws, W.dq), A.dq, bf16, A, A.q_heads, A.dk, A.tokens * all, all, A.dk, s)))
    return rc;
  if (A.dk_out && dk_shared && (rc = head_sum(floats(ws, W.dk), A.dk_out, bf16, A, A.k_heads, A.dk, A.tokens * all, all, A.dk, s)))
    return rc;
  if (A.dv_out && dv_shared)
    rc = head_sum(floats(ws, W.dV), A.dv_out, bf16, A, A.v_heads, A.dv, A.heads * rows * W.vdp, W.vdp, rows * W.vdp, s);
  return rc;
}

extern "C" int ttc_delta_rule_step(const ttc_delta_rule_step_args* args, void* stream) {
  using namespace ttc;
  if (!args) return TTC_LQR_EINVAL;
  const ttc_delta_rule_step_args& A = *args;
  if (const int rc = delta_check(A.dtype, A.gamma_dtype, A.beta_dtype, {A.batch, A.heads, MAX_DIM, MAX_DIM}, A.heads, A.q_heads,
                                 A.k_heads, A.v_heads, A.dk, A.dv))
    return rc;
  if (A.slots < 0 || !countable({A.slots, A.heads, MAX_DIM, MAX_DIM}) || (!A.slot_index && A.slots != A.batch) || !(A.eps >= 0))
    return TTC_LQR_EINVAL;
  if (A.batch == 0) return TTC_LQR_OK;
  if (!A.q || !A.k || !A.v || !A.log_gamma || !A.beta || !A.o || (A.slots > 0 && !A.state)) return TTC_LQR_EINVAL;
  auto side = [&](const void* p, const int64_t* st, int64_t own) { return Side{p, st[0], 0, st[1], (int)(A.heads / own)}; };
  Tokens P{};
  P.q = side(A.q, A.q_stride, A.q_heads);
  P.k = side(A.k, A.k_stride, A.k_heads);
  P.v = side(A.v, A.v_stride, A.v_heads);
  P.gamma = A.log_gamma, P.beta = A.beta;
  P.gb = A.gamma_stride[0], P.gh = A.gamma_stride[1];
  P.bb = A.beta_stride[0], P.bh = A.beta_stride[1];
  P.B = A.batch, P.T = 1, P.nslots = A.slots, P.H = (int)A.heads;
  P.gamma_bf16 = A.gamma_dtype == TTC_DTYPE_BF16, P.beta_bf16 = A.beta_dtype == TTC_DTYPE_BF16;
  P.normalize = A.normalize != 0;
  P.kd = (int)A.dk, P.vd = (int)A.dv;
  P.scale = (float)A.scale, P.eps = (float)A.eps;
  P.state_in = P.state_out = A.state;
  P.slots = A.slot_index;
  P.o = A.o;
  return launch_tokens(P, A.dtype == TTC_DTYPE_BF16, reinterpret_cast<hipStream_t>(stream));
}
