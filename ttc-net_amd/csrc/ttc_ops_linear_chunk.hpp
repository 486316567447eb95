// ttc_ops_linear_chunk.hpp -- the chunked sweep of linear attention on the matrix cores (roles: ttc_ops_linear.hpp).
//
// For a chunk of C tokens with G_t the sum of its decays up to token t and S the state in front of it,
//   o_t = e^{G_t} S' q_t + sum_{s <= t} e^{G_t - G_s} (q_t . k_s) v_s
//   S  <- e^{G_C} S + sum_s e^{G_C - G_s} k_s v_s'
// A workgroup walks down the chunks of one head (or of a segment of its tokens); its waves hold the state's columns
// between them in registers, so that it is never written in between.  Products are 16x16x32 bf16 or 16x16x4 fp32 matrix
// instructions.  The layouts are chosen so that no accumulator has to move before it is an operand:
//   P' = K Q'   lane: token t, 4 neighbouring s     -> shared memory, 4 neighbours at once
//   O' = V' P + S' Q'   lane: token t, 4 neighbouring columns -> stored 4 at once; S as it lies in the accumulators is
//        the operand (rows 4 g + i and 16 + 4 g + i of 32 are the 8 a lane gives, on the other side too)
//   S += K' (w V)   K' and V' by transposing reads of shared memory (bf16) or element by element (fp32).
//
// Numerics.  The sums G are held in 64 bits while they are formed and as pairs of fp32 after, so that differences of
// large sums keep their digits; a decay of 0 is 2^-4096.  In bf16, w V is split into three bf16 parts (exact in fp32's 24
// digits), so the state has fp32's accuracy; P and the state's copy in front of a chunk are rounded to bf16 for a bf16
// output (FAST), and split into three parts too where the sum feeds the decays' gradient (EXACT), a long sum of
// cancelling terms.  Weights that are 0 select: what is masked has no effect, whatever it holds.  Where a chunk's keys or
// values are not all finite, its sums over tokens are formed term by term instead, without the masked ones.
#pragma once
#include "ttc_ops_linear.hpp"

namespace ttc {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;

// ---- operands: 8 values a lane, row or column lane % 16, contraction index 8 (lane / 16) + j ------------------

template <class T>
struct Operand;

template <>
struct Operand<__bf16> {
  using Frag = bf16x8;
  struct Wide {  // a value as the exact sum of three bf16 numbers
    Frag h, m, l;
  };
  static constexpr int CHUNK = 64, PAD = 8;  // chunk_tokens()
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(const Wide& a, Frag b, f32x4 c) {
    return mma(a.h, b, mma(a.m, b, mma(a.l, b, c)));
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, const Wide& b, f32x4 c) {
    return mma(a, b.h, mma(a, b.m, mma(a, b.l, c)));
  }
  static __device__ __forceinline__ Frag row(const __bf16* p) { return *reinterpret_cast<const Frag*>(p); }
  // elements p[0..3] and p[16..19]
  static __device__ __forceinline__ Frag row_split(const __bf16* p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // column col0 + lane % 16, rows 8 (lane / 16) .. + 7 of the 32 from p's row on.  A transposing read gives each lane of 16
  // one column of 4 rows, whose 16 columns lie in 4 lanes' 8 bytes a row.
  static __device__ __forceinline__ Frag column(const __bf16* p, int stride, int col0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    const __bf16* a = p + (8 * g + (i >> 2)) * stride + col0 + (i & 3) * 4;
    typedef __attribute__((address_space(3))) i16x4 lds;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a));
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a + 4 * stride));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ Frag narrow(const float (&x)[8]) {
    Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (__bf16)x[j];
    return r;
  }
  static __device__ __forceinline__ Wide wide(const float (&x)[8]) {
    u32x4 h, m, l;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[2], b[2], c[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float v = x[2 * j + k];
        a[k] = __float_as_uint(v) & 0xffff0000u;
        const float r = v - __uint_as_float(a[k]);
        b[k] = __float_as_uint(r) & 0xffff0000u;
        c[k] = __float_as_uint(r - __uint_as_float(b[k]));
      }
      h[j] = __builtin_amdgcn_perm(a[1], a[0], 0x07060302);
      m[j] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302);
      l[j] = __builtin_amdgcn_perm(c[1], c[0], 0x07060302);
    }
    return Wide{__builtin_bit_cast(Frag, h), __builtin_bit_cast(Frag, m), __builtin_bit_cast(Frag, l)};
  }
  static __device__ __forceinline__ void values(Frag f, float (&x)[8]) {
    const u32x4 u = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(u[j] << 16);
      x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  }
  // the largest magnitude's bits of 16 bytes, joined to m (two 16-bit halves)
  static __device__ __forceinline__ void largest(u32x4 v, uint32_t& m) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, v[j] & 0x7fff7fffu),
                                                                 __builtin_bit_cast(u16x2, m)));
  }
  static __device__ __forceinline__ bool finite(uint32_t m) { return (m & 0xffffu) < 0x7f80u && (m >> 16) < 0x7f80u; }
};

template <>
struct Operand<float> {
  struct Frag {
    float v[8];
  };
  using Wide = Frag;
  static constexpr int CHUNK = 32, PAD = 4;  // chunk_tokens()
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag two(const float* p, const float* q) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(q);
    return Frag{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  static __device__ __forceinline__ Frag row(const float* p) { return two(p, p + 4); }
  static __device__ __forceinline__ Frag row_split(const float* p) { return two(p, p + 16); }
  static __device__ __forceinline__ Frag column(const float* p, int stride, int col0, int lane) {
    const float* a = p + 8 * (lane >> 4) * stride + col0 + (lane & 15);
    Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = a[j * stride];
    return r;
  }
  static __device__ __forceinline__ Frag narrow(const float (&x)[8]) { return wide(x); }
  static __device__ __forceinline__ Frag wide(const float (&x)[8]) {
    Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = x[j];
    return r;
  }
  static __device__ __forceinline__ void values(const Frag& f, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = f.v[j];
  }
  static __device__ __forceinline__ void largest(u32x4 v, uint32_t& m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = v[j] & 0x7fffffffu;
      m = a > m ? a : m;
    }
  }
  static __device__ __forceinline__ bool finite(uint32_t m) { return m < 0x7f800000u; }
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// a product with a decay that may be 0: what is dropped has no effect, whatever it holds
__device__ __forceinline__ float kept(float w, float x) { return w == 0.0f ? 0.0f : w * x; }

template <class T, int KD, int VD>
struct ChunkShape {
  static constexpr int WAVES = VD == 32 ? 2 : 4, NT = WAVES * 64, VW = VD / WAVES, ET = VW / 16;
  static constexpr int C = Operand<T>::CHUNK, TT = C / 16, KB = C / 32, DB = KD / 32, DT = KD / 16;
  static constexpr int VEC = 16 / sizeof(T), QS = KD + Operand<T>::PAD, VS = VD + Operand<T>::PAD;
  static constexpr int KV = C * KD / VEC / NT, VV = C * VD / VEC / NT;  // 16-byte loads a thread
};

// 16 bytes of a row from element c on, zero beyond `dim`
template <class T>
__device__ __forceinline__ u32x4 load16(const T* p, int c, int dim, bool wide) {
  constexpr int VEC = 16 / sizeof(T);
  u32x4 r = {0, 0, 0, 0};
  if (wide) {
    if (c < dim) r = *reinterpret_cast<const u32x4*>(p + c);
  } else {
    T e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = c + j < dim ? p[c + j] : from_f<T>(0.0f);
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

template <class T, int KD, int VD, int MODE>
__global__ __launch_bounds__((ChunkShape<T, KD, VD>::NT), 2) void chunk_sweep_kernel(Sweep A, Segments G, Wides W) {
  using Z = ChunkShape<T, KD, VD>;
  using Op = Operand<T>;
  using PT = std::conditional_t<MODE == EXACT, float, T>;  // the weighted scores in shared memory
  constexpr int C = Z::C, NT = Z::NT, VEC = Z::VEC, QS = Z::QS, VS = Z::VS, PS = C + 16 / (int)sizeof(PT);
  __shared__ __attribute__((aligned(16))) T Qs[MODE == STATE_ONLY ? 1 : C * QS];
  __shared__ __attribute__((aligned(16))) T Ks[C * QS];
  __shared__ __attribute__((aligned(16))) T Vs[C * VS];
  __shared__ __attribute__((aligned(16))) PT Ps[MODE == STATE_ONLY ? 1 : C * PS];
  __shared__ __attribute__((aligned(16))) float Hi[2][C], Lo[2][C], In[2][C], Up[2][C];
  __shared__ float Whole[2], Dot[MODE == EXACT || sizeof(T) == 4 ? Z::WAVES : 1][C];
  __shared__ int Odd[Z::WAVES];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, n = lane & 15;
  const int segs = MODE == STATE_ONLY ? G.count - 1 : G.count;  // the last one's own contribution is not needed
  const int seg = (int)(blockIdx.x % segs);
  const int64_t bh = blockIdx.x / segs, b = bh / A.H;
  const int h = (int)(bh % A.H);
  const T *q = MODE == STATE_ONLY ? nullptr : A.q.at<T>(b, h), *k = A.k.at<T>(b, h), *v = A.v.at<T>(b, h);
  const int64_t gbase = b * A.gb + h * A.gh;
  const int64_t u0 = seg * G.chunks * C;  // tokens in the sweep's order
  const int64_t u1 = u0 + G.chunks * C < A.T ? u0 + G.chunks * C : A.T;
  const int e0 = wave * Z::VW;

  f32x4 S[Z::DT][Z::ET];
  {
    const float* p = nullptr;
    int sr = A.sr, sc = A.sc;
    if (MODE != STATE_ONLY) {
      if (G.count > 1) {
        p = G.state + (bh * G.count + seg) * (int64_t)A.kd * A.vd;
        sr = A.vd, sc = 1;
      } else if (A.state_in) {
        p = A.state_in + bh * (int64_t)A.kd * A.vd;
      }
    }
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * d + 4 * g + i, c = e0 + 16 * e + n;
          S[d][e][i] = p && r < A.kd && c < A.vd ? p[(int64_t)r * sr + (int64_t)c * sc] : 0.0f;
        }
  }

  u32x4 qr[Z::KV], kr[Z::KV], vr[Z::VV];
  auto token = [&](int64_t u) { return A.reverse ? A.T - 1 - u : u; };
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int j = 0; j < Z::KV; ++j) {
      const int i = tid + j * NT, row = i / (KD / VEC), c = i % (KD / VEC) * VEC;
      const u32x4 zero = {0, 0, 0, 0};
      const bool in = at + row < u1;
      const int64_t t = token(at + row);
      kr[j] = in ? load16(k + t * A.k.st, c, A.kd, W.k) : zero;
      if (MODE != STATE_ONLY) qr[j] = in ? load16(q + t * A.q.st, c, A.kd, W.q) : zero;
    }
#pragma unroll
    for (int j = 0; j < Z::VV; ++j) {
      const int i = tid + j * NT, row = i / (VD / VEC), c = i % (VD / VEC) * VEC;
      const u32x4 zero = {0, 0, 0, 0};
      vr[j] = at + row < u1 ? load16(v + token(at + row) * A.v.st, c, A.vd, W.v) : zero;
    }
  };
  // wave 0: the chunk's decays.  Tokens beyond the end have none.
  auto gate_of = [&](int64_t u) {
    if (lane >= C || u >= u1 || (A.reverse && u == 0)) return 0.0f;
    return gamma_at(A, gbase + (A.reverse ? A.T - u : u) * A.gt);
  };
  auto gates = [&](float lg, int buf) {
    double x = (double)lg * 1.4426950408889634;
    x = x < -4096.0 ? -4096.0 : x;
#pragma unroll
    for (int m = 1; m < C; m <<= 1) {
      const double y = __shfl_up(x, m, 64);
      if (lane >= m) x += y;
    }
    const double all = __shfl(x, C - 1, 64), rest = all - x;
    if (lane < C) {
      const float hi = (float)x, lo = (float)(x - (double)hi), uh = (float)rest, ul = (float)(rest - (double)uh);
      Hi[buf][lane] = hi;
      Lo[buf][lane] = lo;
      const float in = exp2_of(hi) * exp2_of(lo);
      In[buf][lane] = in;
      Up[buf][lane] = exp2_of(uh) * exp2_of(ul) * A.key_scale;
      if (lane == C - 1) Whole[buf] = in;
    }
  };

  fetch(u0);
  if (wave == 0) gates(gate_of(u0 + lane), 0);
  float whole_decay = 1.0f;
  int buf = 0;
  int64_t dot_at = -1;
  auto put_dots = [&]() {  // of the chunk before, after a barrier
    if constexpr (MODE == EXACT || sizeof(T) == 4) {
      if (A.x.p != nullptr && dot_at >= 0 && tid < C && dot_at + tid < u1) {
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < Z::WAVES; ++w) d += Dot[w][tid];
        A.dots[bh * A.T + token(dot_at + tid)] = d;
      }
    }
  };

  for (int64_t at = u0; at < u1; at += C, buf ^= 1) {
    // the chunk's tokens to shared memory, and whether all keys and values are finite
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < Z::KV; ++j) {
      const int i = tid + j * NT, row = i / (KD / VEC), c = i % (KD / VEC) * VEC;
      Op::largest(kr[j], most);
      *reinterpret_cast<u32x4*>(&Ks[row * QS + c]) = kr[j];
      if (MODE != STATE_ONLY) *reinterpret_cast<u32x4*>(&Qs[row * QS + c]) = qr[j];
    }
#pragma unroll
    for (int j = 0; j < Z::VV; ++j) {
      const int i = tid + j * NT, row = i / (VD / VEC), c = i % (VD / VEC) * VEC;
      Op::largest(vr[j], most);
      *reinterpret_cast<u32x4*>(&Vs[row * VS + c]) = vr[j];
    }
    const bool odd_here = __ballot(!Op::finite(most)) != 0;
    if (lane == 0) Odd[wave] = odd_here;
    __syncthreads();
    put_dots();
    bool odd = false;
#pragma unroll
    for (int w = 0; w < Z::WAVES; ++w) odd = odd || Odd[w];
    if (at + C < u1) fetch(at + C);
    const float next_gate = wave == 0 ? gate_of(at + C + lane) : 0.0f;
    const float whole = Whole[buf];

    f32x4 O[Z::TT][Z::ET];
    if constexpr (MODE != STATE_ONLY) {
      // scores, tile by tile over the waves: (ti, si <= ti), and zeros where a later product's 32 tokens reach past ti
      int turn = 0;
#pragma unroll
      for (int ti = 0; ti < Z::TT; ++ti)
#pragma unroll
        for (int si = 0; si <= (ti | 1); ++si, ++turn) {
          if (turn % Z::WAVES != wave) continue;
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
          if (si <= ti) {
#pragma unroll
            for (int d = 0; d < Z::DB; ++d)
              p = Op::mma(Op::row(&Ks[(16 * si + n) * QS + 32 * d + 8 * g]), Op::row(&Qs[(16 * ti + n) * QS + 32 * d + 8 * g]),
                          p);
            const float th = Hi[buf][16 * ti + n], tl = Lo[buf][16 * ti + n];
            const f32x4 sh = *reinterpret_cast<const f32x4*>(&Hi[buf][16 * si + 4 * g]),
                        sl = *reinterpret_cast<const f32x4*>(&Lo[buf][16 * si + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = exp2_of((th - sh[i]) + (tl - sl[i])) * A.key_scale;
              p[i] = si < ti || 4 * g + i <= n ? kept(w, p[i]) : 0.0f;
            }
          }
          struct alignas(4 * sizeof(PT)) Four { PT v[4]; };
          Four f;
#pragma unroll
          for (int i = 0; i < 4; ++i) f.v[i] = from_f<PT>(p[i]);
          *reinterpret_cast<Four*>(&Ps[(16 * ti + n) * PS + 16 * si + 4 * g]) = f;
        }
      // the state's part
#pragma unroll
      for (int t = 0; t < Z::TT; ++t)
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) O[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < Z::DB; ++d) {
        using Given = std::conditional_t<MODE == EXACT, typename Op::Wide, typename Op::Frag>;
        Given s[Z::ET];
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = S[2 * d][e][i], x[4 + i] = S[2 * d + 1][e][i];
          if constexpr (MODE == EXACT) s[e] = Op::wide(x); else s[e] = Op::narrow(x);
        }
#pragma unroll
        for (int t = 0; t < Z::TT; ++t) {
          const typename Op::Frag f = Op::row_split(&Qs[(16 * t + n) * QS + 32 * d + 4 * g]);
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) O[t][e] = Op::mma(s[e], f, O[t][e]);
        }
      }
#pragma unroll
      for (int t = 0; t < Z::TT; ++t) {
        const float w = In[buf][16 * t + n];
#pragma unroll
        for (int e = 0; e < Z::ET; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[t][e][i] = kept(w, O[t][e][i]);
      }
      __syncthreads();
    }

    typename Op::Frag vf[Z::KB][Z::ET];
#pragma unroll
    for (int s = 0; s < Z::KB; ++s)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e) vf[s][e] = Op::column(&Vs[32 * s * VS], VS, e0 + 16 * e, lane);

    if constexpr (MODE != STATE_ONLY) {
      if (!odd) {
#pragma unroll
        for (int t = 0; t < Z::TT; ++t)
#pragma unroll
          for (int s = 0; s <= t / 2; ++s) {
            if constexpr (MODE == EXACT) {
              float x[8];
              Operand<float>::values(Operand<float>::row(&Ps[(16 * t + n) * PS + 32 * s + 8 * g]), x);
              const auto p = Op::wide(x);
#pragma unroll
              for (int e = 0; e < Z::ET; ++e) O[t][e] = Op::mma(vf[s][e], p, O[t][e]);
            } else {
              const typename Op::Frag p = Op::row(&Ps[(16 * t + n) * PS + 32 * s + 8 * g]);
#pragma unroll
              for (int e = 0; e < Z::ET; ++e) O[t][e] = Op::mma(vf[s][e], p, O[t][e]);
            }
          }
      } else {
#pragma unroll
        for (int t = 0; t < Z::TT; ++t) {
          const int tt = 16 * t + n;
          for (int s = 0; s < C; ++s) {
            const float w = exp2_of((Hi[buf][tt] - Hi[buf][s]) + (Lo[buf][tt] - Lo[buf][s]));
            if (s > tt || w == 0.0f) continue;
            const float p = to_f(Ps[tt * PS + s]);
#pragma unroll
            for (int e = 0; e < Z::ET; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) O[t][e][i] = fmaf(p, to_f(Vs[s * VS + e0 + 16 * e + 4 * g + i]), O[t][e][i]);
          }
        }
      }
      // out: a lane holds 4 neighbouring columns of one token
      const bool dots = (MODE == EXACT || sizeof(T) == 4) && A.x.p != nullptr;
#pragma unroll
      for (int t = 0; t < Z::TT; ++t) {
        const int64_t u = at + 16 * t + n;
        const int64_t tok = token(u);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          const int c = e0 + 16 * e + 4 * g;
          const int64_t o = ((b * A.T + tok) * A.H + h) * A.vd + c;
          f32x4 r = O[t][e];
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] *= A.out_scale;
          if (u < u1) {
            if (A.out == nullptr) {
            } else if (A.out_f32) {
              float* y = static_cast<float*>(A.out) + o;
              if (W.out) {
                if (c < A.vd) *reinterpret_cast<f32x4*>(y) = r;
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (c + i < A.vd) y[i] = r[i];
              }
            } else {
              T* y = static_cast<T*>(A.out) + o;
              struct alignas(4 * sizeof(T)) Four { T v[4]; };
              Four f;
#pragma unroll
              for (int i = 0; i < 4; ++i) f.v[i] = from_f<T>(r[i]);
              if (W.out) {
                if (c < A.vd) *reinterpret_cast<Four*>(y) = f;
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (c + i < A.vd) y[i] = f.v[i];
              }
            }
            if (dots) {
              const T* x = A.x.at<T>(b, h) + tok * A.x.st + c;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (c + i < A.vd) dot = fmaf(r[i], to_f(x[i]), dot);
            }
          }
        }
        if constexpr (MODE == EXACT || sizeof(T) == 4) {
          if (dots) {
            dot += __shfl_xor(dot, 16, 64);
            dot += __shfl_xor(dot, 32, 64);
            if (g == 0) Dot[wave][16 * t + n] = dot;
          }
        }
      }
      dot_at = at;
    }

    // the state behind the chunk
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[d][e][i] = kept(whole, S[d][e][i]);
    whole_decay *= whole;
    if (!odd) {
#pragma unroll
      for (int s = 0; s < Z::KB; ++s) {
        const f32x4 wa = *reinterpret_cast<const f32x4*>(&Up[buf][32 * s + 8 * g]),
                    wb = *reinterpret_cast<const f32x4*>(&Up[buf][32 * s + 8 * g + 4]);
        typename Op::Wide wv[Z::ET];
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          float x[8];
          Op::values(vf[s][e], x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= j < 4 ? wa[j] : wb[j - 4];
          wv[e] = Op::wide(x);
        }
#pragma unroll
        for (int d = 0; d < Z::DT; ++d) {
          const typename Op::Frag f = Op::column(&Ks[32 * s * QS], QS, 16 * d, lane);
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) S[d][e] = Op::mma(f, wv[e], S[d][e]);
        }
      }
    } else {
      for (int s = 0; s < C; ++s) {
        const float w = Up[buf][s];
        if (w == 0.0f) continue;
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          const float x = w * to_f(Vs[s * VS + e0 + 16 * e + n]);
#pragma unroll
          for (int d = 0; d < Z::DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[d][e][i] = fmaf(to_f(Ks[s * QS + 16 * d + 4 * g + i]), x, S[d][e][i]);
        }
      }
    }
    if (wave == 0 && at + C < u1) gates(next_gate, buf ^ 1);
    __syncthreads();
  }
  put_dots();

  float* p = nullptr;
  int sr = A.sr, sc = A.sc;
  if (MODE == STATE_ONLY) {
    p = G.state + (bh * G.count + seg) * (int64_t)A.kd * A.vd;
    sr = A.vd, sc = 1;
    if (tid == 0) G.decay[bh * G.count + seg] = whole_decay;
  } else if (A.state_out && seg == G.count - 1) {
    p = A.state_out + bh * (int64_t)A.kd * A.vd;
    if (A.reverse && A.T > 0) {
      const float lg = gamma_at(A, gbase), last = lg < RESET ? 0.0f : expf(lg);
#pragma unroll
      for (int d = 0; d < Z::DT; ++d)
#pragma unroll
        for (int e = 0; e < Z::ET; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) S[d][e][i] = kept(last, S[d][e][i]);
    }
  }
  if (p) {
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * d + 4 * g + i, c = e0 + 16 * e + n;
          if (r < A.kd && c < A.vd) p[(int64_t)r * sr + (int64_t)c * sc] = S[d][e][i];
        }
  }
}

template <class T, int KD, int VD>
int launch_chunk(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s) {
  using Z = ChunkShape<T, KD, VD>;
  const int64_t blocks = A.B * A.H * (mode == STATE_ONLY ? G.count - 1 : G.count);
  if (blocks > MAX_GRID) return TTC_LQR_EINVAL;
  const dim3 grid((unsigned)blocks), block(Z::NT);
  if (mode == STATE_ONLY)
    hipLaunchKernelGGL((chunk_sweep_kernel<T, KD, VD, STATE_ONLY>), grid, block, 0, s, A, G, W);
  else if (mode == FAST || sizeof(T) == 4)  // fp32 products are exact enough as they are
    hipLaunchKernelGGL((chunk_sweep_kernel<T, KD, VD, FAST>), grid, block, 0, s, A, G, W);
  else
    hipLaunchKernelGGL((chunk_sweep_kernel<T, KD, VD, sizeof(T) == 4 ? FAST : EXACT>), grid, block, 0, s, A, G, W);
  return launched();
}

}  // namespace ttc

#define TTC_CHUNK_UNIT(T, KD)                                                                                        \
  namespace ttc {                                                                                                    \
  template <>                                                                                                        \
  int launch_chunk_kd##KD<T>(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s) {           \
    return A.vd <= 32   ? launch_chunk<T, KD, 32>(A, G, W, mode, s)                                                  \
           : A.vd <= 64 ? launch_chunk<T, KD, 64>(A, G, W, mode, s)                                                  \
                        : launch_chunk<T, KD, 128>(A, G, W, mode, s);                                                \
  }                                                                                                                  \
  }
