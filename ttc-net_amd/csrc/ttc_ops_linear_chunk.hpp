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
// Bound.  No unit is full: the phases between two barriers do not cover each other.  Of a sweep's cycles
//                                                    vector ALU  matrix cores  shared memory (its bank conflicts)  us
//   64 x 64, 2,048 x 128 heads in 768 parts, FAST        45 %         12 %          29 % (9)    59 MB read, 34 written  50
//   the same, EXACT (a fourth input)                     39           12            29 (9)      76, 36                  62
//   the same, STATE_ONLY                                 34            8            10 (0)      35, 11                  25
//   128 x 128, 16,381 x 16 heads in 512 parts, FAST      43           22            23 (7)      118, 68                102
//   the same, STATE_ONLY                                 42           20            10 (0)      69, 33                  52
// (read and written: as counted behind the XCDs' caches, less than the inputs where the last level holds some).  At 64 x 64
// three workgroups share a CU; at 128 x 128 registers leave two (a wave holds 32 columns of the state, 64 registers), and
// EXACT spills 18 of them.  16 columns a wave need twice the operand reads (2,048 tokens x 512 heads, with scores of 8
// digits: 360 us, with 32 columns 313).  2,048 tokens x 512 heads of 128 that fill the GPU unsplit: 372 us.  fp32 is bound by
// its matrix instructions: the same in 806 us, 104 TFLOP/s (a large library product: 153).
//
// Numerics.  The sums G are held in 64 bits while they are formed and as pairs of fp32 after, so that differences of
// large sums keep their digits; they start anew at a reset.  In bf16, w V is split into three bf16 parts (exact in fp32's 24
// digits), so the state has fp32's accuracy; P, and in FAST the state's copy in front of a chunk, into two (16 digits), so that
// a bf16 output is rounded to 8 digits once.  (Both in one part of 8 digits: the call on 16,381 x 16 heads of 128 takes 143 us,
// so 154, 2,048 tokens x 512 heads of 128 313, so 372, training on 4 x 2,048 tokens x 32 heads of 64 264, so 277, and the
// outputs' error is 2.35e-3 of their norm instead of 1.66e-3.)  The decays' gradient is a long sum of cancelling terms, so the
// dots x . o it is made of are not taken from such an o (EXACT): P's part is sum_s P_ts (v_s . x_t), whose products are exact
// as they are, in fp32; the state's copy is split into three parts.  Weights that are 0 select: what is masked has no effect,
// whatever it holds.  Where a chunk's keys or values are not all finite, its sums over tokens are formed term by term instead,
// without the masked ones.
#pragma once
#include "ttc_ops_linear.hpp"

namespace ttc {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;

// ---- operands: 8 values a lane, row or column lane % 16; which of the 32 contracted indices a lane holds is free as long
// as both sides agree: 8 g + j (row), or 4 g + j and 16 + 4 g + j (row_split, column, accumulators), g = lane / 16

template <class T>
struct Operand;

template <>
struct Operand<__bf16> {
  using Frag = bf16x8;
  struct Wide {  // a value as the exact sum of three bf16 numbers
    Frag h, m, l;
  };
  struct Pair {  // its first 16 digits as the sum of two
    Frag h, l;
  };
  // rows read along them: 4 banks apart (mod 32); rows read across them, 8 rows at once, 8 banks apart
  static constexpr int ROW_PAD = 8, COL_PAD = 16;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(const Wide& a, Frag b, f32x4 c) {
    return mma(a.h, b, mma(a.m, b, mma(a.l, b, c)));
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, const Wide& b, f32x4 c) {
    return mma(a, b.h, mma(a, b.m, mma(a, b.l, c)));
  }
  static __device__ __forceinline__ f32x4 mma(const Pair& a, Frag b, f32x4 c) { return mma(a.h, b, mma(a.l, b, c)); }
  static __device__ __forceinline__ f32x4 mma(Frag a, const Pair& b, f32x4 c) { return mma(a, b.h, mma(a, b.l, c)); }
  static __device__ __forceinline__ Frag row(const __bf16* p) { return *reinterpret_cast<const Frag*>(p); }
  // elements p[0..3] and p[16..19]
  static __device__ __forceinline__ Frag row_split(const __bf16* p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // column col0 + lane % 16, rows 4 g .. + 3 and 16 + 4 g .. + 3 of the 32 from p's row on (g = lane / 16).  A transposing
  // read gives each lane of 16 one column of 4 rows, whose 16 columns lie in 4 lanes' 8 bytes a row.
  static __device__ __forceinline__ Frag column(const __bf16* p, int stride, int col0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    const __bf16* a = p + (4 * g + (i >> 2)) * stride + col0 + (i & 3) * 4;
    typedef __attribute__((address_space(3))) i16x4 lds;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a));
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a + 16 * stride));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // two values cut to bf16, and what that leaves of each
  static __device__ __forceinline__ uint32_t cut(float x, float y, float& dx, float& dy) {
    const uint32_t a = __float_as_uint(x) & 0xffff0000u, b = __float_as_uint(y) & 0xffff0000u;
    dx = x - __uint_as_float(a);
    dy = y - __uint_as_float(b);
    return __builtin_amdgcn_perm(b, a, 0x07060302);
  }
  static __device__ __forceinline__ Pair pair(const float (&x)[8]) {
    u32x4 h;
    Frag l;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float d, e;
      h[j] = cut(x[2 * j], x[2 * j + 1], d, e);
      l[2 * j] = (__bf16)d;
      l[2 * j + 1] = (__bf16)e;
    }
    return Pair{__builtin_bit_cast(Frag, h), l};
  }
  // Scores in tiles of 16 x 16 (SCORE_PARTS such arrays, `part` elements apart): 4 neighbours of a row at p, and those of
  // two neighbouring tiles as an operand (zeros for the second one where there is none)
  static constexpr int SCORE_PARTS = 2;
  static __device__ __forceinline__ void put_scores(__bf16* p, int part, f32x4 x) {
    float d[4];
    const u32x2 h = {cut(x[0], x[1], d[0], d[1]), cut(x[2], x[3], d[2], d[3])};
    *reinterpret_cast<u32x2*>(p) = h;
    *reinterpret_cast<bf16x4*>(p + part) = bf16x4{(__bf16)d[0], (__bf16)d[1], (__bf16)d[2], (__bf16)d[3]};
  }
  static __device__ __forceinline__ Pair scores(const __bf16* p, int part, bool second) {
    auto both = [&](const __bf16* q) {
      const bf16x4 a = *reinterpret_cast<const bf16x4*>(q);
      const bf16x4 b = second ? *reinterpret_cast<const bf16x4*>(q + 256) : bf16x4{};
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    return Pair{both(p), both(p + part)};
  }
  static __device__ __forceinline__ float score(const __bf16* p, int part) { return to_f(p[0]) + to_f(p[part]); }
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
  using Pair = Frag;
  static constexpr int ROW_PAD = 4, COL_PAD = 4;
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
    const float* a = p + 4 * (lane >> 4) * stride + col0 + (lane & 15);
    Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = a[(j < 4 ? j : 12 + j) * stride];
    return r;
  }
  static __device__ __forceinline__ Frag pair(const float (&x)[8]) { return wide(x); }
  static constexpr int SCORE_PARTS = 1;
  static __device__ __forceinline__ void put_scores(float* p, int, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }
  static __device__ __forceinline__ Frag scores(const float* p, int, bool second) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p),
                b = second ? *reinterpret_cast<const f32x4*>(p + 256) : f32x4{0.f, 0.f, 0.f, 0.f};
    return Frag{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  static __device__ __forceinline__ float score(const float* p, int) { return p[0]; }
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
  static constexpr int WAVES = sweep_waves(VD), NT = WAVES * 64, ET = VD / 16 / WAVES;  // a wave's columns: 16 ET
  static constexpr int C = chunk_tokens(sizeof(T) == 2), TT = C / 16, KB = C / 32, DB = KD / 32, DT = KD / 16, VB = VD / 32;
  static constexpr int VEC = 16 / sizeof(T), QS = KD + Operand<T>::ROW_PAD, KS = KD + Operand<T>::COL_PAD,
                       VS = VD + Operand<T>::COL_PAD;
  static constexpr int KV = (C * KD / VEC + NT - 1) / NT, VV = (C * VD / VEC + NT - 1) / NT;  // 16-byte loads a thread
};

// 16 bytes of a row from element c on, zero beyond `dim`, for rows of any alignment
template <class T>
__device__ __forceinline__ u32x4 load_any(const T* p, int c, int dim) {
  constexpr int VEC = 16 / sizeof(T);
  u32x4 r;
  T e[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) e[j] = c + j < dim ? p[c + j] : from_f<T>(0.0f);
  __builtin_memcpy(&r, e, 16);
  return r;
}

// `bytes` from p on, for loads that give 0 and stores that do nothing past the bound instead of branching: all loads of a
// chunk are in flight at once.  A chunk's offsets are below 2^30 bytes (the host sees to it).
constexpr int BEYOND = 0x7ffffff0;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bounded(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}

// WIDE: rows of 16-byte multiples at 16-byte addresses
template <class T, int KD, int VD, int MODE, bool WIDE>
__global__ __launch_bounds__((ChunkShape<T, KD, VD>::NT), 2) void chunk_sweep_kernel(Sweep A, Segments G, Wides W) {
  using Z = ChunkShape<T, KD, VD>;
  using Op = Operand<T>;
  // the dots x . o: from products of scores and of v . x (PAIRED), or from fp32's o as it is (DIRECT)
  constexpr bool PAIRED = MODE == EXACT, DIRECT = MODE == FAST && sizeof(T) == 4, DOTS = PAIRED || DIRECT;
  // With x there too, 128 x 128 stays below half of the 160 KB a CU has only if columns are padded as rows are, the last
  // rows end without a pad, and x has none: its rows' 16 bytes change places instead (x_at).
  constexpr bool TIGHT = PAIRED && KD + VD > 192;
  constexpr int C = Z::C, NT = Z::NT, VEC = Z::VEC, QS = Z::QS, XS = TIGHT ? VD : VD + Op::ROW_PAD, KS = TIGHT ? QS : Z::KS,
                VS = TIGHT ? VD + Op::ROW_PAD : Z::VS, TAIL = PAIRED ? 16 / (int)sizeof(T) : 0;
  constexpr int PART = Z::TT * (Z::TT + 1) / 2 * 256;  // the scores' tiles (ti, si <= ti)
  // The rows of 4 neighbours that are read or written at once lie in different banks (training on 4 x 2,048 tokens x 32
  // heads of 64: 277 us, in order 291); at 128 x 128 with x they are in order, which needs fewer registers (8 x 2,048 x 32
  // heads: 1,098 us and 18 spills, otherwise 1,135 and 24)
  auto score_at = [](int ti, int si, int row, int col) {
    return ((ti * (ti + 1) / 2 + si) * 16 + row) * 16 + (col ^ (row & (TIGHT ? 0 : sizeof(T) == 2 ? 8 : 12)));
  };
  auto x_at = [](int row, int c) { return row * XS + (TIGHT ? c ^ (row % 16 * VEC) : c); };
  __shared__ __attribute__((aligned(16))) T Qs[MODE == STATE_ONLY ? 1 : C * QS - TAIL];
  __shared__ __attribute__((aligned(16))) T Ks[C * KS - TAIL];
  __shared__ __attribute__((aligned(16))) T Vs[C * VS - TAIL];
  __shared__ __attribute__((aligned(16))) T Xs[PAIRED ? C * XS - (TIGHT ? 0 : TAIL) : 1];
  __shared__ __attribute__((aligned(16))) T Ps[MODE == STATE_ONLY ? 1 : Op::SCORE_PARTS * PART];  // the weighted scores
  __shared__ __attribute__((aligned(16))) float Hi[2][C], Lo[2][C], In[2][C], Up[2][C];
  __shared__ float Whole[2], Dot[DOTS ? Z::WAVES : 1][C];
  __shared__ int Odd[Z::WAVES];

  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int segs = MODE == STATE_ONLY ? G.count - 1 : G.count;  // the last one's own contribution is not needed
  const int seg = (int)(blockIdx.x % segs);
  const int64_t bh = A.first + blockIdx.x / segs, b = bh / A.H, elems = (int64_t)A.kd * A.vd;
  const int h = (int)(bh % A.H);
  const T *q = MODE == STATE_ONLY ? nullptr : A.q.at<T>(b, h), *k = A.k.at<T>(b, h), *v = A.v.at<T>(b, h);
  const T* x = DOTS && A.x.p ? A.x.at<T>(b, h) : nullptr;
  const int64_t gbase = b * A.gb + h * A.gh;
  // Places in the sweep's order: whole chunks, whose boundaries lie between the same tokens in both orders
  const int64_t places = (A.T + C - 1) / C * C, u0 = seg * G.chunks * C;
  const int64_t u1 = u0 + G.chunks * C < places ? u0 + G.chunks * C : places;
  const int e0 = wave * 16 * Z::ET;  // the wave's columns
  // A chunk holds tokens low .. low + left - 1 (left <= C: the last ones may be missing); the sweep's row r is its token
  // place(r)
  auto low_of = [&](int64_t at) { return A.reverse ? places - C - at : at; };
  auto left_of = [&](int64_t at) { return (int)(A.T - low_of(at) < C ? A.T - low_of(at) : C); };
  auto place = [&](int r) { return A.reverse ? C - 1 - r : r; };

  // S: lane's rows 16 d + 4 g + i, columns e0 + 16 e + n.  The lane's place is hidden from the compiler, which
  // would otherwise keep 32 addresses in registers over the whole loop.
  f32x4 S[Z::DT][Z::ET];
  auto each = [&](auto f) {
    int r = 4 * g, c = e0 + n;
    asm volatile("" : "+v"(r), "+v"(c));
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[d][e][i] = f((float)S[d][e][i], 16 * d + r + i, c + 16 * e);
  };
  // a state in memory (NULL: zero): loads and stores bounded, since those in branches would wait for each other
  auto state_of = [&](const float* p) { return bounded(p, p ? A.kd * A.vd * 4 : 0); };
  auto entry = [&](int r, int c, int sr, int sc) { return r < A.kd && c < A.vd ? (r * sr + c * sc) * 4 : BEYOND; };
  auto load_f = [&](__amdgpu_buffer_rsrc_t from, int off) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(from, off, 0, 0));
  };
  auto put_state = [&](float* p, int sr, int sc) {
    const auto to = state_of(p);
    each([&](float s, int r, int c) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s), to, entry(r, c, sr, sc), 0, 0);
      return s;
    });
  };
  {
    const float* p = nullptr;
    int sr = A.sr, sc = A.sc;
    if (MODE != STATE_ONLY) {
      if (G.count > 1) {
        p = G.state + (bh * G.count + seg) * elems;
        sr = G.sr, sc = G.sc;
      } else if (A.state_in) {
        p = A.state_in + bh * elems;
      }
    }
    const auto from = state_of(p);
    each([&](float, int r, int c) { return load_f(from, entry(r, c, sr, sc)); });
  }
  // <S, p>, the wave's part of it: the decays' gradient at a boundary
  auto meet = [&](const float* p, int sr, int sc, float w, int64_t mark) {
    float d = 0.0f;
    const auto from = state_of(p);
    each([&](float s, int r, int c) {
      d = fmaf(s, load_f(from, entry(r, c, sr, sc)), d);  // both are 0 where there is no row or column
      return s;
    });
    d = lane_sum(d, 64);
    if (lane == 0) A.joins[(bh * (A.marks + 1) + mark) * MAX_WAVES + wave] = kept(w, d);
  };
  if (DOTS && A.joins && A.reverse && seg == 0 && A.last) meet(A.last + bh * elems, A.sr, A.sc, 1.0f, A.marks);

  u32x4 qr[Z::KV], kr[Z::KV], vr[Z::VV], xr[Z::VV];
  int ko[Z::KV], qo[Z::KV], vo[Z::VV], xo[Z::VV];  // offsets of this thread's 16 bytes from the chunk's lowest address
  auto offsets = [&](int64_t st, int dim, auto& o, auto width) {
    constexpr int D = decltype(width)::value;
#pragma unroll
    for (int j = 0; j < (int)(sizeof(o) / sizeof(o[0])); ++j) {
      const int i = tid + j * NT, row = i / (D / VEC), c = i % (D / VEC) * VEC;
      o[j] = row < C && c < dim ? (place(row) * (int)st + c) * (int)sizeof(T) : BEYOND;
    }
  };
  if constexpr (WIDE) {
    offsets(A.k.st, A.kd, ko, std::integral_constant<int, KD>{});
    if constexpr (MODE != STATE_ONLY) offsets(A.q.st, A.kd, qo, std::integral_constant<int, KD>{});
    offsets(A.v.st, A.vd, vo, std::integral_constant<int, VD>{});
    if constexpr (PAIRED) offsets(A.x.st, A.vd, xo, std::integral_constant<int, VD>{});
  }
  auto fetch_side = [&](const T* p, int64_t st, int dim, int64_t at, auto& r, const auto& o, auto width) {
    constexpr int D = decltype(width)::value;
    const T* from = p + low_of(at) * st;
    const int left = left_of(at);
    const auto rows = bounded(from, left * (int)st * (int)sizeof(T));  // rows do not overlap: st >= dim
#pragma unroll
    for (int j = 0; j < (int)(sizeof(r) / sizeof(r[0])); ++j) {
      if constexpr (WIDE) {
        r[j] = __builtin_amdgcn_raw_buffer_load_b128(rows, o[j], 0, 0);
      } else {
        const int i = tid + j * NT, row = i / (D / VEC), c = i % (D / VEC) * VEC;
        const u32x4 zero = {0, 0, 0, 0};
        r[j] = row < C && place(row) < left ? load_any(from + place(row) * st, c, dim) : zero;
      }
    }
  };
  auto fetch = [&](int64_t at) {
    fetch_side(k, A.k.st, A.kd, at, kr, ko, std::integral_constant<int, KD>{});
    if constexpr (MODE != STATE_ONLY) fetch_side(q, A.q.st, A.kd, at, qr, qo, std::integral_constant<int, KD>{});
    fetch_side(v, A.v.st, A.vd, at, vr, vo, std::integral_constant<int, VD>{});
    if constexpr (PAIRED) fetch_side(x, A.x.st, A.vd, at, xr, xo, std::integral_constant<int, VD>{});
  };
  // One wave: a chunk's decays, one a lane (before a token in reverse order, that of the one after it), as they are stored
  constexpr int GATES = Z::WAVES - 1;
  auto gate_bits = [&](int64_t at) {
    const int r = place(lane) + (A.reverse ? 1 : 0);
    const int64_t t = low_of(at) + r;
    if (lane >= C || at >= u1 || t >= A.T) return 0u;
    const int64_t i = gbase + t * A.gt;
    return A.gamma_bf16 ? (uint32_t) static_cast<const uint16_t*>(A.gamma)[i] : static_cast<const uint32_t*>(A.gamma)[i];
  };
  auto gates = [&](uint32_t bits, int buf) {
    // Sums start anew at a reset, so that nothing in front of it is in those behind it.  What Hi and Lo hold is 2^15 lower for
    // each reset so far, and infinite where a sum is lost (a NaN, or growth beyond e^128, which fp32 does not hold), so that
    // Hi_t - Hi_s gives a weight of 0 across a reset, whatever s holds: sums between resets lie within 64 x 185.
    const float lg = __uint_as_float(A.gamma_bf16 ? bits << 16 : bits), inf = __builtin_inff();
    const bool cut = lane < C && lg < RESET;
    const uint64_t cuts = __ballot(cut), so_far = cuts & (((uint64_t)2 << lane) - 1);
    const int start = so_far == 0 ? 0 : 63 - __builtin_clzll(so_far);
    double y = cut ? 0.0 : lg <= 128.0f ? (double)lg * 1.4426950408889634 : (double)inf;
#pragma unroll
    for (int m = 1; m < C; m <<= 1) {
      const double z = __shfl_up(y, m, 64);
      if (lane - m >= start) y += z;
    }
    const double rest = __shfl(y, C - 1, 64) - y;
    if (lane < C) {
      const double low = y - 32768.0 * __builtin_popcountll(so_far);
      const float uh = (float)rest, ul = (float)(rest - (double)uh), hi = (float)low;
      const float lo = hi < inf ? (float)(low - (double)hi) : 0.0f;
      Hi[buf][lane] = hi;
      Lo[buf][lane] = lo;
      const float in = so_far != 0 ? 0.0f : exp2_of(hi) * exp2_of(lo);
      In[buf][lane] = in * A.out_scale;
      Up[buf][lane] = so_far != cuts ? 0.0f : hi < inf ? exp2_of(uh) * exp2_of(ul) * A.key_scale : inf;
      if (lane == C - 1) Whole[buf] = in;
    }
  };
  auto put_dots = [&](int64_t at) {  // after the barrier behind what a chunk's waves left
    if constexpr (DOTS) {
      if (x && tid < C && place(tid) < left_of(at)) {
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < Z::WAVES; ++w) d += Dot[w][tid];
        A.dots[bh * A.T + low_of(at) + place(tid)] = d;
      }
    }
  };

  fetch(u0);
  uint32_t gate = 0;
  if (wave == GATES) {
    gates(gate_bits(u0), 0);
    gate = gate_bits(u0 + C);
  }
  float whole_decay = 1.0f;
  int buf = 0;
  for (int64_t at = u0; at < u1; at += C, buf ^= 1) {
    // Addresses follow from the lane: hidden from the compiler, which would otherwise keep some 70 of them in registers
    // over the whole loop and spill
    asm volatile("" : "+v"(lane), "+v"(tid));
    g = lane >> 4, n = lane & 15;
    // the chunk's tokens to shared memory, and whether all keys and values are finite
    uint32_t most = 0;
    auto stage = [&](T* to, auto place_of, auto& r, auto width, bool look) {
      constexpr int D = decltype(width)::value;
#pragma unroll
      for (int j = 0; j < (int)(sizeof(r) / sizeof(r[0])); ++j) {
        const int i = tid + j * NT, row = i / (D / VEC), c = i % (D / VEC) * VEC;
        if (look) Op::largest(r[j], most);
        if (C * D / VEC % NT == 0 || row < C) *reinterpret_cast<u32x4*>(&to[place_of(row, c)]) = r[j];
      }
    };
    auto rows_of = [](auto stride) { return [](int row, int c) { return row * decltype(stride)::value + c; }; };
    stage(Ks, rows_of(std::integral_constant<int, KS>{}), kr, std::integral_constant<int, KD>{}, true);
    if constexpr (MODE != STATE_ONLY)
      stage(Qs, rows_of(std::integral_constant<int, QS>{}), qr, std::integral_constant<int, KD>{}, false);
    stage(Vs, rows_of(std::integral_constant<int, VS>{}), vr, std::integral_constant<int, VD>{}, true);
    if constexpr (PAIRED) stage(Xs, x_at, xr, std::integral_constant<int, VD>{}, false);
    const bool odd_here = __ballot(!Op::finite(most)) != 0;
    if (lane == 0) Odd[wave] = odd_here;
    __syncthreads();
    if (DIRECT && at > u0) put_dots(at - C);
    bool odd = false;
#pragma unroll
    for (int w = 0; w < Z::WAVES; ++w) odd = odd || Odd[w];
    if (at + C < u1) fetch(at + C);
    const float whole = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(Whole[buf])));
    const int64_t low = low_of(at);
    const int left = left_of(at);
    if (wave == GATES && at + C < u1) {
      gates(gate, buf ^ 1);
      gate = gate_bits(at + 2 * C);
    }
    struct alignas(4 * sizeof(T)) Four { T v[4]; };
    Four xs[DIRECT ? Z::TT : 1][Z::ET];
    if constexpr (DIRECT) {
      if (x) {
        const auto xrows = bounded(x + low * A.x.st, left * (int)A.x.st * (int)sizeof(T));
#pragma unroll
        for (int t = 0; t < Z::TT; ++t) {
          const int r = place(16 * t + n);
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) {
            const int c = e0 + 16 * e + 4 * g;
            if constexpr (WIDE) {
              const int off = c < A.vd ? (r * (int)A.x.st + c) * (int)sizeof(T) : BEYOND;
              xs[t][e] = __builtin_bit_cast(Four, __builtin_amdgcn_raw_buffer_load_b128(xrows, off, 0, 0));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                xs[t][e].v[i] = r < left && c + i < A.vd ? x[(low + r) * A.x.st + c + i] : from_f<T>(0.0f);
            }
          }
        }
      }
    }
    if constexpr (DOTS) {
      if (A.states && !A.reverse && at > 0 && at % A.mark_tokens == 0) {  // the state in front of a boundary
        put_state(A.states + (bh * A.marks + at / A.mark_tokens) * elems, A.vd, 1);
      }
    }

    f32x4 O[Z::TT][Z::ET];
    float dots[PAIRED ? Z::TT : 1] = {};  // this lane's part of x . o of token 16 t + n
    if constexpr (MODE != STATE_ONLY) {
      // scores, tile by tile over the waves
      int turn = 0;
#pragma unroll
      for (int ti = 0; ti < Z::TT; ++ti)
#pragma unroll
        for (int si = 0; si <= ti; ++si, ++turn) {
          if (turn % Z::WAVES != wave) continue;
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = 0; d < Z::DB; ++d)
            p = Op::mma(Op::row(&Ks[(16 * si + n) * KS + 32 * d + 8 * g]),
                        Op::row(&Qs[(16 * ti + n) * QS + 32 * d + 8 * g]), p);
          f32x4 vx = {0.f, 0.f, 0.f, 0.f};
          if constexpr (PAIRED) {
#pragma unroll
            for (int d = 0; d < Z::VB; ++d)
              vx = Op::mma(Op::row(&Vs[(16 * si + n) * VS + 32 * d + 8 * g]), Op::row(&Xs[x_at(16 * ti + n, 32 * d + 8 * g)]),
                           vx);
          }
          const float th = Hi[buf][16 * ti + n], tl = Lo[buf][16 * ti + n];
          const f32x4 sh = *reinterpret_cast<const f32x4*>(&Hi[buf][16 * si + 4 * g]),
                      sl = *reinterpret_cast<const f32x4*>(&Lo[buf][16 * si + 4 * g]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = exp2_of((th - sh[i]) + (tl - sl[i])) * (A.key_scale * A.out_scale);
            p[i] = si < ti || 4 * g + i <= n ? kept(w, p[i]) : 0.0f;
            if constexpr (PAIRED) dots[ti] += (si < ti || 4 * g + i <= n) && w != 0.0f ? p[i] * vx[i] : 0.0f;
          }
          Op::put_scores(&Ps[score_at(ti, si, n, 4 * g)], PART, p);
        }
      // the state's part
#pragma unroll
      for (int t = 0; t < Z::TT; ++t)
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) O[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < Z::DB; ++d) {
        std::conditional_t<MODE == EXACT, typename Op::Wide, typename Op::Pair> s[Z::ET];
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = S[2 * d][e][i], y[4 + i] = S[2 * d + 1][e][i];
          if constexpr (MODE == EXACT) s[e] = Op::wide(y); else s[e] = Op::pair(y);
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
        if (__ballot(w == 0.0f) == 0) {
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) O[t][e] *= w;
        } else {
#pragma unroll
          for (int e = 0; e < Z::ET; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[t][e][i] = kept(w, O[t][e][i]);
        }
        if constexpr (PAIRED) {
          float dot = dots[t];
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) {
            const Four f = *reinterpret_cast<const Four*>(&Xs[x_at(16 * t + n, e0 + 16 * e + 4 * g)]);
#pragma unroll
            for (int i = 0; i < 4; ++i) dot = fmaf(O[t][e][i], to_f(f.v[i]), dot);
          }
          dot += __shfl_xor(dot, 16, 64);
          dot += __shfl_xor(dot, 32, 64);
          if (g == 0) Dot[wave][16 * t + n] = dot;
        }
      }
      __syncthreads();
      if constexpr (PAIRED) put_dots(at);
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
            const typename Op::Pair f = Op::scores(&Ps[score_at(t, 2 * s, n, 4 * g)], PART, 2 * s < t);
#pragma unroll
            for (int e = 0; e < Z::ET; ++e) O[t][e] = Op::mma(vf[s][e], f, O[t][e]);
          }
      } else {
#pragma unroll
        for (int t = 0; t < Z::TT; ++t) {
          const int tt = 16 * t + n;
          for (int s = 0; s < C; ++s) {
            const float w = exp2_of((Hi[buf][tt] - Hi[buf][s]) + (Lo[buf][tt] - Lo[buf][s]));
            if (s > tt || w == 0.0f) continue;
            const float p = Op::score(&Ps[score_at(t, s / 16, n, s % 16)], PART);
#pragma unroll
            for (int e = 0; e < Z::ET; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) O[t][e][i] = fmaf(p, to_f(Vs[s * VS + e0 + 16 * e + 4 * g + i]), O[t][e][i]);
          }
        }
      }
      // out: a lane holds 4 neighbouring columns of one token
      const int64_t first = ((b * A.T + low) * A.H + h) * A.vd;
      auto put = [&](auto* y, int r, int c, const f32x4& o) {
        using Y = std::remove_pointer_t<decltype(y)>;
        Y f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = from_f<Y>(o[i]);
        if (W.out) {
          const int row = A.H * A.vd;  // below 2^22 here: the host sees to it
          const auto rows = bounded(y + first, ((left - 1) * row + A.vd) * (int)sizeof(Y));
          const int off = c < A.vd ? (r * row + c) * (int)sizeof(Y) : BEYOND;
          if constexpr (sizeof(Y) == 4)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f), rows, off, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f), rows, off, 0, 0);
        } else if (r < left) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < A.vd) y[first + (int64_t)r * A.H * A.vd + c + i] = f[i];
        }
      };
#pragma unroll
      for (int t = 0; t < Z::TT; ++t) {
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          const int c = e0 + 16 * e + 4 * g;
          const f32x4 r = O[t][e];
          if (A.out != nullptr) {
            if (A.out_f32) put(static_cast<float*>(A.out), place(16 * t + n), c, r);
            else put(static_cast<T*>(A.out), place(16 * t + n), c, r);
          }
          if constexpr (DIRECT) {
            if (x) {
#pragma unroll
              for (int i = 0; i < 4; ++i) dot = fmaf(r[i], to_f(xs[t][e].v[i]), dot);
            }
          }
        }
        if constexpr (DIRECT) {
          if (x) {
            dot += __shfl_xor(dot, 16, 64);
            dot += __shfl_xor(dot, 32, 64);
            if (g == 0) Dot[wave][16 * t + n] = dot;
          }
        }
      }
    }

    // the state behind the chunk
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int e = 0; e < Z::ET; ++e) S[d][e] = whole == 0.0f ? f32x4{0.f, 0.f, 0.f, 0.f} : S[d][e] * whole;
    whole_decay = whole == 0.0f ? 0.0f : kept(whole_decay, whole);  // a reset stays one beside decays that are not finite
    if (!odd) {
#pragma unroll
      for (int s = 0; s < Z::KB; ++s) {
        const f32x4 wa = *reinterpret_cast<const f32x4*>(&Up[buf][32 * s + 4 * g]),
                    wb = *reinterpret_cast<const f32x4*>(&Up[buf][32 * s + 16 + 4 * g]);
        typename Op::Wide wv[Z::ET];
#pragma unroll
        for (int e = 0; e < Z::ET; ++e) {
          float y[8];
          Op::values(vf[s][e], y);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= j < 4 ? wa[j] : wb[j - 4];
          wv[e] = Op::wide(y);
        }
#pragma unroll
        for (int d = 0; d < Z::DT; ++d) {
          const typename Op::Frag f = Op::column(&Ks[32 * s * KS], KS, 16 * d, lane);
#pragma unroll
          for (int e = 0; e < Z::ET; ++e) S[d][e] = Op::mma(f, wv[e], S[d][e]);
        }
      }
    } else {
      for (int s = 0; s < C; ++s) {
        const float w = Up[buf][s];
        if (w == 0.0f) continue;
        each([&](float o, int r, int c) { return fmaf(to_f(Ks[s * KS + r]), w * to_f(Vs[s * VS + c]), o); });
      }
    }
    if (DOTS && A.joins && A.reverse) {  // a boundary in front of token t: its decay's gradient
      const int64_t t = low;
      if (t > 0 && t % A.mark_tokens == 0) {
        const float lg = gamma_at(A, gbase + t * A.gt);
        meet(A.states + (bh * A.marks + t / A.mark_tokens) * elems, A.vd, 1, lg < RESET ? 0.0f : expf(lg), t / A.mark_tokens);
      }
    }
    __syncthreads();
  }
  if (DIRECT) put_dots(u1 - C);

  float* p = nullptr;
  int sr = A.sr, sc = A.sc;
  if (MODE == STATE_ONLY) {
    p = G.state + (bh * G.count + seg) * elems;
    sr = A.vd, sc = 1;
    if (tid == 0) G.decay[bh * G.count + seg] = whole_decay;
  } else if (A.state_out && seg == G.count - 1) {
    p = A.state_out + bh * elems;
    if (A.reverse) {
      const float lg = gamma_at(A, gbase), last = lg < RESET ? 0.0f : expf(lg);
      each([&](float s, int, int) { return kept(last, s); });
    }
  }
  if (p) put_state(p, sr, sc);
}

template <class T, int KD, int VD, int MODE>
int launch_mode(const Sweep& A, const Segments& G, const Wides& W, hipStream_t s) {
  using Z = ChunkShape<T, KD, VD>;
  const int segs = MODE == STATE_ONLY ? G.count - 1 : G.count;
  return in_launches(A.B * A.H * segs, Z::NT, [&](int64_t first, dim3 grid) {
    Sweep part = A;
    part.first = first / segs;
    if (W.in)
      hipLaunchKernelGGL((chunk_sweep_kernel<T, KD, VD, MODE, true>), grid, dim3(Z::NT), 0, s, part, G, W);
    else
      hipLaunchKernelGGL((chunk_sweep_kernel<T, KD, VD, MODE, false>), grid, dim3(Z::NT), 0, s, part, G, W);
  }, segs);
}

template <class T, int KD, int VD>
int launch_chunk(const Sweep& A, const Segments& G, const Wides& W, int mode, hipStream_t s) {
  if (mode == STATE_ONLY) return launch_mode<T, KD, VD, STATE_ONLY>(A, G, W, s);
  if (mode == FAST || sizeof(T) == 4) return launch_mode<T, KD, VD, FAST>(A, G, W, s);  // fp32 products are exact enough
  return launch_mode<T, KD, VD, sizeof(T) == 4 ? FAST : EXACT>(A, G, W, s);
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
