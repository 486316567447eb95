// ttc_ops_delta_chunk.hpp -- the gated delta rule in chunks on the matrix cores (formulas: ttc_ops_delta.hpp).
//
// A sweep's wave holds 16 columns of the state in registers, all rows, and needs nothing of the other waves: the columns of
// S, E, O, R and dV never meet.  Products are laid out so that no accumulator moves before it is an operand:
//   K S         lane: column n, 4 neighbouring tokens       -> with V, rows of the next product's right side
//   E = T Y     T in tiles as operands; E as it lies in the accumulators is the next right side
//   O' = S' Q' + E' (P b)'   lane: token n, 4 neighbouring columns -> stored 4 at once
//   S += K' (w E)            K' by transposing reads of shared memory (bf16) or element by element (fp32)
// Tokens that are not finite: where E (dV) of a wave's columns is not, the wave goes through that chunk token by token, so that
// no token has an effect on earlier ones and none passes a reset.
//
// Numerics.  In bf16 every operand that is not an input is split into three bf16 parts (24 digits), so that sums are those of 32
// bits.  Against 64 bits: bf16 outputs and gradients 1.7e-3 of their norm (one rounding), states and the decays' gradient 2e-7 to
// 4e-7; 0.03 % of the outputs round to the other neighbour of the exact value.  From two parts 1 % did (of queries' and keys'
// gradients 0.4 %), for 1.5 % less time in a long prompt and in training, 6 % where heads fill the GPU by themselves.
//
// Bound.  Of a kernel's cycles (one MI355X)             vector ALU  matrix cores  waits  read, written (MB)    us
//   16,381 tokens x 16 heads of 128 x 128, 16 segments
//     prepare                                             41 %          9 %        57 %     70, 139            74
//     sweep, STATE (values and matrix)                    59           40          24       99,  32           173
//     join                                                14            5          46       17,  17            52
//     sweep                                               50           36          26      179,  68           163
//   training on 4 x 2,048 tokens x 32 heads of 64 x 64, 4 segments
//     prepare                                             48           10          59       35, 139            56
//     sweep, STATE (values and matrix)                    61           35          27       67,  13            62
//     sweep, with what the backward needs                 35           20          24      124, 168            93
//     sweep back, STATE                                   41           29          30       90,   6            58
//     sweep back                                          33           20          22      124, 135            83
//     gradients                                           39           15          48      195, 112           205
// (read and written behind the XCDs' caches).  The sweeps wait for their own chain, one chunk after the other, and split three
// ways what the state is multiplied with (176 of some 650 vector instructions a chunk at 128 rows); more waves a SIMD would
// cover it, but a wave needs 150 to 250 registers.  Operands of different sums are read first and their instructions issued
// in turn; arrays in shared memory are mixed so that reads along and across rows meet each bank once (with 4 reads of 5 in
// conflict: STATE at 128 x 128 218 us, so 176).  8 waves of 16 columns a workgroup instead of two workgroups of 4: the same at
// 128 x 128, fp32 of 48 x 80 slower (27 us against 19).
#pragma once
#include "ttc_ops_delta.hpp"
#include "ttc_ops_mfma.hpp"

namespace ttc {

template <class T, int KD>
struct DeltaShape {
  static constexpr int C = chunk_tokens(sizeof(T) == 2), TT = C / 16, KB = C / 32, DB = KD / 32, DT = KD / 16;
  static constexpr int TILES = TT * (TT + 1) / 2, QS = KD + Operand<T>::ROW_PAD, KS = KD + Operand<T>::COL_PAD;
};
constexpr int tile_of(int t, int s) { return t * (t + 1) / 2 + s; }

// A chunk's rows of D elements: 16-byte loads, all in flight at once, then to shared memory.  Rows that do not exist and
// elements behind `dim` are 0.  A thread's vectors lie in one column, STEP rows apart, so that its places follow from the first
// one's.
template <class T, int D, int C, int NT>
struct Stage {
  static constexpr int VEC = 16 / sizeof(T), COLS = D / VEC, STEP = NT / COLS, N = (C + STEP - 1) / STEP;
  static_assert(NT % COLS == 0, "whole rows of threads");
  u32x4 r[N];
  __device__ __forceinline__ void fetch(const T* p, int64_t st, int dim, int left, bool wide, int tid) {
    const int row = tid / COLS, c = tid % COLS * VEC;
    if (wide) {
      const auto rows = bounded(p, left * (int)st * (int)sizeof(T));  // rows do not overlap: st >= dim
      const unsigned at = c < dim ? (unsigned)(row * (int)st + c) * (unsigned)sizeof(T) : (unsigned)BEYOND;
      const unsigned step = (unsigned)(STEP * (int)st) * (unsigned)sizeof(T);  // a chunk's rows lie within 2^30 bytes: no overflow
#pragma unroll
      for (int j = 0; j < N; ++j) r[j] = __builtin_amdgcn_raw_buffer_load_b128(rows, (int)(at + j * step), 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const u32x4 zero = {0, 0, 0, 0};
        r[j] = row + j * STEP < left ? load_any(p + (int64_t)(row + j * STEP) * st, c, dim) : zero;
      }
    }
  }
  template <int STRIDE>
  __device__ __forceinline__ void put(T* to, int tid) const {
    T* p = to + tid / COLS * STRIDE + tid % COLS * VEC;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (C % STEP == 0 || tid / COLS + j * STEP < C) *reinterpret_cast<u32x4*>(p + j * STEP * STRIDE) = r[j];
  }
  template <int STRIDE>
  __device__ __forceinline__ void put_mixed(T* to, int tid) const {
    static_assert(C % STEP == 0, "whole rows");
    if constexpr (STEP % 16 == 0) {  // rows that are mixed alike
      T* p = to + Operand<T>::mixed_place(tid / COLS, tid % COLS * VEC, STRIDE);
#pragma unroll
      for (int j = 0; j < N; ++j) *reinterpret_cast<u32x4*>(p + j * STEP * STRIDE) = Operand<T>::mixed(tid / COLS, r[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int row = tid / COLS + j * STEP;
        *reinterpret_cast<u32x4*>(to + Operand<T>::mixed_place(row, tid % COLS * VEC, STRIDE)) = Operand<T>::mixed(row, r[j]);
      }
    }
  }
  __device__ __forceinline__ void largest(uint32_t& m) const {
#pragma unroll
    for (int j = 0; j < N; ++j) Operand<T>::largest(r[j], m);
  }
};

// A token's place among the decays, and e^{G_t - G_s}: 0 across a reset, whatever the sums hold
struct Place {
  float hi, lo, part;
};
__device__ __forceinline__ float weight_of(const Place& t, const Place& s) {
  return t.part == s.part ? exp2_of((t.hi - s.hi) + (t.lo - s.lo)) : 0.0f;
}

// m + 0 x: a sum that starts at 0 ends there only if all that it met is finite
__device__ __forceinline__ float met(float m, const f32x4& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaf(x[i], 0.0f, m);
  return m;
}

// c[i] += a[i] b, or b a[i], for i in [LO, HI): instructions of the different sums in turn
template <class Op, int LO, int HI, int N, class A, class B, int M>
__device__ __forceinline__ void mma_left(const A (&a)[N], const B& b, f32x4 (&c)[M]) {
#pragma unroll
  for (int p = 0; p < Op::steps((const A*)nullptr, (const B*)nullptr); ++p)
#pragma unroll
    for (int i = LO; i < HI; ++i) c[i] = Op::step(p, a[i], b, c[i]);
}
template <class Op, int LO, int HI, int N, class A, class B, int M>
__device__ __forceinline__ void mma_right(const B& b, const A (&a)[N], f32x4 (&c)[M]) {
#pragma unroll
  for (int p = 0; p < Op::steps((const B*)nullptr, (const A*)nullptr); ++p)
#pragma unroll
    for (int i = LO; i < HI; ++i) c[i] = Op::step(p, b, a[i], c[i]);
}

// f(0), ..., f(N - 1) of constants
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (N > 0) {
    unrolled<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// ---- prepare: decays, lengths, scores and the triangle's inverse, one workgroup a chunk ----------------------------

// acc + a b of 16 x 16 blocks in fp32
__device__ __forceinline__ f32x4 block_mma(const float* a, int stride_a, const float* b, int stride_b, f32x4 acc, int lane) {
  const int g = lane >> 4, n = lane & 15;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[n * stride_a + 4 * s + g], b[(4 * s + g) * stride_b + n], acc, 0, 0, 0);
  return acc;
}

template <class T, int KD>
__global__ __launch_bounds__(256) void delta_prepare_kernel(Delta A) {
  using Z = DeltaShape<T, KD>;
  using Op = Operand<T>;
  constexpr int C = Z::C, TT = Z::TT, QS = Z::QS, LS = C + 4, SUB = 256 / C, BS = 20;
  // Tiles of N b (rows of BS), and the inverse in the place of keys and queries, which are not needed any more: four workgroups a
  // CU for keys of up to 64 (4,096 chunks: 56 us; with a place of its own, two workgroups: 77), three for 128
  constexpr int ROOM = 2 * C * QS * (int)sizeof(T) > C * LS * 4 ? 2 * C * QS * (int)sizeof(T) : C * LS * 4;
  __shared__ __attribute__((aligned(16))) char Room[ROOM];
  __shared__ __attribute__((aligned(16))) float Lm[Z::TILES * 16 * BS];
  T *Ks = reinterpret_cast<T*>(Room), *Qs = Ks + C * QS;
  float* Tm = reinterpret_cast<float*>(Room);
  __shared__ __attribute__((aligned(16))) float Row[ROWS][C];
  __shared__ int Odd[4];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = A.first + blockIdx.x, bh = unit / A.chunks, t0 = unit % A.chunks * C, b = bh / A.H;
  const int h = (int)(bh % A.H), left = A.T - t0 < C ? (int)(A.T - t0) : C;
  {
    Stage<T, KD, C, 256> k, q;
    k.fetch(A.k.at<T>(b, h) + t0 * A.k.st, A.k.st, A.kd, left, A.wide_k, tid);
    q.fetch(A.q.at<T>(b, h) + t0 * A.q.st, A.q.st, A.kd, left, A.wide_q, tid);
    if (wave == 3) {
      const int64_t t = t0 + lane;
      const bool here = lane < left;
      const float lg = here ? gate_value(A.gamma, A.gamma_bf16, b * A.gb + h * A.gh + t * A.gt) : 0.0f;
      const float strength = here ? gate_value(A.beta, A.beta_bf16, b * A.bb + h * A.bh + t * A.bt) : 0.0f;
      const float inf = __builtin_inff();
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
        const float uh = (float)rest, ul = (float)(rest - (double)uh), hi = (float)y;
        const float lo = hi < inf ? (float)(y - (double)hi) : 0.0f;
        Row[HI][lane] = hi;
        Row[LO][lane] = lo;
        Row[PART][lane] = (float)__builtin_popcountll(so_far);
        Row[IN][lane] = so_far != 0 ? 0.0f : exp2_of(hi) * exp2_of(lo);
        Row[UP][lane] = so_far != cuts ? 0.0f : hi < inf ? exp2_of(uh) * exp2_of(ul) : inf;
        Row[DEC][lane] = cut ? -1.0f : expf(lg);
        Row[BETA][lane] = strength;
      }
    }
    k.template put<QS>(Ks, tid);
    q.template put<QS>(Qs, tid);
    uint32_t most = 0;
    k.largest(most);
    const bool odd = __ballot(!Op::finite(most)) != 0;
    if (lane == 0) Odd[wave] = odd;
  }
  __syncthreads();
  {
    const int row = tid / SUB, sub = tid % SUB;
    float kk = 1.0f, qq = 1.0f;
    if (A.normalize) {
      kk = qq = 0.0f;
      for (int c = sub; c < KD; c += SUB) {
        const float x = to_f(Ks[row * QS + c]), y = to_f(Qs[row * QS + c]);
        kk = fmaf(x, x, kk);
        qq = fmaf(y, y, qq);
      }
      kk = 1.0f / sqrtf(lane_sum(kk, SUB) + A.eps);
      qq = 1.0f / sqrtf(lane_sum(qq, SUB) + A.eps);
    }
    if (sub == 0) {
      const bool here = row < left;
      const float in = Row[IN][row], up = Row[UP][row];
      Row[RK][row] = here ? kk : 0.0f;
      Row[RQ][row] = here ? qq : 0.0f;
      Row[WK][row] = here ? kept(in, kk) : 0.0f;
      Row[WU][row] = here ? kept(up, kk * Row[BETA][row]) : 0.0f;
      Row[WQ][row] = here ? kept(in, qq * A.scale) : 0.0f;
    }
  }
  __syncthreads();
  constexpr int PLANE = Z::TILES * 256;
  T* scores = static_cast<T*>(A.scores) + unit * Op::WIDE_PARTS * PLANE;
  T* inverse = static_cast<T*>(A.inverse) + unit * Op::WIDE_PARTS * PLANE;
  for (int i = tid; i < ROWS * C / 4; i += 256)
    reinterpret_cast<f32x4*>(A.rows + unit * ROWS * C)[i] = reinterpret_cast<const f32x4*>(&Row[0][0])[i];
  int turn = 0;
#pragma unroll
  for (int ti = 0; ti < TT; ++ti)
#pragma unroll
    for (int si = 0; si <= ti; ++si, ++turn) {
      if (turn % 4 != wave) continue;
      f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;  // lane: token t = n, 4 neighbouring s
#pragma unroll
      for (int d = 0; d < Z::DB; ++d) {
        const typename Op::Frag f = Op::row(&Ks[(16 * si + n) * QS + 32 * d + 8 * g]);
        kk = Op::mma(f, Op::row(&Ks[(16 * ti + n) * QS + 32 * d + 8 * g]), kk);
        qk = Op::mma(f, Op::row(&Qs[(16 * ti + n) * QS + 32 * d + 8 * g]), qk);
      }
      const int t = 16 * ti + n, s = 16 * si + 4 * g;
      const Place at_t = {Row[HI][t], Row[LO][t], Row[PART][t]};
      const float rk = Row[RK][t], rq = Row[RQ][t] * A.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = weight_of(at_t, Place{Row[HI][s + i], Row[LO][s + i], Row[PART][s + i]});
        const float by = Row[RK][s + i] * Row[BETA][s + i];
        kk[i] = s + i < t ? kept(w, kk[i] * rk * by) : 0.0f;
        qk[i] = s + i <= t ? kept(w, qk[i] * rq * by) : 0.0f;
      }
      *reinterpret_cast<f32x4*>(&Lm[(tile_of(ti, si) * 16 + n) * BS + 4 * g]) = kk;
      Op::put_wide(scores + tile_of(ti, si) * 256 + Op::tile_at(n, 4 * g), PLANE, qk);
    }
  __syncthreads();
  // the diagonal blocks' inverses: a lane's column by forward substitution
  if (wave == 0 && lane < C) {
    const float* L = Lm + tile_of(lane >> 4, lane >> 4) * 16 * BS;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a = i == n ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) a = fmaf(-L[i * BS + j], x[j], a);
      x[i] = a;
      Tm[((lane & ~15) + i) * LS + lane] = a;
    }
  }
  __syncthreads();
  // [[a, 0], [c, b]]^-1 = [[a^-1, 0], [-b^-1 c a^-1, b^-1]]: blocks of 16, then of 32.  c a^-1 goes where nothing else is: above
  // the diagonal
  const f32x4 none = {0.f, 0.f, 0.f, 0.f};
  auto put = [&](int r, int c, const f32x4& x, float sign) {
#pragma unroll
    for (int i = 0; i < 4; ++i) Tm[(16 * r + 4 * g + i) * LS + 16 * c + n] = sign * x[i];
  };
  auto inv = [&](int r, int c) { return Tm + 16 * r * LS + 16 * c; };
  auto low = [&](int r, int c) { return Lm + tile_of(r, c) * 16 * BS; };
  if (wave < TT / 2)
    put(2 * wave, 2 * wave + 1, block_mma(low(2 * wave + 1, 2 * wave), BS, inv(2 * wave, 2 * wave), LS, none, lane), 1.0f);
  __syncthreads();
  if (wave < TT / 2)
    put(2 * wave + 1, 2 * wave, block_mma(inv(2 * wave + 1, 2 * wave + 1), LS, inv(2 * wave, 2 * wave + 1), LS, none, lane),
        -1.0f);
  if constexpr (TT == 4) {
    const int r = wave >> 1, c = wave & 1;
    __syncthreads();
    f32x4 x = none;
    for (int k = c; k < 2; ++k) x = block_mma(low(2 + r, k), BS, inv(k, c), LS, x, lane);
    put(r, 2 + c, x, 1.0f);
    __syncthreads();
    x = none;
    for (int k = 0; k <= r; ++k) x = block_mma(inv(2 + r, 2 + k), LS, inv(k, 2 + c), LS, x, lane);
    put(2 + r, c, x, -1.0f);
  }
  __syncthreads();
  float all = 0.0f;
#pragma unroll
  for (int ti = 0; ti < TT; ++ti)
#pragma unroll
    for (int si = 0; si <= ti; ++si) {
      if (tile_of(ti, si) % 4 != wave) continue;
      const f32x4 x = *reinterpret_cast<const f32x4*>(&Tm[(16 * ti + n) * LS + 16 * si + 4 * g]);
      all = met(all, x);
      Op::put_wide(inverse + tile_of(ti, si) * 256 + Op::tile_at(n, 4 * g), PLANE, x);
    }
  const bool bad = __ballot(all != 0.0f) != 0;
  if (lane == 0) Odd[wave] |= bad;
  __syncthreads();
  if (tid == 0) A.odd[unit] = Odd[0] | Odd[1] | Odd[2] | Odd[3];
}

// ---- sweeps ----------------------------------------------------------------------------------------------------

// 8 values of two accumulators: rows 4 g + i of both
__device__ __forceinline__ void eight(const f32x4& a, const f32x4& b, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}

// A segment's chunks.  STATE: nothing but the state behind them, of nothing in front; forwards also, by further workgroups, of the
// unit matrix in front and no values.
template <class T, int KD, int WAVES, bool BACK, bool STATE>
__global__ __launch_bounds__(WAVES * 64, 2) void delta_sweep_kernel(Delta A) {
  using Z = DeltaShape<T, KD>;
  using Op = Operand<T>;
  using Wide = typename Op::Wide;
  using Frag = typename Op::Frag;
  constexpr int C = Z::C, TT = Z::TT, KB = Z::KB, NT = WAVES * 64, COLS = 16 * WAVES, KS = Z::KS,
                VS = COLS + Op::COL_PAD;
  __shared__ __attribute__((aligned(16))) T Ks[C * KS], Qs[C * KS], Vs[C * VS];  // Vs: V, or dO
  constexpr int PLANE = Z::TILES * 256, PARTS = Op::WIDE_PARTS;
  __shared__ __attribute__((aligned(16))) T inverse[PARTS * PLANE], scores[PARTS * PLANE];  // their tiles in parts
  __shared__ __attribute__((aligned(16))) float Row[ROWS][C];
  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int blocks = STATE && !BACK ? A.colblocks + (KD + COLS - 1) / COLS : A.colblocks;
  const Spread W = spread(A.first, blocks);
  const int block = W.block;
  const bool matrix = STATE && !BACK && block >= A.colblocks;
  const int c0 = (matrix ? block - A.colblocks : block) * COLS, e0 = wave * 16;  // the workgroup's columns, the wave's of those
  const int64_t part = W.group, bh = part / A.segs, b = bh / A.H;
  const int seg = (int)(part % A.segs);
  const int h = (int)(bh % A.H);
  const T *q = A.q.at<T>(b, h), *k = A.k.at<T>(b, h), *v = (BACK ? A.d_o : A.v).at<T>(b, h) + c0;
  const int64_t vst = BACK ? A.d_o.st : A.v.st;
  const bool wide_v = BACK ? A.wide_d : A.wide_v;

  f32x4 S[Z::DT];  // the state (BACK: its gradient): rows 16 d + 4 g + i, column e0 + n
  auto each = [&](auto f) {
    int r = 4 * g, c = c0 + e0 + n;
    asm volatile("" : "+v"(r), "+v"(c));  // otherwise the addresses stay in registers over the whole loop
#pragma unroll
    for (int d = 0; d < Z::DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[d][i] = f((float)S[d][i], 16 * d + r + i, c);
  };
  float* const seg_state = A.segs > 1 ? A.seg_state + part * KD * A.vdp : nullptr;
  if constexpr (STATE) {
    // Nothing follows the last segment, and its matrix is the backward's alone; nothing is in front of the first one where no
    // state comes in (training on 4 x 2,048 tokens x 32 heads of 64: 66 us forward and 68 back, so 64 and 58)
    const bool last = seg == A.segs - 1, first = seg == 0;
    if (BACK ? first : matrix ? (last && !A.S) || (first && !A.state_in) : last) {
      if (matrix && c0 == 0 && tid == 0) A.seg_dead[part] = 1;
      return;
    }
    each([&](float, int r, int c) { return matrix && r == c ? 1.0f : 0.0f; });
  } else {
    const float* p = A.segs > 1 ? seg_state : A.state_in ? A.state_in + bh * A.kd * A.vd : nullptr;
    const int rows = A.segs > 1 ? KD : A.kd, cols = A.segs > 1 ? A.vdp : A.vd;
    const auto from = bounded(p, p ? rows * cols * 4 : 0);
    each([&](float, int r, int c) {
      return __builtin_bit_cast(
          float, __builtin_amdgcn_raw_buffer_load_b32(from, r < rows && c < cols ? (r * cols + c) * 4 : BEYOND, 0, 0));
    });
  }
  Stage<T, KD, C, NT> kr, qr;
  Stage<T, COLS, C, NT> vr;
  Stage<float, C, ROWS, NT> rr;
  Stage<T, 256, PARTS * Z::TILES, NT> ir, sr;
  int odd_next = 0;
  const int64_t begin = seg * A.seg_chunks, end = begin + A.seg_chunks < A.chunks ? begin + A.seg_chunks : A.chunks;
  auto chunk_of = [&](int64_t i) { return BACK ? end - 1 - i : begin + i; };
  auto fetch = [&](int64_t i) {
    const int64_t ch = chunk_of(i), t0 = ch * C;
    const int left = A.T - t0 < C ? (int)(A.T - t0) : C;
    kr.fetch(k + t0 * A.k.st, A.k.st, A.kd, left, A.wide_k, tid);
    if constexpr (BACK || !STATE) qr.fetch(q + t0 * A.q.st, A.q.st, A.kd, left, A.wide_q, tid);
    if (matrix) vr.fetch(q, 1, 0, 0, true, tid);  // zeros
    else vr.fetch(v + t0 * vst, vst, A.vd - c0, left, wide_v, tid);
    const int64_t unit = bh * A.chunks + ch;
    rr.fetch(A.rows + unit * ROWS * C, C, C, ROWS, true, tid);
    ir.fetch(static_cast<const T*>(A.inverse) + unit * PARTS * PLANE, 256, 256, PARTS * Z::TILES, true, tid);
    if constexpr (BACK || !STATE)
      sr.fetch(static_cast<const T*>(A.scores) + unit * PARTS * PLANE, 256, 256, PARTS * Z::TILES, true, tid);
    odd_next = A.odd[unit];
  };
  fetch(0);
  bool dead = false;
  for (int64_t i = 0; i < end - begin; ++i) {
    asm volatile("" : "+v"(lane), "+v"(tid));
    g = lane >> 4, n = lane & 15;
    const int64_t ch = chunk_of(i), t0 = ch * C, unit = bh * A.chunks + ch;
    const int left = A.T - t0 < C ? (int)(A.T - t0) : C;
    kr.template put_mixed<KS>(Ks, tid);
    if constexpr (BACK || !STATE) qr.template put_mixed<KS>(Qs, tid);
    vr.template put<VS>(Vs, tid);
    rr.template put<C>(&Row[0][0], tid);
    ir.template put<256>(inverse, tid);
    if constexpr (BACK || !STATE) sr.template put<256>(scores, tid);
    bool odd = odd_next != 0;
    __syncthreads();
    if (i + 1 < end - begin) fetch(i + 1);
    const float whole = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(Row[IN][C - 1])));
    dead = dead || Row[PART][C - 1] > 0.0f;
    float* kept_state = STATE ? nullptr : BACK ? A.R : A.S;
    if (kept_state) {
      float* p = kept_state + unit * KD * A.vdp;
      each([&](float s, int r, int c) {
        p[r * A.vdp + c] = s;
        return s;
      });
    }
    auto row4 = [&](int which, int t) { return *reinterpret_cast<const f32x4*>(&Row[which][t]); };  // of 4 neighbouring tokens

    const int rows_at = Op::row_place(KS, lane), columns_at = Op::column_place(KS, lane);
    // X = K S: lane's tokens 16 t + 4 g + i, column e0 + n.  Forward's O' = S' Q': lane's token 16 t + n, 4 columns
    f32x4 X[TT], O[BACK || STATE ? 1 : TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      X[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (!BACK && !STATE) O[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int d = 0; d < Z::DB; ++d) {
      Frag f[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) f[t] = Op::row_split(Ks + rows_at + 16 * t * KS + 32 * d);
      float y[8];
      eight(S[2 * d], S[2 * d + 1], y);
      const Wide s = Op::wide(y);
      mma_left<Op, 0, TT>(f, s, X);
      if constexpr (!BACK && !STATE) {
#pragma unroll
        for (int t = 0; t < TT; ++t) f[t] = Op::row_split(Qs + rows_at + 16 * t * KS + 32 * d);
        mma_right<Op, 0, TT>(s, f, O);
      }
    }
    // what the triangle is solved for: V - e^G K S, or b (e^{G_C - G} K R + P' dO).  A weight of 0 does not select here: where the
    // state is not finite, X is not, and the tokens go one by one below
    Frag vf[KB];
#pragma unroll
    for (int s = 0; s < KB; ++s) vf[s] = Op::column(&Vs[32 * s * VS], VS, e0, lane);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const f32x4 w = row4(BACK ? WU : WK, 16 * t + 4 * g);
      float y[8];
      if constexpr (!BACK) Op::values(vf[t / 2], y);
#pragma unroll
      for (int j = 0; j < 4; ++j) X[t][j] = BACK ? w[j] * X[t][j] : fmaf(-w[j], X[t][j], y[t % 2 * 4 + j]);
    }
    // E (dV): the inverse's (its transpose's) rows times that.  Row t of a lower triangle of tiles meets tiles up to t, of its
    // transpose from t on
    f32x4 E[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) E[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (BACK)
      unrolled<KB>([&](auto s_) {
        constexpr int s = decltype(s_)::value;
        Wide f[TT];
#pragma unroll
        for (int t = 0; t < 2 * s + 2; ++t)
          f[t] = Op::template wide_tiles<false>(2 * s >= t, scores + tile_of(2 * s, t) * 256, true, scores + tile_of(2 * s + 1, t) * 256,
                                                PLANE, lane);
        mma_left<Op, 0, 2 * s + 2>(f, vf[s], X);
      });
    Wide y[KB];
#pragma unroll
    for (int s = 0; s < KB; ++s) {
      float x[8];
      eight(X[2 * s], X[2 * s + 1], x);
      y[s] = Op::wide(x);
    }
    unrolled<KB>([&](auto s_) {
      constexpr int s = decltype(s_)::value, LO = BACK ? 0 : 2 * s, HI = BACK ? 2 * s + 2 : TT;
      Wide f[TT];
#pragma unroll
      for (int t = LO; t < HI; ++t)
        f[t] = BACK ? Op::template wide_tiles<false>(2 * s >= t, inverse + tile_of(2 * s, t) * 256, true,
                                                     inverse + tile_of(2 * s + 1, t) * 256, PLANE, lane)
                    : Op::template wide_tiles<true>(true, inverse + tile_of(t, 2 * s) * 256, 2 * s < t,
                                                    inverse + tile_of(t, 2 * s + 1) * 256, PLANE, lane);
      mma_left<Op, LO, HI>(f, y[s], E);
    });
    float all = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) all = met(all, E[t]);
    odd = odd || __ballot(all != 0.0f) != 0;
    float* const all_rows = STATE ? nullptr : BACK ? A.dV : A.E;
    float* const kept_rows = all_rows ? all_rows + unit * C * A.vdp + c0 + e0 : nullptr;
    const int64_t first = ((b * A.T + t0) * A.H + h) * A.vd;  // of the output
    const int64_t row = (int64_t)A.H * A.vd;
    if (!odd) {
      if (kept_rows) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) kept_rows[(16 * t + 4 * g + j) * A.vdp + n] = E[t][j];
      }
      if constexpr (!BACK && !STATE) {
#pragma unroll
        for (int t = 0; t < TT; ++t) O[t] *= Row[WQ][16 * t + n];
        unrolled<KB>([&](auto s_) {
          constexpr int s = decltype(s_)::value;
          float x[8];
          eight(E[2 * s], E[2 * s + 1], x);
          const Wide e = Op::wide(x);
          Wide f[TT];
#pragma unroll
          for (int t = 2 * s; t < TT; ++t)
            f[t] = Op::template wide_tiles<true>(true, scores + tile_of(t, 2 * s) * 256, 2 * s < t,
                                                 scores + tile_of(t, 2 * s + 1) * 256, PLANE, lane);
          mma_right<Op, 2 * s, TT>(e, f, O);
        });
#pragma unroll
        for (int t = 0; t < TT; ++t) {  // a lane holds 4 neighbouring columns of one token
          const int r = 16 * t + n, c = c0 + e0 + 4 * g;
          T f[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = from_f<T>(O[t][j]);
          T* to = static_cast<T*>(A.o) + first;
          if (A.wide_o) {
            const auto rows = bounded(to, ((left - 1) * (int)row + A.vd) * (int)sizeof(T));
            const int off = c < A.vd ? (r * (int)row + c) * (int)sizeof(T) : BEYOND;
            if constexpr (sizeof(T) == 4)
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f), rows, off, 0, 0);
            else
              __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f), rows, off, 0, 0);
          } else if (r < left) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < A.vd) to[r * row + c + j] = f[j];
          }
        }
      }
      // the state behind the chunk, or its gradient in front of it
#pragma unroll
      for (int d = 0; d < Z::DT; ++d) S[d] *= whole;
#pragma unroll
      for (int s = 0; s < KB; ++s) {
        const f32x4 wa = row4(BACK ? WK : WU, 32 * s + 4 * g), wb = row4(BACK ? WK : WU, 32 * s + 16 + 4 * g);
        float x[8];
        if constexpr (BACK) eight(E[2 * s] * -wa, E[2 * s + 1] * -wb, x);
        else eight(E[2 * s] * wa, E[2 * s + 1] * wb, x);
        const Wide we = Op::wide(x);
        Frag f[Z::DT];
#pragma unroll
        for (int d = 0; d < Z::DT; ++d) f[d] = Op::column_mixed(Ks + columns_at + 32 * s * KS + 16 * d, KS);
        mma_left<Op, 0, Z::DT>(f, we, S);
        if constexpr (BACK) {
          const f32x4 qa = row4(WQ, 32 * s + 4 * g), qb = row4(WQ, 32 * s + 16 + 4 * g);
          Op::values(vf[s], x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= j < 4 ? qa[j % 4] : qb[j % 4];
          const Wide wd = Op::wide(x);
#pragma unroll
          for (int d = 0; d < Z::DT; ++d) f[d] = Op::column_mixed(Qs + columns_at + 32 * s * KS + 16 * d, KS);
          mma_left<Op, 0, Z::DT>(f, wd, S);
        }
      }
    } else {  // token by token: a column needs nothing but its own entries
      for (int a = 0; a < left; ++a) {
        const int t = BACK ? left - 1 - a : a;
        const float rk = Row[RK][t], rq = Row[RQ][t] * A.scale, be = Row[BETA][t], dec = Row[DEC][t];
        const float in = to_f(Vs[t * VS + e0 + n]);
        float x = 0.0f, o = 0.0f;
        auto decay = [&](float s) { return dec < 0.0f ? 0.0f : kept(dec, s); };
#pragma unroll
        for (int d = 0; d < Z::DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 16 * d + 4 * g + j;
            const float kk = to_f(Ks[Op::at(t, r, KS)]), qq = STATE && !BACK ? 0.0f : to_f(Qs[Op::at(t, r, KS)]);
            S[d][j] = BACK ? fmaf(rq * qq, in, S[d][j]) : decay(S[d][j]);
            x = r < A.kd ? fmaf(kk, S[d][j], x) : x;
          }
        x += __shfl_xor(x, 16, 64);
        x += __shfl_xor(x, 32, 64);
        x = BACK ? be * (rk * x) : in - rk * x;  // dV, or E
        if (kept_rows && g == 0) kept_rows[t * A.vdp + n] = x;
#pragma unroll
        for (int d = 0; d < Z::DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 16 * d + 4 * g + j;
            const float kk = to_f(Ks[Op::at(t, r, KS)]), qq = STATE && !BACK ? 0.0f : to_f(Qs[Op::at(t, r, KS)]);
            if constexpr (BACK) {
              S[d][j] = r < A.kd ? decay(fmaf(-rk * kk, x, S[d][j])) : 0.0f;
            } else {
              S[d][j] = r < A.kd ? fmaf(rk * kk, be * x, S[d][j]) : 0.0f;
              o = r < A.kd ? fmaf(qq, S[d][j], o) : o;
            }
          }
        if constexpr (!BACK && !STATE) {
          o += __shfl_xor(o, 16, 64);
          o += __shfl_xor(o, 32, 64);
          const int c = c0 + e0 + n;
          if (g == 0 && c < A.vd) static_cast<T*>(A.o)[first + t * row + c] = from_f<T>(rq * o);
        }
      }
      if (kept_rows && left < C) {  // rows that do not exist
        for (int t = left; t < C; ++t)
          if (g == 0) kept_rows[t * A.vdp + n] = 0.0f;
      }
    }
    __syncthreads();
  }
  if constexpr (STATE) {
    float* p = matrix ? A.seg_matrix + part * KD * KD : seg_state;
    const int cols = matrix ? KD : A.vdp;
    each([&](float s, int r, int c) {
      if (c < cols) p[r * cols + c] = s;
      return s;
    });
    if (matrix && c0 == 0 && tid == 0) A.seg_dead[part] = dead;
  } else if (A.state_out && seg == (BACK ? 0 : A.segs - 1)) {
    float* p = A.state_out + bh * A.kd * A.vd;
    const auto to = bounded(p, A.kd * A.vd * 4);
    each([&](float s, int r, int c) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s), to, r < A.kd && c < A.vd ? (r * A.vd + c) * 4 : BEYOND, 0, 0);
      return s;
    });
  }
}

// ---- gradients: of queries, keys, decays and strengths, one workgroup a chunk ----------------------------------------
//
//   L = dO E',  M = dV E',  A = b e^{G_t - G_s} L (s <= t),  B = -b e^{G_t - G_s} M (s < t)
//   dq_t = sum_s A_ts k_s + e^{G_t} S dO_t,   dk_s = sum_t A_ts q_t + sum_t B_ts k_t + sum_t B_st k_t + b e^{G_C - G_s} R E_s
//          - e^{G_s} S dV_s       (q with its scale, both at their lengths)
// and with x_ts = P_ts L_ts - N_ts M_ts, f_s = e^{G_C - G_s} k_s . R E_s,
//   db_s = sum_t x_ts + f_s,   dg_t = the sum over all terms of the loss's gradient that decay across token t: pairs s < t <= t',
//   the state in front (into tokens from t on), the state behind (from tokens before t), and the state through the chunk.
// Values come 32 columns at a time, split into their parts once (all at once, split by each wave that reads them: 4,096 chunks of
// 64 x 64 265 us, so 193 with score tiles in two parts).  Waves share the score tiles, in three parts of which those that meet the
// tokens in front of each take turns with those that meet the tokens behind (205 us; all four sets in two parts 193), and each wave
// takes 16 columns of the keys; its lanes hold one token and 4 neighbouring columns.  Bound by latency: two workgroups a CU (66 KB at
// 64), each of which loads, meets, multiplies and stores; of the 193, without the second 32 columns 160 us, without the tiles' sums
// 175, without the products with keys and queries 182.
template <class T, int KD>
__global__ __launch_bounds__((KD / 16 * 64), 2) void delta_gradients_kernel(Delta A) {
  using Z = DeltaShape<T, KD>;
  using Op = Operand<T>;
  using Wide = typename Op::Wide;
  using Frag = typename Op::Frag;
  constexpr int C = Z::C, TT = Z::TT, KB = Z::KB, WAVES = KD / 16, NT = WAVES * 64, KS = Z::KS, MINE = (Z::TILES + WAVES - 1) / WAVES;
  constexpr int W = 32, DS = W + Op::ROW_PAD, BLOCK = C * DS, PARTS = Op::WIDE_PARTS;  // columns of values, and their rows
  constexpr int PLANE = Z::TILES * 256, SET = PARTS * PLANE, ROOM = (2 * PARTS + 1) * BLOCK;
  __shared__ __attribute__((aligned(16))) T Ks[C * KS], Qs[C * KS];
  __shared__ __attribute__((aligned(16))) T Big[ROOM > 2 * SET ? ROOM : 2 * SET];  // E, dV and dO, then A and B as they are used
  __shared__ __attribute__((aligned(16))) float Row[ROWS][C];
  __shared__ float Part[TT][3][C];    // by tile: sums over s of b P L and of b N M (by si), over t of x (by ti)
  __shared__ float Dot[WAVES][3][C];  // by wave: q . S dO, k . S dV, k . R E
  __shared__ float Through[WAVES], Qd[C], Kd[C];
  __shared__ int Odd[WAVES];
  T *Es = Big, *Vs = Big + PARTS * BLOCK, *Ds = Big + 2 * PARTS * BLOCK;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = A.first + blockIdx.x, bh = unit / A.chunks, t0 = unit % A.chunks * C, b = bh / A.H;
  const int h = (int)(bh % A.H), left = A.T - t0 < C ? (int)(A.T - t0) : C, blocks = A.vdp / W;
  uint32_t most = 0, most_f = 0;
  const int r0 = wave * 16;
  // 8 neighbouring values of E and of dV a thread (UNITS of them)
  constexpr int UNITS = (C * W / 8 + NT - 1) / NT;
  u32x4 er[UNITS][2], vr[UNITS][2];
  Stage<T, W, C, NT> dr;
  f32x4 sr[4];  // 8 neighbours of a row of S and of R
  const float *Sp = A.S + (unit * KD + r0 + n) * A.vdp + 8 * g, *Rp = A.R + (unit * KD + r0 + n) * A.vdp + 8 * g;
  auto fetch = [&](int d) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sr[i] = reinterpret_cast<const f32x4*>(Sp + d * W)[i];
      sr[2 + i] = reinterpret_cast<const f32x4*>(Rp + d * W)[i];
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      const int u = tid + j * NT, row = u / 4 < C ? u / 4 : 0, c = d * W + u % 4 * 8;
      const float *e = A.E + (unit * C + row) * A.vdp + c, *v = A.dV + (unit * C + row) * A.vdp + c;
#pragma unroll
      for (int i = 0; i < 2; ++i) er[j][i] = reinterpret_cast<const u32x4*>(e)[i], vr[j][i] = reinterpret_cast<const u32x4*>(v)[i];
    }
    const int c0 = d * W;
    dr.fetch(A.d_o.at<T>(b, h) + t0 * A.d_o.st + c0, A.d_o.st, A.vd - c0, left, A.wide_d, tid);
  };
  auto put = [&](int d) {
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      const int u = tid + j * NT, row = u / 4, c = u % 4 * 8;
      if (row >= C) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Operand<float>::largest(er[j][i], most_f);
        Operand<float>::largest(vr[j][i], most_f);
        Op::put_wide(Es + row * DS + c + 4 * i, BLOCK, __builtin_bit_cast(f32x4, er[j][i]));
        Op::put_wide(Vs + row * DS + c + 4 * i, BLOCK, __builtin_bit_cast(f32x4, vr[j][i]));
      }
      if (A.dv && row < left) {  // values' gradients, where each head has its own
        T* to = static_cast<T*>(A.dv) + ((b * A.T + t0 + row) * A.H + h) * A.vd + d * W + c;
        T f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = from_f<T>(__uint_as_float(vr[j][i / 4][i % 4]));
        if (A.wide_dv && d * W + c < A.vd) {
          __builtin_memcpy(__builtin_assume_aligned(to, 16), f, sizeof(f));
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (d * W + c + i < A.vd) to[i] = f[i];
        }
      }
    }
    dr.template put<DS>(Ds, tid);
    dr.largest(most);
  };
  auto wide_row = [&](const T* p, int row) {  // 8 neighbours
    const T* at = p + row * DS + 8 * g;
    if constexpr (PARTS == 3) return Wide{Op::row(at), Op::row(at + BLOCK), Op::row(at + 2 * BLOCK)};
    else return Op::row(at);
  };

  // Over the columns of the values: L and M of the wave's tiles (lane: token t = n, 4 neighbouring s), and the state's parts S dO,
  // S dV and R E (rows r0 + n of S and R; lane's token n, columns r0 + 4 g + i)
  f32x4 lt[MINE], mt[MINE], dq[TT], sv[TT], re[TT], dk[TT];
#pragma unroll
  for (int i = 0; i < MINE; ++i) lt[i] = mt[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < TT; ++t) dq[t] = sv[t] = re[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float through = 0.0f;
  {  // all loads of the first columns on their way together
    Stage<T, KD, C, NT> k, q;
    Stage<float, C, ROWS, NT> r;
    k.fetch(A.k.at<T>(b, h) + t0 * A.k.st, A.k.st, A.kd, left, A.wide_k, tid);
    q.fetch(A.q.at<T>(b, h) + t0 * A.q.st, A.q.st, A.kd, left, A.wide_q, tid);
    r.fetch(A.rows + unit * ROWS * C, C, C, ROWS, true, tid);
    fetch(0);
    k.template put_mixed<KS>(Ks, tid);
    q.template put_mixed<KS>(Qs, tid);
    r.template put<C>(&Row[0][0], tid);
    k.largest(most);
    q.largest(most);
  }
  for (int d = 0; d < blocks; ++d) {
    put(d);
    float s8[8], r8[8];
    eight(sr[0], sr[1], s8);
    eight(sr[2], sr[3], r8);
    __syncthreads();
    if (d + 1 < blocks) fetch(d + 1);
    int turn = 0;
#pragma unroll
    for (int ti = 0; ti < TT; ++ti)
#pragma unroll
      for (int si = 0; si <= ti; ++si, ++turn) {
        if (turn % WAVES != wave) continue;
        const Wide f = wide_row(Es, 16 * si + n);
        lt[turn / WAVES] = Op::mma(f, Op::row(&Ds[(16 * ti + n) * DS + 8 * g]), lt[turn / WAVES]);
        mt[turn / WAVES] = Op::mma(f, wide_row(Vs, 16 * ti + n), mt[turn / WAVES]);
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) through = fmaf(s8[i], r8[i], through);
    const Wide s = Op::wide(s8);
    Wide f[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) f[t] = wide_row(Vs, 16 * t + n);
    mma_right<Op, 0, TT>(s, f, sv);
    Frag x[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) x[t] = Op::row(&Ds[(16 * t + n) * DS + 8 * g]);
    mma_right<Op, 0, TT>(s, x, dq);
    const Wide r = Op::wide(r8);
#pragma unroll
    for (int t = 0; t < TT; ++t) f[t] = wide_row(Es, 16 * t + n);
    mma_right<Op, 0, TT>(r, f, re);
    __syncthreads();
  }
  {
    const bool odd_here = __ballot(!Op::finite(most) || !Operand<float>::finite(most_f)) != 0;
    if (lane == 0) Odd[wave] = odd_here;
  }

  // the tiles: their sums, and A and B in the place of E, dV and dO, with the weights of what each is multiplied with: first that
  // of the tokens in front, then, in the same place, of those behind (in lt and mt until then)
  T *As = Big, *Bs = Big + SET;
  const int rows_at = Op::row_place(KS, lane), columns_at = Op::column_place(KS, lane);
  {
    int turn = 0;
#pragma unroll
    for (int ti = 0; ti < TT; ++ti)
#pragma unroll
      for (int si = 0; si <= ti; ++si, ++turn) {
        if (turn % WAVES != wave) continue;
        f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;
#pragma unroll
        for (int d = 0; d < Z::DB; ++d) {
          const Frag f = Op::row_split(Ks + rows_at + 16 * si * KS + 32 * d);
          kk = Op::mma(f, Op::row_split(Ks + rows_at + 16 * ti * KS + 32 * d), kk);
          qk = Op::mma(f, Op::row_split(Qs + rows_at + 16 * ti * KS + 32 * d), qk);
        }
        const int t = 16 * ti + n, s = 16 * si + 4 * g;
        const Place at_t = {Row[HI][t], Row[LO][t], Row[PART][t]};
        const float rk = Row[RK][t], rq = Row[RQ][t] * A.scale;
        const f32x4 l = lt[turn / WAVES], m = mt[turn / WAVES];
        float sum_p = 0.0f, sum_n = 0.0f, by_s[4];
        f32x4 at, bt, as, bs;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = weight_of(at_t, Place{Row[HI][s + i], Row[LO][s + i], Row[PART][s + i]}), be = Row[BETA][s + i],
                      rs = Row[RK][s + i];
          const float pl = s + i <= t ? kept(w, rq * rs * qk[i] * l[i]) : 0.0f;
          const float nm = s + i < t ? kept(w, rk * rs * kk[i] * m[i]) : 0.0f;
          sum_p = s + i <= t && w != 0.0f ? fmaf(be, pl, sum_p) : sum_p;
          sum_n = s + i < t && w != 0.0f ? fmaf(be, nm, sum_n) : sum_n;
          by_s[i] = pl - nm;
          at[i] = s + i <= t ? kept(w, be * l[i]) : 0.0f;
          bt[i] = s + i < t ? kept(w, -be * m[i]) : 0.0f;
          as[i] = at[i] * rs, bs[i] = bt[i] * rs;
        }
        const int tile = tile_of(ti, si) * 256 + Op::tile_at(n, 4 * g);
        Op::put_wide(As + tile, PLANE, as);
        Op::put_wide(Bs + tile, PLANE, bs);
        lt[turn / WAVES] = at * rq, mt[turn / WAVES] = bt * rk;
        sum_p += __shfl_xor(sum_p, 16, 64);
        sum_p += __shfl_xor(sum_p, 32, 64);
        sum_n += __shfl_xor(sum_n, 16, 64);
        sum_n += __shfl_xor(sum_n, 32, 64);
        if (g == 0) Part[si][0][t] = sum_p, Part[si][1][t] = sum_n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int x = 1; x <= 8; x <<= 1) by_s[i] += __shfl_xor(by_s[i], x, 64);
          if (n == 0) Part[ti][2][s + i] = by_s[i];
        }
      }
  }
  // the state's parts with their weights, and their dots with q and k
  auto four = [&](const T* p, int t) {  // the lane's columns of token t
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    };
    return *reinterpret_cast<const Four*>(p + Op::at(t, r0 + 4 * g, KS));
  };
  through = lane_sum(through, 64);
  if (lane == 0) Through[wave] = through;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int tt = 16 * t + n;
    const float in = Row[IN][tt], up = Row[UP][tt], be = Row[BETA][tt], rq = Row[RQ][tt] * A.scale, rk = Row[RK][tt];
    const auto q4 = four(Qs, tt), k4 = four(Ks, tt);
    float c = 0.0f, d = 0.0f, f = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float qq = rq * to_f(q4.v[i]), kk = rk * to_f(k4.v[i]);
      dq[t][i] = kept(in, dq[t][i]);
      sv[t][i] = kept(in, sv[t][i]);
      re[t][i] = kept(up, re[t][i]);
      if (r0 + 4 * g + i < A.kd) {
        c = in == 0.0f ? c : fmaf(qq, dq[t][i], c);
        d = in == 0.0f ? d : fmaf(kk, sv[t][i], d);
        f = up == 0.0f ? f : fmaf(kk, re[t][i], f);
      }
      dk[t][i] = up == 0.0f ? -sv[t][i] : be * re[t][i] - sv[t][i];
    }
    c += __shfl_xor(c, 16, 64);
    c += __shfl_xor(c, 32, 64);
    d += __shfl_xor(d, 16, 64);
    d += __shfl_xor(d, 32, 64);
    f += __shfl_xor(f, 16, 64);
    f += __shfl_xor(f, 32, 64);
    if (g == 0) Dot[wave][0][tt] = c, Dot[wave][1][tt] = d, Dot[wave][2][tt] = f;
  }
  __syncthreads();
  bool odd = A.odd[unit] != 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) odd = odd || Odd[w];
  // one wave: what a token's sums come to, and the gradients of its decay and strength
  if (wave == 0) {
    const int t = lane < C ? lane : C - 1, own = t / 16;
    float sum_p = 0.0f, sum_n = 0.0f, x = 0.0f, c = 0.0f, d = 0.0f, f = 0.0f, through = 0.0f;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      if (i <= own) sum_p += Part[i][0][t], sum_n += Part[i][1][t];
      if (i >= own) x += Part[i][2][t];
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w) c += Dot[w][0][t], d += Dot[w][1][t], f += Dot[w][2][t], through += Through[w];
    const float be = Row[BETA][t], whole = Row[IN][C - 1];
    if (lane < C) {
      Qd[t] = c + sum_p;
      Kd[t] = be * (x + f) - sum_n - d;
    }
    // suffix sums within the texts that resets part, and of f those in front
    const bool cut = lane < C && Row[DEC][t] < 0.0f;
    const uint64_t cuts = __ballot(cut);
    const uint64_t later = lane < 63 ? cuts & (~(uint64_t)0 << (lane + 1)) : 0, so_far = cuts & (((uint64_t)2 << lane) - 1);
    const int end = later ? __builtin_ctzll(later) : C, start = so_far ? 63 - __builtin_clzll(so_far) : 0;
    double suffix = lane < C ? (double)sum_p - sum_n + c - d - (double)be * x : 0.0, before = lane < C ? (double)be * f : 0.0;
#pragma unroll
    for (int m = 1; m < C; m <<= 1) {
      const double up = __shfl_down(suffix, m, 64), low = __shfl_up(before, m, 64);
      if (lane + m < end) suffix += up;
      if (lane - m >= start) before += low;
    }
    before = __shfl_up(before, 1, 64);
    if (lane == start) before = 0.0;
    if (lane < left) {
      const double dg = cut ? 0.0 : suffix + before + (cuts ? 0.0 : (double)kept(whole, through));
      const int64_t at = (b * A.T + t0 + lane) * A.H + h;
      if (A.dgamma) {
        if (A.gamma_bf16) static_cast<__bf16*>(A.dgamma)[at] = from_f<__bf16>((float)dg);
        else static_cast<float*>(A.dgamma)[at] = (float)dg;
      }
      if (A.dbeta) {
        if (A.beta_bf16) static_cast<__bf16*>(A.dbeta)[at] = from_f<__bf16>(x + f);
        else static_cast<float*>(A.dbeta)[at] = x + f;
      }
    }
  }
  // products with the tokens in front (A K to dq, B K to dk), or with those behind (A' Q and B' K to dk); what is not finite: term
  // by term, without those whose weight is 0
  auto products = [&](auto front_) {
    constexpr bool FRONT = decltype(front_)::value;
    if (!odd) {
      unrolled<KB>([&](auto s_) {
        constexpr int s = decltype(s_)::value, LO = FRONT ? 2 * s : 0, HI = FRONT ? TT : 2 * s + 2;
        const Frag kf = Op::column_mixed(Ks + columns_at + 32 * s * KS + r0, KS);
        const Frag xf = FRONT ? kf : Op::column_mixed(Qs + columns_at + 32 * s * KS + r0, KS);
        auto tiles = [&](const T* p, int t) {
          if constexpr (FRONT)
            return Op::template wide_tiles<true>(true, p + tile_of(t, 2 * s) * 256, 2 * s < t, p + tile_of(t, 2 * s + 1) * 256, PLANE, lane);
          else
            return Op::template wide_tiles<false>(2 * s >= t, p + tile_of(2 * s, t) * 256, true, p + tile_of(2 * s + 1, t) * 256, PLANE, lane);
        };
        Wide f[TT];
#pragma unroll
        for (int t = LO; t < HI; ++t) f[t] = tiles(As, t);
        mma_right<Op, LO, HI>(xf, f, FRONT ? dq : dk);
#pragma unroll
        for (int t = LO; t < HI; ++t) f[t] = tiles(Bs, t);
        mma_right<Op, LO, HI>(kf, f, dk);
      });
      return;
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int tt = 16 * t + n;
      for (int s = 0; s < C; ++s) {
        if (FRONT ? s > tt : s < tt) continue;
        const int r = FRONT ? tt : s, c = FRONT ? s : tt, at = tile_of(r / 16, c / 16) * 256 + Op::tile_at(r % 16, c % 16);
        const float wa = Op::whole(As + at, PLANE), wb = Op::whole(Bs + at, PLANE);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float kk = to_f(Ks[Op::at(s, r0 + 4 * g + i, KS)]), qq = to_f(Qs[Op::at(s, r0 + 4 * g + i, KS)]);
          if (FRONT && wa != 0.0f) dq[t][i] = fmaf(wa, kk, dq[t][i]);
          if (!FRONT && wa != 0.0f) dk[t][i] = fmaf(wa, qq, dk[t][i]);
          if (s != tt && wb != 0.0f) dk[t][i] = fmaf(wb, kk, dk[t][i]);
        }
      }
    }
  };
  products(std::true_type{});
  __syncthreads();  // Qd and Kd; the tiles have been read
  {
    int turn = 0;
#pragma unroll
    for (int ti = 0; ti < TT; ++ti)
#pragma unroll
      for (int si = 0; si <= ti; ++si, ++turn) {
        if (turn % WAVES != wave) continue;
        const int tile = tile_of(ti, si) * 256 + Op::tile_at(n, 4 * g);
        Op::put_wide(As + tile, PLANE, lt[turn / WAVES]);
        Op::put_wide(Bs + tile, PLANE, mt[turn / WAVES]);
      }
  }
  __syncthreads();
  products(std::false_type{});
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int tt = 16 * t + n;
    const float rk = Row[RK][tt], rq = Row[RQ][tt];
    if (A.normalize) {  // the part along the vector itself is no change
      const auto q4 = four(Qs, tt), k4 = four(Ks, tt);
      const float along_q = -Qd[tt] * (rq * rq), along_k = -Kd[tt] * rk;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dq[t][i] = fmaf(to_f(q4.v[i]), along_q, dq[t][i] * (rq * A.scale));
        dk[t][i] = rk * fmaf(to_f(k4.v[i]), along_k, dk[t][i]);
      }
    } else {
      dq[t] *= A.scale;
    }
    if (tt >= left) continue;
    const int64_t at = ((b * A.T + t0 + tt) * A.H + h) * A.kd + r0 + 4 * g;
    auto store = [&](auto* to, const f32x4& x) {
      using Y = std::remove_pointer_t<decltype(to)>;
      Y f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = from_f<Y>(x[i]);
      if (A.wide_dqk && r0 + 4 * g < A.kd) {
        __builtin_memcpy(__builtin_assume_aligned(to + at, 4 * sizeof(Y)), f, sizeof(f));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r0 + 4 * g + i < A.kd) to[at + i] = f[i];
      }
    };
    if (A.dq) {
      if (A.dq_f32) store(static_cast<float*>(A.dq), dq[t]);
      else store(static_cast<T*>(A.dq), dq[t]);
    }
    if (A.dk) {
      if (A.dk_f32) store(static_cast<float*>(A.dk), dk[t]);
      else store(static_cast<T*>(A.dk), dk[t]);
    }
  }
}

// ---- launches --------------------------------------------------------------------------------------------------

template <class T, int KD, int WAVES, bool BACK, bool STATE>
int launch_delta_part(const Delta& A, hipStream_t s) {
  constexpr int COLS = 16 * WAVES;
  Delta P = A;
  P.colblocks = (int)ceil_div(A.vd, COLS);
  const int blocks = STATE && !BACK ? P.colblocks + (KD + COLS - 1) / COLS : P.colblocks;
  return in_launches(A.B * A.H * A.segs * blocks, WAVES * 64, [&](int64_t first, dim3 grid) {
    P.first = first / blocks;
    hipLaunchKernelGGL((delta_sweep_kernel<T, KD, WAVES, BACK, STATE>), grid, dim3(WAVES * 64), 0, s, P);
  }, blocks);
}

template <class T, int KD, int WAVES, bool BACK>
int launch_delta_sweep(const Delta& A, hipStream_t s) {
  if (A.segs > 1) {
    if (const int rc = launch_delta_part<T, KD, WAVES, BACK, true>(A, s)) return rc;
    if (const int rc = launch_delta_join(A, BACK, s)) return rc;
  }
  return launch_delta_part<T, KD, WAVES, BACK, false>(A, s);
}

template <class T, int KD, bool BACK>
int launch_delta_sweeps(const Delta& A, hipStream_t s) {
  if (A.vd <= 32) return launch_delta_sweep<T, KD, 2, BACK>(A, s);
  return launch_delta_sweep<T, KD, 4, BACK>(A, s);
}

template <class T, int KD>
int launch_delta_gradients(const Delta& A, hipStream_t s) {
  return in_launches(A.B * A.H * A.chunks, KD / 16 * 64, [&](int64_t first, dim3 grid) {
    Delta P = A;
    P.first = first;
    hipLaunchKernelGGL((delta_gradients_kernel<T, KD>), grid, dim3(KD / 16 * 64), 0, s, P);
  });
}

template <class T, int KD>
int launch_delta(const Delta& A, int what, hipStream_t s) {
  if (what == PREPARE)
    return in_launches(A.B * A.H * A.chunks, 256, [&](int64_t first, dim3 grid) {
      Delta P = A;
      P.first = first;
      hipLaunchKernelGGL((delta_prepare_kernel<T, KD>), grid, dim3(256), 0, s, P);
    });
  if (what == SWEEP) return launch_delta_sweeps<T, KD, false>(A, s);
  if (what == SWEEP_BACK) return launch_delta_sweeps<T, KD, true>(A, s);
  return launch_delta_gradients<T, KD>(A, s);
}

}  // namespace ttc

#define TTC_DELTA_UNIT(T, KD)                                                                                        \
  namespace ttc {                                                                                                    \
  template <>                                                                                                        \
  int launch_delta_kd##KD<T>(const Delta& A, int what, hipStream_t s) { return launch_delta<T, KD>(A, what, s); }   \
  }
