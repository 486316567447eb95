// ttc_ops_mfma.hpp -- operands of the matrix instructions for the sequence operators' chunked kernels: reads of shared
// memory as operands, values as sums of bf16 numbers, scores in tiles, loads that are bounded instead of branching.
#pragma once
#include "ttc_ops_common.hpp"

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
  static __device__ __forceinline__ f32x4 mma(const Wide& a, const Wide& b, f32x4 c) {  // 24 digits of the product
    c = mma(a.m, b.m, mma(a.l, b.h, mma(a.h, b.l, c)));
    return mma(a.h, b.h, mma(a.h, b.m, mma(a.m, b.h, c)));
  }
  // A product as single instructions, small terms first: those of several sums are issued in turn, so that none waits for the
  // one before it
  static constexpr int steps(const Frag*, const Wide*) { return 3; }
  static constexpr int steps(const Wide*, const Frag*) { return 3; }
  static constexpr int steps(const Wide*, const Wide*) { return 6; }
  static __device__ __forceinline__ f32x4 step(int p, Frag a, const Wide& b, f32x4 c) {
    return mma(a, p == 0 ? b.l : p == 1 ? b.m : b.h, c);
  }
  static __device__ __forceinline__ f32x4 step(int p, const Wide& a, Frag b, f32x4 c) {
    return mma(p == 0 ? a.l : p == 1 ? a.m : a.h, b, c);
  }
  static __device__ __forceinline__ f32x4 step(int p, const Wide& a, const Wide& b, f32x4 c) {
    return mma(p == 1 ? a.l : p == 2 || p == 3 ? a.m : a.h, p == 0 ? b.l : p == 2 || p == 4 ? b.m : b.h, c);
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
  // Rows of 8 banks' distance that are read along them and across them: 8 bytes of a row change places with its number / 4, so
  // that both reads meet each bank once.  at: where an element of such an array (of tile_at: of a 16 x 16 tile) lies
  static __device__ __forceinline__ int at(int row, int c, int stride) { return row * stride + (c ^ ((row >> 2 & 3) << 2)); }
  static __device__ __forceinline__ int tile_at(int row, int c) { return row * 16 + (c ^ (row & 12)); }
  static __device__ __forceinline__ int mixed_place(int row, int c, int stride) { return row * stride + (c ^ (row & 8)); }
  static __device__ __forceinline__ u32x4 mixed(int row, u32x4 v) {  // 8 elements as they lie there
    const bool swap = row & 4;
    return u32x4{swap ? v[2] : v[0], swap ? v[3] : v[1], swap ? v[0] : v[2], swap ? v[1] : v[3]};
  }
  // A lane's place for `row_split` (row n, elements 4 g on) and for `column_mixed` (as `column`); whole rows and multiples of 16
  // elements are added to it
  static __device__ __forceinline__ int row_place(int stride, int lane) { return at(lane & 15, lane >> 4 << 2, stride); }
  static __device__ __forceinline__ int column_place(int stride, int lane) {
    return at((lane >> 4 << 2) + (lane >> 2 & 3), (lane & 3) * 4, stride);
  }
  static __device__ __forceinline__ Frag column_mixed(const __bf16* a, int stride) {
    typedef __attribute__((address_space(3))) i16x4 lds;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a));
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(a + 16 * stride));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // Values in memory as their three parts (WIDE_PARTS such arrays, `part` elements apart): 4 neighbours put at p, and two
  // 16 x 16 tiles as an operand (zeros for one that is not there): rows n of both, or of their transposes
  static constexpr int WIDE_PARTS = 3;
  static __device__ __forceinline__ void put_wide(__bf16* p, int part, f32x4 x) {
    float d[4], e[4];
    const u32x2 h = {cut(x[0], x[1], d[0], d[1]), cut(x[2], x[3], d[2], d[3])};
    const u32x2 m = {cut(d[0], d[1], e[0], e[1]), cut(d[2], d[3], e[2], e[3])};
    *reinterpret_cast<u32x2*>(p) = h;
    *reinterpret_cast<u32x2*>(p + part) = m;
    *reinterpret_cast<bf16x4*>(p + 2 * part) = bf16x4{(__bf16)e[0], (__bf16)e[1], (__bf16)e[2], (__bf16)e[3]};
  }
  template <bool ROW>
  static __device__ __forceinline__ Frag tiles(bool has_a, const __bf16* a, bool has_b, const __bf16* b, int lane) {
    const int g = lane >> 4, i = lane & 15;
    typedef __attribute__((address_space(3))) i16x4 lds;
    auto one = [&](const __bf16* p) {
      if (ROW) return *reinterpret_cast<const i16x4*>(p + tile_at(i, 4 * g));
      return (i16x4)__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(p + tile_at(4 * g + (i >> 2), (i & 3) * 4)));
    };
    const i16x4 x = has_a ? one(a) : i16x4{0, 0, 0, 0}, y = has_b ? one(b) : i16x4{0, 0, 0, 0};
    return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  template <bool ROW>
  static __device__ __forceinline__ Wide wide_tiles(bool has_a, const __bf16* a, bool has_b, const __bf16* b, int part, int lane) {
    return Wide{tiles<ROW>(has_a, a, has_b, b, lane), tiles<ROW>(has_a, a + part, has_b, b + part, lane),
                tiles<ROW>(has_a, a + 2 * part, has_b, b + 2 * part, lane)};
  }
  static __device__ __forceinline__ float whole(const __bf16* p, int part) { return to_f(p[0]) + (to_f(p[part]) + to_f(p[2 * part])); }
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
  static constexpr int steps(const Frag*, const Frag*) { return 8; }
  static __device__ __forceinline__ f32x4 step(int p, const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[p], b.v[p], c, 0, 0, 0);
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
  static __device__ __forceinline__ int at(int row, int c, int stride) { return row * stride + c; }
  static __device__ __forceinline__ int tile_at(int row, int c) { return row * 16 + c; }
  static __device__ __forceinline__ int mixed_place(int row, int c, int stride) { return row * stride + c; }
  static __device__ __forceinline__ u32x4 mixed(int, u32x4 v) { return v; }
  static __device__ __forceinline__ int row_place(int stride, int lane) { return (lane & 15) * stride + (lane >> 4 << 2); }
  static __device__ __forceinline__ int column_place(int stride, int lane) { return (lane >> 4 << 2) * stride + (lane & 15); }
  static __device__ __forceinline__ Frag column_mixed(const float* a, int stride) {
    Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = a[(j < 4 ? j : 12 + j) * stride];
    return r;
  }
  static constexpr int WIDE_PARTS = 1;
  static __device__ __forceinline__ void put_wide(float* p, int, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }
  template <bool ROW>
  static __device__ __forceinline__ Frag wide_tiles(bool has_a, const float* a, bool has_b, const float* b, int, int lane) {
    const int g = lane >> 4, n = lane & 15;
    Frag r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = ROW ? n * 16 + 4 * g + j : (4 * g + j) * 16 + n;
      r.v[j] = has_a ? a[at] : 0.0f;
      r.v[4 + j] = has_b ? b[at] : 0.0f;
    }
    return r;
  }
  static __device__ __forceinline__ float whole(const float* p, int) { return p[0]; }
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

}  // namespace ttc
