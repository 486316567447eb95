// ttc_ops_common.hpp -- types, conversions and reductions shared by the sequence operators' kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "ttc_lqr.h"
#include "ttc_ops.h"

namespace ttc {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__bf16 x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_f(float x) { return (T)x; }  // bf16: to nearest, ties to even

// sum over aligned groups of `width` lanes (a power of two up to 64), in every lane
__device__ __forceinline__ float lane_sum(float v, int width) {
  for (int m = width >> 1; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? TTC_LQR_OK : TTC_LQR_ELAUNCH; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// whether sizes of at least 0 have a product of at most 2^58, so that byte counts and offsets of several such arrays
// stay within 64 bits
inline bool countable(std::initializer_list<int64_t> sizes) {
  __int128 p = 1;
  for (int64_t v : sizes) {
    p *= v > 1 ? v : 1;  // an empty array's other sizes are bounded too
    if (p > ((__int128)1 << 58)) return false;
  }
  return true;
}

// A launch of 2^32 threads or more does not run whole: the workgroups that one launch can have
inline int64_t max_blocks(int threads) { return ((int64_t)1 << 32) / threads - 1; }

// go(first workgroup, workgroups) for as many launches as that takes, each of a multiple of `unit` workgroups
template <class F>
int in_launches(int64_t blocks, int threads, F go, int64_t unit = 1) {
  const int64_t most = max_blocks(threads) / unit * unit;
  for (int64_t first = 0; first < blocks; first += most) {
    const int64_t left = blocks - first;
    go(first, dim3((unsigned)(left < most ? left : most)));
    if (const int rc = launched()) return rc;
  }
  return TTC_LQR_OK;
}

}  // namespace ttc
