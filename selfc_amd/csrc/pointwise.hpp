// What the kernels of adamw.hip, rmsnorm.hip and linear.hip share: the caller's number types (chosen per call, apart from the
// operand type this library is built for), 8-value vectors of them, sums and maxima over lanes.
#pragma once
#include "common.hpp"
#include "../../include/selfc_hip.h"

namespace selfc {

typedef _Float16 h16;
typedef __bf16 b16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

inline int pw_rc(const hipError_t e) { return e == hipSuccess ? 0 : -(int)e - 1000; }
__device__ __forceinline__ bool aligned16(const void* p) { return ((size_t)p & 15) == 0; }
inline bool aligned_to(const void* p, const size_t bytes) { return ((size_t)p & (bytes - 1)) == 0; }

// Eight consecutive values of a row as fp32, `run` values (8, 4, 2 or 1) per load: the largest that base, pitch and width are multiples
// of, so that rows of any width, offset and pitch are read in place.  Values from `left` on are not read and come back as 0.
template <int R, typename T>
__device__ __forceinline__ void load8_runs(const T* const p, const long left, float* const out) {
  typedef T vr __attribute__((ext_vector_type(R)));
#pragma unroll
  for (int k = 0; k < 8; k += R) {
    vr a = {};
    if (k < left) a = *reinterpret_cast<const vr*>(p + k);
#pragma unroll
    for (int i = 0; i < R; ++i) out[k + i] = (float)a[i];
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* const p, const long left, const int run, float* const out) {
  if (run == 8) {
    if constexpr (sizeof(T) == 4) load8_runs<4>(p, left, out);
    else load8_runs<8>(p, left, out);
  } else if (run == 4) {
    load8_runs<4>(p, left, out);
  } else if (run == 2) {
    load8_runs<2>(p, left, out);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < left ? (float)p[i] : 0.f;
  }
}

template <int R, typename T>
__device__ __forceinline__ void store8_runs(T* const p, const long left, const float* const v) {
  typedef T vr __attribute__((ext_vector_type(R)));
#pragma unroll
  for (int k = 0; k < 8; k += R) {
    vr a;
#pragma unroll
    for (int i = 0; i < R; ++i) a[i] = (T)v[k + i];
    if (k < left) *reinterpret_cast<vr*>(p + k) = a;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* const p, const long left, const int run, const float* const v) {
  if (run == 8) {
    if constexpr (sizeof(T) == 4) store8_runs<4>(p, left, v);
    else store8_runs<8>(p, left, v);
  } else if (run == 4) {
    store8_runs<4>(p, left, v);
  } else if (run == 2) {
    store8_runs<2>(p, left, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}
// the run that a base, a pitch and a width (both in values of `es` bytes) allow
inline int row_run(const void* const p, const size_t pitch, const size_t width, const size_t es) {
  for (int r = 8; r > 1; r >>= 1)
    if (pitch % r == 0 && width % r == 0 && ((size_t)p & ((r * es < 16 ? r * es : 16) - 1)) == 0) return r;
  return 1;
}

// butterflies over groups of L consecutive lanes (L a power of two up to 64): every lane gets the same result
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

}  // namespace selfc
