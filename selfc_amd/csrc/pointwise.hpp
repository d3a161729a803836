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

// Eight consecutive values of a row as fp32.  VEC: 16-byte loads (base and row pitch aligned); else element by element, so that
// any width, offset and pitch is read in place.  Values from `left` on are not read and come back as 0.
template <typename T>
__device__ __forceinline__ void load8(const T* const p, const long left, const bool vec, float* const out) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { out[i] = a[i]; out[4 + i] = b[i]; }
    } else {
      typedef T v8 __attribute__((ext_vector_type(8)));
      const v8 a = *reinterpret_cast<const v8*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = (float)a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < left ? (float)p[i] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* const p, const long left, const bool vec, const float* const v) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      typedef T v8 __attribute__((ext_vector_type(8)));
      v8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
      *reinterpret_cast<v8*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)v[i];
  }
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
