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
inline bool aligned_to(const void* p, const size_t bytes) { return ((size_t)p & (bytes - 1)) == 0; }

// Eight consecutive values of a row, at any address their type allows (the memory pipeline takes 16-byte accesses at 2-byte addresses):
// `left` values of the row lie at and behind p, `before` in front of it.  Behind the row nothing is read: where it ends inside the
// eight, the row's last eight are read and shifted down.  Values from `left` on come back as 0.
template <typename T>
__device__ __forceinline__ u32x4 raw8(const T* const p, const int left, const int before) {
  static_assert(sizeof(T) == 2, "16-bit values");
  u32x4 r = {0, 0, 0, 0};
  if (left >= 8) {
    __builtin_memcpy(&r, p, 16);
  } else if (left > 0) {
    if (before >= 8) {
      unsigned long long v[2];
      __builtin_memcpy(v, p - (8 - left), 16);
      const int down = (8 - left) * 16;
      const unsigned long long lo = down < 64 ? v[0] >> down | v[1] << (64 - down) : v[1] >> (down - 64), hi = down < 64 ? v[1] >> down : 0;
      r = u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
    } else {
      const unsigned short* const u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) r[i / 2] |= (unsigned)u[i] << (16 * (i & 1));
    }
  }
  return r;
}
// the same for a later expansion: what a prefetch keeps in registers
template <typename T>
struct Raw8 {
  u32x4 v;
  __device__ __forceinline__ void load(const T* const p, const int left, const int before) { v = raw8(p, left, before); }
  __device__ __forceinline__ void expand(float* const out) const {
    typedef T v8 __attribute__((ext_vector_type(8)));
    const v8 a = __builtin_bit_cast(v8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (float)a[i];
  }
};
template <>
struct Raw8<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* const p, const int left, const int) {
    if (left >= 8) {
      __builtin_memcpy(v, p, 32);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
  }
  __device__ __forceinline__ void expand(float* const out) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = v[i];
  }
};
template <typename T>
__device__ __forceinline__ void load8(const T* const p, const long left, const long before, float* const out) {
  if constexpr (sizeof(T) == 2) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    const v8 a = __builtin_bit_cast(v8, raw8(p, left > 8 ? 8 : (int)left, before > 8 ? 8 : (int)before));
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (float)a[i];
  } else if (left >= 8) {
    float a[8];
    __builtin_memcpy(a, p, 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* const p, const long left, const float* const v) {
  T a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
  if (left >= 8) {
    __builtin_memcpy(p, a, sizeof(a));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = a[i];
  }
}

// Sums and maxima over groups of L consecutive lanes (L a power of two up to 64); every lane gets the same result.  Partner lanes come
// through the data-parallel paths of the vector unit (a lane's neighbours, mirrored halves, exchanged rows), not through shared memory.
struct OpSum { static __device__ __forceinline__ float run(const float a, const float b) { return a + b; } };
struct OpMax {
  static __device__ __forceinline__ float run(const float a, const float b) { return fmaxf(a, b); }
  static __device__ __forceinline__ unsigned run(const unsigned a, const unsigned b) { return a > b ? a : b; }
};
template <int CTRL, typename V>
__device__ __forceinline__ V dpp(const V v) {
  return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L, typename OP, typename V>
__device__ __forceinline__ V lanes_op(V v) {
  if constexpr (L > 1) v = OP::run(v, dpp<0xB1>(v));           // quad_perm [1, 0, 3, 2]
  if constexpr (L > 2) v = OP::run(v, dpp<0x4E>(v));           // quad_perm [2, 3, 0, 1]
  if constexpr (L > 4) v = OP::run(v, dpp<0x141>(v));          // row_half_mirror: the other four of eight
  if constexpr (L > 8) v = OP::run(v, dpp<0x140>(v));          // row_mirror: the other eight of sixteen
  if constexpr (L > 16) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const u32x2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];           // (a bit cast of a vector's element takes element 0)
    v = OP::run(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
  }
  if constexpr (L > 32) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const u32x2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    v = OP::run(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
  }
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(const float v) { return lanes_op<L, OpSum>(v); }
template <int L, typename V>
__device__ __forceinline__ V lanes_max(const V v) { return lanes_op<L, OpMax>(v); }

}  // namespace selfc
