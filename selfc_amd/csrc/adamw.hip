// AdamW over a list of tensors in as few launches as the kernel-argument segment allows, with the moments in 32 or in 8 bits,
// and the global norm of a list of gradients.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))            (only with max_norm)
//   m' = b1 m + (1 - b1) g',   v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Arithmetic in fp32, every operation of the moments rounded by itself (no contraction): in 8 bits the outcome of a comparison
// hangs on their last bit, and this way it is the same for every implementation of the formulas above.
//
// The moments of all tensors live in one buffer each; a tensor starts at a multiple of 256 values, so a block of 256 belongs to
// one tensor.  In 8 bits each block has two power-of-two scales.  m is held as e4m3 (largest value of the block in [128, 256)
// steps of its scale), v as e5m2 (in [2^14, 2^15)): v spans twice the octaves that m does, because it is m's square.
// Rounding: v moves by 0.1 % of itself per step at b2 = 0.999 while a step of its code is 12 to 25 % - rounded to nearest it would
// never move.  So a value is rounded down after adding u steps, u in [0, 1) from an integer hash of (seed, step, tensor, place):
// right on average.  With scales that are powers of two a value that is on the grid stays on it when the scale changes, so the
// noise enters only with the few values that move (a fixed grid moves with probability 0.001 |g^2/v - 1| / 0.18 per step: about
// 30 % standard deviation of v, 15 % of the step's size, against 160 % if every step re-rounded every value).  A nonzero v never
// rounds to zero: m / sqrt(v) stays bounded.  Values that are not finite are held as NaN and do not enter their block's scale.
//
// Bound: memory (28 bytes a value in 32 bits; 16 in 8 bits with fp32 tensors, 10 with 16-bit ones), as long as the 8-bit form stays below
// about 100 vector instructions a value: its first form, with every value's end-of-tensor check and general rounding, took 106 and
// was bound by them (134 M bf16 values: 382 us).  Measured for 134 M values in 20 tensors: 32 bits with fp32 tensors 707 us (3.76 GB, 5.3 TB/s, a
// large copy's rate), with bf16 ones 557 (3.0 GB), 8 bits with bf16 ones 250 us (1.35 GB, 5.4 TB/s), with fp32 ones 397 (2.2 GB); the norm of the gradients in front
// of a clipped step 91 (fp32), 49 (bf16).  A single layer's five tensors 3.7 us.  Step numbers on the device cost every lane two powers in fp64: nothing next
// to 32-bit moments, 8 bits with bf16 tensors 250 -> 264 us.
#include "pointwise.hpp"
#include <math.h>

namespace selfc {
namespace {

constexpr int AW_BLOCK = 256;              // values per scale; also what one wave handles at a time, four consecutive ones per lane
constexpr int AW_U = 4;                    // blocks per wave: their loads are in flight together
constexpr int AW_CHUNK = 4 * AW_U * AW_BLOCK;
constexpr int AW_MAX = 96;                 // tensors per launch: 96 entries of 40 bytes stay below 4 KiB of kernel arguments

struct AwEntry { void* p; const void* g; const float* step; unsigned long long n; unsigned block0, wg0; };
struct AwTable {
  AwEntry e[AW_MAX];
  int count, place0;
};
struct AwHyper {
  const float *lr_dev, *norm;
  double beta1_d, beta2_d;
  float lr, bc1, bc2s, b1, omb1, b2, omb2, eps, wd, max_norm;
  unsigned seed, key;
};

__host__ __device__ inline unsigned aw_mix(unsigned x) {        // multipliers: digits of pi
  x ^= x >> 16; x *= 0x85A308D3u;
  x ^= x >> 15; x *= 0x13198A2Fu;
  return x ^ (x >> 16);
}
__host__ __device__ inline double aw_pow(double b, unsigned long long e) {
  double r = 1.0;
  for (; e; e >>= 1, b *= b)
    if (e & 1) r *= b;
  return r;
}

// which tensor of the table holds workgroup `wg`: entries start at ascending workgroups, two entries per lane
__device__ __forceinline__ int aw_find(const AwTable& t, const unsigned wg) {
  const int lane = threadIdx.x & 63;
  const bool a = lane < t.count && t.e[lane].wg0 <= wg;
  const int j = lane + 64;
  const bool b = j < t.count && t.e[j < AW_MAX ? j : 0].wg0 <= wg;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(a)) + __popcll(__ballot(b)) - 1);
}

// biased exponent of a block's scale 2^(floor(log2 most) - top), not below 2^-126; of 1 for an empty block
__device__ __forceinline__ int aw_exponent(const unsigned most, const int top) {
  const int e = (int)(most >> 23) - top;
  return most == 0 ? 127 : e < 1 ? 1 : e;
}

// |y| rounded down after adding u steps of the 8-bit format's grid (least: exponent of its smallest normal number, digits: of its
// mantissa); not a number if y is not finite
template <int LEAST, int DIGITS, bool FLOOR>
__device__ __forceinline__ float aw_round(const float y, const float u) {
  const unsigned ay = __builtin_bit_cast(unsigned, y) & 0x7fffffffu;
  int e = (int)(ay >> 23);
  e = e < 127 + LEAST ? 127 + LEAST : e;
  const float q = __builtin_bit_cast(float, (unsigned)(e - DIGITS) << 23);
  const float iq = __builtin_bit_cast(float, (unsigned)(254 - e + DIGITS) << 23);
  float k = floorf(__builtin_bit_cast(float, ay) * iq + u);
  if (FLOOR) k = ay ? fmaxf(k, 1.f) : k;
  const float r = __builtin_copysignf(k * q, y);
  return ay < 0x7f800000u ? r : __builtin_nanf("");
}

// Four moments -> 8 bits with the block's scale.  x[i]: the dither's 16 bits.  For normal numbers of the 8-bit format, adding u steps and
// rounding down is an integer addition below the kept digits and a mask; a block that holds smaller ones (or some that are not finite)
// takes the general form.
template <int TOP, int LEAST, int DIGITS, bool FLOOR>
__device__ __forceinline__ float aw_hold(const float* const m, const unsigned* const x, float* const q) {
  unsigned a[4], most = 0, least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = __builtin_bit_cast(unsigned, m[i]) & 0x7fffffffu;
    most = a[i] > most ? a[i] : most;
    least = a[i] - 1 < least ? a[i] - 1 : least;             // the smallest that is not 0, less one
  }
  most = lanes_max<64>(most);
  int e = aw_exponent(most, TOP);
  const int floor_e = e + LEAST;                             // exponent of the smallest moment that is a normal number of the format
  bool plain = most < 0x7f800000u && floor_e >= 1;
  if (plain) plain = __all(least >= ((unsigned)floor_e << 23) - 1);
  if (plain) {
    const float inv = __builtin_bit_cast(float, (unsigned)(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = m[i] * inv;
      q[i] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, y) + (x[i] << (23 - DIGITS - 16))) & (0xffffffffu << (23 - DIGITS)));
    }
  } else {
    most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = a[i] < 0x7f800000u && a[i] > most ? a[i] : most;
    e = aw_exponent(lanes_max<64>(most), TOP);
    const float inv = __builtin_bit_cast(float, (unsigned)(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = aw_round<LEAST, DIGITS, FLOOR>(m[i] * inv, (float)x[i] * 0x1p-16f);
  }
  return __builtin_bit_cast(float, (unsigned)e << 23);
}

// what a step's number, rate and norm make of the formulas; small: subnormal moments count
struct AwStep { float keep, rate, ibc2, coef; unsigned key; bool small; };

// m / (sqrt(v) ibc2 + eps) where a root or a denominator may be too small for the root's and the reciprocal's instructions, which take
// subnormal numbers for 0
__device__ __forceinline__ float aw_ratio(const float m, const float v, const float ibc2, const float eps) {
  const bool low = v < 0x1p-96f;
  const float root = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v) * (low ? 0x1p-32f : 1.f);
  const float den = fmaf(root, ibc2, eps);
  const float up = den < 0x1p-96f ? 0x1p64f : 1.f;
  return m * up * __builtin_amdgcn_rcpf(den * up);
}

// 256 values of a tensor, four consecutive ones per lane.  FULL: all of them exist and p and g are aligned.
template <typename T, int BITS, bool FULL>
struct AwPart {
  typedef T T4 __attribute__((ext_vector_type(4)));
  float p[4], g[4], m[4], v[4];
  // pt, gt: the tensor's first value of this part; left: how many it has; st: the part's first value in the state, bk: its block
  __device__ __forceinline__ void load(const T* const pt, const T* const gt, const unsigned long long left, const void* const ms, const void* const vs,
                                       const float* const sm, const float* const sv, const int lane) {
    const int at = lane * 4;
    if (FULL) {
      const T4 a = *reinterpret_cast<const T4*>(pt + at), b = *reinterpret_cast<const T4*>(gt + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) { p[i] = (float)a[i]; g[i] = (float)b[i]; }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = (unsigned)(at + i) < left ? (float)pt[at + i] : 0.f;
        g[i] = (unsigned)(at + i) < left ? (float)gt[at + i] : 0.f;
      }
    }
    if constexpr (BITS == 32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>((const float*)ms + at), b = *reinterpret_cast<const f32x4*>((const float*)vs + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) { m[i] = a[i]; v[i] = b[i]; }
    } else {
      const unsigned m8 = *reinterpret_cast<const unsigned*>((const unsigned char*)ms + at), v8 = *reinterpret_cast<const unsigned*>((const unsigned char*)vs + at);
      const float ss = *sm, qs = *sv;
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(m8, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(m8, true);
      const f32x2 c = __builtin_amdgcn_cvt_pk_f32_bf8(v8, false), d = __builtin_amdgcn_cvt_pk_f32_bf8(v8, true);
      m[0] = a[0] * ss; m[1] = a[1] * ss; m[2] = b[0] * ss; m[3] = b[1] * ss;
      v[0] = c[0] * qs; v[1] = c[1] * qs; v[2] = d[0] * qs; v[3] = d[1] * qs;
    }
  }
  __device__ __forceinline__ void step(T* const pt, const unsigned long long left, const unsigned place, void* const ms, void* const vs,
                                       float* const sm, float* const sv, const int lane, const AwStep& s, const AwHyper& hy) {
#pragma clang fp contract(off)
    const int at = lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float gi = g[i];
      if (hy.norm) gi = gi * s.coef;
      m[i] = hy.b1 * m[i] + hy.omb1 * gi;
      v[i] = hy.b2 * v[i] + hy.omb2 * (gi * gi);
    }
    // one-ulp square root and reciprocal: the step is a small part of p, its last bits are below p's
    if (!s.small) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float den = fmaf(__builtin_amdgcn_sqrtf(v[i]), s.ibc2, hy.eps);
        p[i] = fmaf(-s.rate, m[i] * __builtin_amdgcn_rcpf(den), p[i] * s.keep);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = fmaf(-s.rate, aw_ratio(m[i], v[i], s.ibc2, hy.eps), p[i] * s.keep);
    }
    if (FULL) {
      *reinterpret_cast<T4*>(pt + at) = T4{(T)p[0], (T)p[1], (T)p[2], (T)p[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((unsigned)(at + i) < left) pt[at + i] = (T)p[i];
    }
    if constexpr (BITS == 32) {
      if (FULL) {
        *reinterpret_cast<f32x4*>((float*)ms + at) = f32x4{m[0], m[1], m[2], m[3]};
        *reinterpret_cast<f32x4*>((float*)vs + at) = f32x4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((unsigned)(at + i) < left) { ((float*)ms)[at + i] = m[i]; ((float*)vs)[at + i] = v[i]; }
      }
    } else {
      if (!FULL)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((unsigned)(at + i) >= left) m[i] = v[i] = 0.f;               // behind the tensor's end: as they were
      unsigned um[4], uv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned x = aw_mix((place + at + i) ^ s.key);
        um[i] = x & 0xffffu;
        uv[i] = x >> 16;
      }
      float mq[4], vq[4];
      const float ss = aw_hold<7, -6, 3, false>(m, um, mq), qs = aw_hold<14, -14, 2, true>(v, uv, vq);
      int a = __builtin_amdgcn_cvt_pk_fp8_f32(mq[0], mq[1], 0, false);
      a = __builtin_amdgcn_cvt_pk_fp8_f32(mq[2], mq[3], a, true);
      int b = __builtin_amdgcn_cvt_pk_bf8_f32(vq[0], vq[1], 0, false);
      b = __builtin_amdgcn_cvt_pk_bf8_f32(vq[2], vq[3], b, true);
      *reinterpret_cast<int*>((unsigned char*)ms + at) = a;
      *reinterpret_cast<int*>((unsigned char*)vs + at) = b;
      if (lane == 0) { *sm = ss; *sv = qs; }
    }
  }
};

template <typename T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const AwTable tab, const AwHyper hy, void* const m_, void* const v_,
                                                    float* const ms, float* const vs) {
  const unsigned wg = blockIdx.x;
  const int ti = aw_find(tab, wg);
  const AwEntry& en = tab.e[ti];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned long long n = en.n;
  const unsigned long long base = (unsigned long long)(wg - en.wg0) * AW_CHUNK + (unsigned)wave * (AW_U * AW_BLOCK);
  if (base >= n) return;
  T* const p = (T*)en.p + base;
  const T* const g = (const T*)en.g + base;
  const size_t blk0 = (size_t)en.block0 + (size_t)(base / AW_BLOCK);       // first of this wave's blocks in the state
  constexpr int SB = BITS / 8;
  unsigned char* const m = (unsigned char*)m_ + blk0 * AW_BLOCK * SB;
  unsigned char* const v = (unsigned char*)v_ + blk0 * AW_BLOCK * SB;
  float* const sm = ms + blk0;
  float* const sv = vs + blk0;
  const unsigned long long left = n - base;
  const bool full = left >= AW_U * AW_BLOCK && (((size_t)p | (size_t)g) & (4 * sizeof(T) - 1)) == 0;

  AwPart<T, BITS, true> part[AW_U];
  if (full) {
#pragma unroll
    for (int u = 0; u < AW_U; ++u)
      part[u].load(p + u * AW_BLOCK, g + u * AW_BLOCK, AW_BLOCK, m + u * AW_BLOCK * SB, v + u * AW_BLOCK * SB, sm + u, sv + u, lane);
  }
  // from the host, or (captured steps) from device memory
  float bc1 = hy.bc1, bc2s = hy.bc2s;
  AwStep s;
  s.key = hy.key;
  if (en.step) {
    const unsigned long long t = (unsigned long long)*en.step;
    bc1 = (float)(1.0 - aw_pow(hy.beta1_d, t));
    bc2s = (float)sqrt(1.0 - aw_pow(hy.beta2_d, t));
    s.key = aw_mix(hy.seed ^ aw_mix((unsigned)t));
  }
  const float lr = hy.lr_dev ? *hy.lr_dev : hy.lr;
  s.keep = 1.f - lr * hy.wd;
  s.rate = lr / bc1;
  s.ibc2 = 1.f / bc2s;
  s.small = hy.eps < s.ibc2 * 0x1p-39f;      // else the root of a subnormal v, below 2^-63, is less than 2^-24 of eps after its correction
  s.coef = 1.f;
  if (hy.norm) {                             // a norm that is not a number leaves none behind: min(1, NaN) is NaN here
    const float c = hy.max_norm / (*hy.norm + 1e-6f);
    s.coef = c >= 1.f ? 1.f : c;
  }
  s.key = aw_mix(s.key ^ aw_mix((unsigned)(tab.place0 + ti)));

  if (full) {
#pragma unroll
    for (int u = 0; u < AW_U; ++u)
      part[u].step(p + u * AW_BLOCK, AW_BLOCK, (unsigned)base + u * AW_BLOCK, m + u * AW_BLOCK * SB, v + u * AW_BLOCK * SB, sm + u, sv + u, lane, s, hy);
  } else {
    AwPart<T, BITS, false> one;
#pragma unroll 1
    for (int u = 0; u < AW_U && (unsigned long long)u * AW_BLOCK < left; ++u) {
      const unsigned long long l = left - u * AW_BLOCK;
      one.load(p + u * AW_BLOCK, g + u * AW_BLOCK, l, m + u * AW_BLOCK * SB, v + u * AW_BLOCK * SB, sm + u, sv + u, lane);
      one.step(p + u * AW_BLOCK, l, (unsigned)base + u * AW_BLOCK, m + u * AW_BLOCK * SB, v + u * AW_BLOCK * SB, sm + u, sv + u, lane, s, hy);
    }
  }
}

// ---- |g| over a list: per-workgroup sums of squares in fp64 (an fp32 square overflows from 2^64 on), then one workgroup adds them
// in a fixed order
constexpr int GN_WG = 1024;
template <typename T>
__global__ __launch_bounds__(256) void grad_norm_kernel(const AwTable tab, const unsigned chunks, double* const partial) {
  double acc = 0.0;
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const AwEntry& en = tab.e[aw_find(tab, c)];
    const T* const g = (const T*)en.g;
    const unsigned long long base = (unsigned long long)(c - en.wg0) * AW_CHUNK;
    const unsigned long long left = en.n - base;
    const T* const q = g + base;
#pragma unroll
    for (int j = 0; j < AW_CHUNK / 2048; ++j) {
      const long at = j * 2048 + threadIdx.x * 8;
      if ((unsigned long long)at < left) {
        float v[8];
        const unsigned long long l = left - at;
        load8(q + at, l > 8 ? 8 : (long)l, at + base ? 8 : 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc += (double)v[i] * (double)v[i];
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}
__global__ __launch_bounds__(1024) void grad_norm_final_kernel(const double* const partial, const int n, float* const out) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) acc += partial[i];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
  __shared__ double red[16];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < 16; ++i) s += red[i];
    *out = (float)sqrt(s);
  }
}

// the tensors [i, i + AW_MAX) that have values and a gradient, as a table; returns how many workgroups they take
struct AwFill {
  size_t block = 0;         // state blocks in front of tensor i (tensors without a gradient keep theirs)
  int i = 0;
  unsigned long long next(const selfc_adamw_tensor* const ts, const int count, AwTable& tab, bool& ok) {
    unsigned long long wgs = 0;
    tab.count = 0;
    tab.place0 = i;
    int left = AW_MAX;
    for (; i < count && left > 0; ++i, --left) {
      // an entry per tensor, so that its number in the table gives its place in the list; an empty one takes no workgroup
      const selfc_adamw_tensor& t = ts[i];
      const size_t blocks = (t.n + AW_BLOCK - 1) / AW_BLOCK;
      const unsigned long long need = t.grad && t.n ? (t.n + AW_CHUNK - 1) / AW_CHUNK : 0;
      if (block > 0xffffffffull || wgs + need > 0x7fffffffull) { ok = false; return 0; }
      tab.e[tab.count++] = AwEntry{t.param, t.grad, t.step, t.n, (unsigned)block, (unsigned)wgs};
      wgs += need;
      block += blocks;
    }
    return wgs;
  }
};

}  // namespace
}  // namespace selfc

using namespace selfc;

extern "C" {

int selfc_adamw_block(void) { return AW_BLOCK; }

int selfc_adamw_step(const selfc_adamw_tensor* tensors, int count, int dtype, int state_bits, void* m, void* v, float* m_scale,
                     float* v_scale, float lr, const float* lr_dev, double beta1, double beta2, float eps, float weight_decay,
                     double step, unsigned seed, const float* norm, float max_norm, void* stream) {
  if (!tensors || count < 0 || (state_bits != 32 && state_bits != 8) || dtype < 0 || dtype > 2) return SELFC_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return SELFC_EINVAL;
  bool any = false, host_step = false;
  for (int i = 0; i < count; ++i) {
    if (!tensors[i].grad || !tensors[i].n) continue;
    any = true;
    if (!tensors[i].param || !aligned_to(tensors[i].param, dtype ? 2 : 4) || !aligned_to(tensors[i].grad, dtype ? 2 : 4)) return SELFC_EINVAL;
    host_step |= tensors[i].step == nullptr;
  }
  if (!any) return SELFC_OK;
  if (host_step && !(step >= 1.0)) return SELFC_EINVAL;
  if (!m || !v || !aligned_to(m, 16) || !aligned_to(v, 16) || (state_bits == 8 && (!m_scale || !v_scale))) return SELFC_EINVAL;
  AwHyper hy{};
  hy.lr_dev = lr_dev; hy.norm = norm; hy.beta1_d = beta1; hy.beta2_d = beta2; hy.lr = lr;
  hy.bc1 = (float)(1.0 - pow(beta1, step)); hy.bc2s = (float)sqrt(1.0 - pow(beta2, step));
  hy.b1 = (float)beta1; hy.omb1 = (float)(1.0 - beta1); hy.b2 = (float)beta2; hy.omb2 = (float)(1.0 - beta2);
  hy.eps = eps; hy.wd = weight_decay; hy.max_norm = max_norm; hy.seed = seed;
  hy.key = aw_mix(seed ^ aw_mix((unsigned)(unsigned long long)(step > 0.0 ? step : 0.0)));
  AwFill fill;
  AwTable tab;
  hipStream_t s = (hipStream_t)stream;
  bool ok = true;
  { AwFill dry; while (dry.i < count && ok) dry.next(tensors, count, tab, ok); }      // refuse before anything is launched
  if (!ok) return SELFC_EINVAL;
  while (fill.i < count) {
    const unsigned long long wgs = fill.next(tensors, count, tab, ok);
    if (!wgs) continue;
    const dim3 grid((unsigned)wgs), blk(256);
    if (state_bits == 32) {
      if (dtype == 0) hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
      else if (dtype == 1) hipLaunchKernelGGL((adamw_kernel<b16, 32>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
      else hipLaunchKernelGGL((adamw_kernel<h16, 32>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
    } else {
      if (dtype == 0) hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
      else if (dtype == 1) hipLaunchKernelGGL((adamw_kernel<b16, 8>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
      else hipLaunchKernelGGL((adamw_kernel<h16, 8>), grid, blk, 0, s, tab, hy, m, v, m_scale, v_scale);
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return pw_rc(e);
  }
  return SELFC_OK;
}

size_t selfc_grad_norm_partials(int count) { return count < 1 ? 1 : (size_t)((count + AW_MAX - 1) / AW_MAX) * GN_WG; }

int selfc_grad_norm(const selfc_adamw_tensor* tensors, int count, int dtype, double* partial, float* out, void* stream) {
  if (!tensors || count < 0 || !partial || !out || dtype < 0 || dtype > 2) return SELFC_EINVAL;
  for (int i = 0; i < count; ++i)
    if (tensors[i].grad && !aligned_to(tensors[i].grad, dtype ? 2 : 4)) return SELFC_EINVAL;
  AwTable tab;
  bool ok = true;
  { AwFill dry; while (dry.i < count && ok) dry.next(tensors, count, tab, ok); }
  if (!ok) return SELFC_EINVAL;
  AwFill fill;
  hipStream_t s = (hipStream_t)stream;
  int used = 0;
  while (fill.i < count) {
    const unsigned long long chunks = fill.next(tensors, count, tab, ok);
    if (!chunks) continue;
    const int wgs = chunks < GN_WG ? (int)chunks : GN_WG;
    const dim3 grid((unsigned)wgs), blk(256);
    if (dtype == 0) hipLaunchKernelGGL((grad_norm_kernel<float>), grid, blk, 0, s, tab, (unsigned)chunks, partial + used);
    else if (dtype == 1) hipLaunchKernelGGL((grad_norm_kernel<b16>), grid, blk, 0, s, tab, (unsigned)chunks, partial + used);
    else hipLaunchKernelGGL((grad_norm_kernel<h16>), grid, blk, 0, s, tab, (unsigned)chunks, partial + used);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return pw_rc(e);
    used += wgs;
  }
  hipLaunchKernelGGL(grad_norm_final_kernel, dim3(1), dim3(1024), 0, s, partial, used, out);
  return pw_rc(hipGetLastError());
}

}  // extern "C"
