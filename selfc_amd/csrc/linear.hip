// Matrix products of rows with a weight, with everything that follows the product in the same launch:
//   y[m][n] = act( sx[m] sw[n] sum_k x[m][k] W[n][k] + b[n] ) + r[m][n]                       (sx, sw: 8-bit operands only)
// for 16-bit operands with the gradients
//   dz = dy act'(z),   dx = dz W,   dW = dz^T x,   db = sum over rows of dz
// and for e4m3 operands (one scale per row of x and of W) without.  Sums in fp32 on the matrix units.
//
// One kernel computes out[q][p] = sum over r of Q(q, r) P(p, r); an operand is either stored with r contiguous ("straight": x and W
// of the forward product) or with r as its row index ("crossed": W in dx, both in dW), and the latter is transposed on the way
// from shared memory to registers (ds_read_b64_tr_b16), never in memory.
//
// The derivative act'(z) is kept for the backward pass: of ReLU and LeakyReLU one bit per value (z > 0), of the others a 16-bit
// fixed-point number (steps of 2^-15 from -0.5; 65535: not a number): their derivatives lie in [-0.13, 1.13], 0 and 1 are exact, and the
// error is 2^-16 everywhere - after it the backward pass needs neither z nor the activation's formula.  Keeping z in bf16 instead would cost up
// to 85 times that (GELU, near |z| = 0.7; in f16 11 times), but less where the activation is all but flat: from |z| = 4.2 on (f16: 3.5; SiLU 9.9 and
// 7.0).  There the fixed step shows as a relative error: GELU's slope -5.0e-4 at z = -4 is kept to 3 %, the -7e-6 at -5 as 0; SiLU's
// -4.1e-4 at -10 to 4 %, the -1.1e-5 at -14 as 0.
// (Bits against codes - LeakyReLU against GELU, launches replayed from a graph: a layer of 200,704 x 128 x 128 in f16 with its gradients 108 us, 131; of
// 72,576 x 204 x 51 60, 79.)
//
// Four forms, chosen by the rules beside gemm_plan, gemv_takes and rows_plan below (and, between the last two, by the caller): tiles that meet in
// shared memory (bound by the matrix units), the weight straight into registers for few rows (bound by the weight's bytes), the whole weight
// in shared memory for narrow layers (bound by the rows' bytes).  Measured, bf16: 8192 x 8192 x 8192 788 us (1,395 TFLOP/s; a library's plain product
// 666), its two crossed forms 800 and 810 (library 785 and 905); e4m3 395 us (2,780 TFLOP/s).  What follows the product shows where a unit has one tile
// after the other: 8192 x 8192 x 2048 232 us plain, 256 with GELU, 284 with its derivative's 134 MB too.  In the large tiles the matrix units are busy for 60 % of
// the cycles and the clock has fallen to 2.0 GHz; no shared-memory conflicts; the waves wait at the stages' barriers for 28 % of the time.  With four
// waves of 128 x 128 instead of eight of 64 x 128 (a third less shared-memory traffic, one wave per SIMD) 1,062 us.
#include "pointwise.hpp"
#include <math.h>

namespace selfc {

int pw_colsum(const float* partial, int rows, int C, int dtype, void* out, hipStream_t s);      // rmsnorm.hip

namespace {

enum { ACT_NONE, ACT_RELU, ACT_LRELU, ACT_GELU, ACT_SILU };
constexpr float LRELU = 0.2f;
__host__ __device__ inline bool act_bits(const int act) { return act == ACT_RELU || act == ACT_LRELU; }

typedef h16 h16x8 __attribute__((ext_vector_type(8)));
typedef b16 b16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

// ---- what follows the product ---------------------------------------------------------------------------------------------
struct Epilogue {
  void* out;                      // [M][ldo] of `dtype`
  const void *bias, *res;         // [N]; [M][ldr]
  const float *qs, *ps;           // scales of the rows and of the columns
  unsigned char* d;               // [M][ldd bytes] derivative: bits, eight neighbouring columns to a byte, or 16-bit codes
  size_t ldo, ldr, ldd;
  int dtype, act;
};

// N values z -> activation y and, with D, its derivative d.  GELU: z phi(z) with phi = 1 - erfc(|z| / sqrt 2) / 2 mirrored at 0, erfc by
// the polynomial of Abramowitz and Stegun 7.1.26 (absolute error 1.5e-7) times the exponential that the derivative needs too.
template <int N, bool D>
__device__ __forceinline__ void act_apply(const int act, const float* const z, float* const y, float* const d) {
  if (act == ACT_NONE) {
#pragma unroll
    for (int i = 0; i < N; ++i) { y[i] = z[i]; if (D) d[i] = 1.f; }
  } else if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) { y[i] = z[i] <= 0.f ? 0.f : z[i]; if (D) d[i] = z[i] > 0.f ? 1.f : 0.f; }        // a NaN stays one
  } else if (act == ACT_LRELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) { const float s = z[i] > 0.f ? 1.f : LRELU; y[i] = z[i] * s; if (D) d[i] = s; }
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float az = __builtin_amdgcn_fmed3f(fabsf(z[i]), 0.f, 20.f);             // infinities: the exponential is 0 from there on
      const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, az, 1.f));
      const float e = __builtin_amdgcn_exp2f(az * az * -0.72134752f);               // exp(-z^2 / 2)
      float q = fmaf(1.061405429f, t, -1.453152027f);
      q = fmaf(q, t, 1.421413741f);
      q = fmaf(q, t, -0.284496736f);
      q = fmaf(q, t, 0.254829592f);
      const float tail = 0.5f * q * t * e;                                          // of the normal distribution, beyond |z|
      const float phi = z[i] > 0.f ? 1.f - tail : tail;
      y[i] = z[i] < -20.f ? 0.f : z[i] * phi;                                       // (a NaN in z comes through z)
      if (D) d[i] = fmaf(z[i] < 0.f ? -az : az, e * 0.39894228f, phi);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[i] * -1.44269504f));
      y[i] = z[i] < -100.f ? 0.f : z[i] * s;
      const float zc = __builtin_amdgcn_fmed3f(z[i], -100.f, 100.f);
      if (D) d[i] = s * fmaf(zc, 1.f - s, 1.f);
    }
  }
}
// derivative -> 16-bit fixed point, rounded to nearest: (d + 0.5) 2^15 is in [0, 65534] for every activation here
__device__ __forceinline__ unsigned act_code(const float d, const float z) {
  const unsigned c = (unsigned)fmaf(d, 32768.f, 16384.5f);
  return z != z ? 65535u : c;
}
__device__ __forceinline__ float act_slope(const unsigned c) {
  return c == 65535u ? __builtin_nanf("") : (float)((int)c - 16384) * 0x1p-15f;
}

// dy times the derivative that a bit stands for; under a 0 of ReLU nothing comes through, whatever dy is
__device__ __forceinline__ float bit_slope(const float dy, const unsigned bits, const int i, const float low) {
  return bits >> i & 1 ? dy : low == 0.f ? 0.f : dy * low;
}

__device__ __forceinline__ void load8_as(const int dtype, const void* const p, const size_t at, const int left, const int before, float* const v) {
  if (dtype == 0) load8((const float*)p + at, left, before, v);
  else if (dtype == 1) load8((const b16*)p + at, left, before, v);
  else load8((const h16*)p + at, left, before, v);
}

// eight neighbouring columns of one row: acc is the product's sum, b and ps the columns' bias and scale
__device__ __forceinline__ void epilogue8(const Epilogue& e, const float* const acc, const int row, const int col, const int left,
                                          const float* const b, const float* const ps) {
  float z[8], y[8], d[8], r[8];
  const float qs = e.qs ? e.qs[row] : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = (e.qs ? acc[i] * (qs * ps[i]) : acc[i]) + b[i];
  if (e.d && !act_bits(e.act)) {
    act_apply<8, true>(e.act, z, y, d);
    u16x8 c;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (unsigned short)act_code(d[i], z[i]);
    *reinterpret_cast<u16x8*>(e.d + (size_t)row * e.ldd + col * 2) = c;      // a row holds a multiple of 8: always 16 bytes at a time
  } else {
    act_apply<8, false>(e.act, z, y, d);
    if (e.d) {
      unsigned c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) c |= (z[i] > 0.f ? 1u : 0u) << i;
      e.d[(size_t)row * e.ldd + col / 8] = (unsigned char)c;
    }
  }
  if (e.res) {
    load8_as(e.dtype, e.res, (size_t)row * e.ldr + col, left, col, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] += r[i];
  }
  const size_t at = (size_t)row * e.ldo + col;
  if (e.dtype == 0) store8((float*)e.out + at, left, y);
  else if (e.dtype == 1) store8((b16*)e.out + at, left, y);
  else store8((h16*)e.out + at, left, y);
}
// the same where nothing follows the product
template <typename T>
__device__ __forceinline__ void plain8(const Epilogue& e, const float* const acc, const int row, const int col, const int left) {
  store8((T*)e.out + (size_t)row * e.ldo + col, left, acc);
}
__device__ __forceinline__ void epilogue_columns(const Epilogue& e, const int col, const int left, float* const b, float* const ps) {
#pragma unroll
  for (int i = 0; i < 8; ++i) { b[i] = 0.f; ps[i] = 1.f; }
  if (e.bias) load8_as(e.dtype, e.bias, col, left, col, b);
  if (e.ps) load8(e.ps + col, left, col, ps);
}

// ---- the product ----------------------------------------------------------------------------------------------------------
struct GemmArgs {
  const void *q, *p;
  size_t ldq, ldp;                // pitches in elements
  int M, N, R;                    // rows and columns of the output, length of the sum (R: a multiple of 16 bytes where an operand is straight)
  int qx, px;                     // crossed operands: readable columns (a multiple of 8)
  int splits, per;                // parts of the sum, and stages of each
  float* ws;                      // [splits][M][ldw] partial sums when splits > 1, and behind them [splits][M] of the rows' own sums
  size_t ldw;
  void* sums;                     // dW: NULL, or [M]: the sum of each row of Q (db), of the output's type
  Epilogue e;
};

// global -> shared memory without registers: lane i's 16 bytes land at lds + 16 i; an offset beyond the resource reads zeros
__device__ __forceinline__ void dma16(const i32x4 rsrc, const unsigned voff, const unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds) : "memory");
}
template <int VM>
__device__ __forceinline__ void wait_barrier() {            // loads but the last VM done, own LDS reads done; then everybody's
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

template <typename T> struct Mma;
template <> struct Mma<h16> {
  static __device__ __forceinline__ f32x4 run(const i32x4 a, const i32x4 b, const f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma<b16> {
  static __device__ __forceinline__ f32x4 run(const i32x4 a, const i32x4 b, const f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
};
// e4m3 x e4m3: 32 values per lane; both operands hand over the same two 16-byte pieces, so whichever k they belong to, it is the same
// e4m3: the form whose rate is twice 16 bits'.  The unit adds eight neighbouring products aligned to the largest of them and cuts the others below
// 2^-13 of its power of two; the eights are then added in 24 bits.  So a sum is off by less than 7 x 2^-13 of each eight's largest product
// (normal random rows: 2e-6 of the sum of the magnitudes on average, 6e-5 at most of 2 M sums): next to the 2^-4 that each value was rounded by to fit
// into e4m3, full 32-bit sums at half the rate would buy nothing.
__device__ __forceinline__ f32x4 mma8(const i32x4 a0, const i32x4 a1, const i32x4 b0, const i32x4 b1, const f32x4 c) {
  const i32x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

// One operand's side of a stage: B rows (straight: [B][128 bytes]) or B columns (crossed: [64][B] 16-bit values) in shared memory.
// 16-byte pieces are stored at a permuted place of their row so that the reads below never meet in a bank: the loads write shared
// memory in lane order, so the permutation is applied to the global address.
template <int B, bool X, int ES, int NT>
struct Side {
  static constexpr int LOADS = B * 8 / NT;                  // 16-byte pieces per thread and stage
  static constexpr int RB = X ? B * 2 : 128;                // bytes of a row in shared memory
  unsigned voff[LOADS];                                     // byte offset of each piece from the stage's base, or out of range
  int kk[LOADS];                                            // its place along the sum
  const char* base;                                         // the stage's base
  const char* end;
  size_t step;                                              // bytes from one stage to the next

  static __device__ __forceinline__ int swz(const int r) {  // crossed: which pair of pieces row r moves its columns by
    return B >= 128 ? (r & 3) | ((r >> 3) & 1) << 2 : ((r >> 1) & 1) | ((r >> 3) & 1) << 1;
  }
  __device__ __forceinline__ void init(const void* const src, const size_t ld, const int i0, const int extent, const int R, const int stage0) {
    constexpr int PIECE = 16 / ES;
    const char* const s = (const char*)src;
    if (X) {
      step = 64 * ld * ES;
      base = s + (size_t)i0 * ES + (size_t)stage0 * step;
      end = s + ((size_t)(R - 1) * ld + extent) * ES;
    } else {
      step = 128;
      base = s + (size_t)i0 * ld * ES + (size_t)stage0 * 128;
      end = s + (size_t)(extent - 1) * ld * ES + (((size_t)R * ES + 15) & ~(size_t)15);
    }
    const int tid = threadIdx.x;
#pragma unroll
    for (int it = 0; it < LOADS; ++it) {
      const int l = it * NT + tid;
      if (X) {
        const int r = l / (B / 8), c = (l % (B / 8)) ^ (swz(r) << 1);
        kk[it] = r;
        voff[it] = i0 + c * 8 < extent ? (unsigned)(r * ld * ES + c * 16) : BUF_OOB;
      } else {
        const int r = l >> 3, c = (l & 7) ^ ((r >> 1) & 7);
        kk[it] = c * PIECE;
        voff[it] = i0 + r < extent ? (unsigned)(r * ld * ES + c * 16) : BUF_OOB;
      }
    }
  }
  // request a stage of which `left` places of the sum remain (none: zeros), piece by piece, and move on to the next
  i32x4 rsrc;
  unsigned at;
  int room;
  __device__ __forceinline__ void begin(const unsigned lds, const int left) {
    const size_t bytes = left > 0 ? (size_t)(end - base) : 0;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)(size_t)base), hi = __builtin_amdgcn_readfirstlane((unsigned)((size_t)base >> 32));
    rsrc = i32x4{(int)lo, (int)(hi & 0xffffu), (int)__builtin_amdgcn_readfirstlane(bytes < 0x7fffffffu ? (unsigned)bytes : 0x7fffffffu), 0x00020000};
    at = lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
    room = left;
    base += step;
  }
  __device__ __forceinline__ void issue(const int it) const { dma16(rsrc, kk[it] < room ? voff[it] : BUF_OOB, at + it * (NT * 16)); }
};

// fragments of a 16-wide tile: 16 x 32 16-bit values (straight or crossed) or 16 x 64 bytes of 8-bit ones
template <int B, bool X>
struct Frag {
  int a0, a1;            // this lane's addresses in a stage
  __device__ __forceinline__ void init(const int i0) {        // i0: the wave's first row / column (a multiple of 16)
    const int lane = threadIdx.x & 63, g = lane >> 4;
    if (X) {
      const int q = (lane >> 2) & 3, p = lane & 3;
      const int r = g * 8 + q;
      a0 = r * (B * 2) + ((Side<B, X, 2, 256>::swz(r) << 5) ^ (i0 << 1)) + p * 8;
      a1 = 0;
    } else {
      const int row = i0 + (lane & 15), sw = (lane >> 1) & 7;
      a0 = row * 128 + ((g ^ sw) << 4);
      a1 = row * 128 + (((g ^ sw) ^ 4) << 4);
    }
  }
  // tile t of the wave, half ks of the stage
  __device__ __forceinline__ i32x4 read(const unsigned char* const side, const int t, const int ks) const {
    if constexpr (X) {
      typedef short s16x4 __attribute__((__vector_size__(8)));
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const unsigned char* const at = side + (a0 ^ (t << 5)) + ks * 32 * (B * 2);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * (B * 2)));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(i32x4, v);
    } else {
      return *reinterpret_cast<const i32x4*>(side + (ks ? a1 : a0) + t * 2048);
    }
  }
};

// BQ x BP outputs per workgroup of NQ x NP waves.  T: h16, b16, or unsigned char for e4m3.
// The stages of the sum (64 values of 16 bits, 128 of 8) go through two shared-memory buffers: while one is multiplied, the loads of
// the next are on their way to the other; one barrier per stage.
template <typename T, bool QX, bool PX, int BQ, int BP, int NQ, int NP>
__global__ __launch_bounds__(NQ * NP * 64) void gemm_kernel(const GemmArgs a) {
  constexpr int NT = NQ * NP * 64, ES = sizeof(T), BK = 128 / ES;
  constexpr int SQ = BQ * 128, STAGE = (BQ + BP) * 128;
  constexpr int WQ = BQ / NQ, WP = BP / NP, TQ = WQ / 16, TP = WP / 16;
  extern __shared__ __align__(16) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)lds;

  // workgroup -> (part of the sum, tile): consecutive tiles on one XCD; tiles in bands of 8 rows, so that neighbours share operands
  const int nq = (a.M + BQ - 1) / BQ, np = (a.N + BP - 1) / BP, tiles = nq * np;
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int part = id / tiles;
  id -= part * tiles;
  const int band = id / (8 * np), in = id - band * 8 * np, rows = nq - band * 8 < 8 ? nq - band * 8 : 8;
  const int q0 = (band * 8 + in % rows) * BQ, p0 = (in / rows) * BP;
  const int stages = (a.R + BK - 1) / BK;
  const int s0 = part * a.per, s1 = s0 + a.per < stages ? s0 + a.per : stages;

  Side<BQ, QX, ES, NT> sq;
  Side<BP, PX, ES, NT> sp;
  sq.init(a.q, a.ldq, q0, QX ? a.qx : a.M, a.R, s0);
  sp.init(a.p, a.ldp, p0, PX ? a.px : a.N, a.R, s0);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wq = wave / NP, wp = wave % NP;
  Frag<BQ, QX> fq;
  Frag<BP, PX> fp;
  fq.init(wq * WQ);
  fp.init(wp * WP);

  f32x4 acc[TP][TQ];
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // db: the rows' own sums are one more column of the product, against a fragment of ones.  They are sums of dz as it is multiplied, rounded to
  // T once; without dW there is no such product, and dz_kernel adds dz before it is rounded (one rounding of 2^-9 or 2^-12 a term less)
  const bool own = QX && PX && a.sums && p0 == 0 && wp == 0;
  f32x4 osum[QX && PX ? TQ : 1];
  i32x4 ones;
  if constexpr (QX && PX) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (T)1.f;
    ones = __builtin_bit_cast(i32x4, o);
#pragma unroll
    for (int j = 0; j < TQ; ++j) osum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // TQ multiplies per step and piece of P; the pieces are requested AHEAD steps before their multiplies, and the schedule is held to
  // that (left alone, the compiler moves every read to right in front of its use and the matrix units wait for shared memory).
  // A large tile has a compute unit to itself, so nothing hides what it waits for between two stages.  Its barrier stands AHEAD steps
  // before a stage's end, where its last read is out: behind it the next stage's first pieces are read, and the loads of the stage after
  // that set out over the last steps (8192 x 8192 x 8192 bf16: 828 us with the barrier between the stages, 788 this way).  Small tiles
  // share a compute unit and fill each other's gaps: barrier between the stages, the next one's loads at once behind it, so that they have
  // all of a stage to arrive (4096 x 2048 x 8192: 118 us, 142 to 155 with the early barrier).
  constexpr bool EARLY = BQ * BP >= 256 * 256;
  constexpr int HALF = ES == 1 ? 1 : 2, STEPS = HALF * TP, AHEAD = STEPS < 4 ? STEPS - 1 : 3, W = ES == 1 ? 2 : 1;
  constexpr int TURN = EARLY ? STEPS - AHEAD : STEPS, RING = AHEAD + 1;
  constexpr int RP = (PX ? 2 : 1) * W, RQ = (QX ? 2 : 1) * W;           // reads per piece
  static_assert(STEPS % RING == 0, "a piece keeps its place in the ring from stage to stage");
  constexpr int ALL = decltype(sq)::LOADS + decltype(sp)::LOADS;
  i32x4 q[HALF][TQ][W], p[RING][W];
  const auto read_q = [&](const int buf, const int h) {
#pragma unroll
    for (int j = 0; j < TQ; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) q[h][j][w] = fq.read(lds + buf * STAGE, j, ES == 1 ? w : h);
  };
  const auto read_p = [&](const int buf, const int n) {
#pragma unroll
    for (int w = 0; w < W; ++w) p[n % RING][w] = fp.read(lds + buf * STAGE + SQ, n % TP, ES == 1 ? w : n / TP);
  };
  const auto read_first = [&](const int buf) {
    read_q(buf, 0);
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) read_p(buf, n);
    __builtin_amdgcn_sched_group_barrier(0x100, TQ * RQ + AHEAD * RP, 0);
  };
  const auto begin = [&](const int buf, const int s) {                  // behind the last stage: nothing is read, zeros are written
    const int left = s < s1 ? a.R - s * BK : 0;
    sq.begin(lds0 + buf * STAGE, left);
    sp.begin(lds0 + buf * STAGE + SQ, left);
  };
  const auto issue = [&](const int k) {
    if (k < sq.LOADS) sq.issue(k);
    else sp.issue(k - sq.LOADS);
  };
  const auto load = [&](const int buf, const int s) {
    begin(buf, s);
#pragma unroll
    for (int k = 0; k < ALL; ++k) issue(k);
  };
  if (s0 < s1) load(0, s0);
  if constexpr (EARLY) {                  // both buffers are there whatever the number of stages
    wait_barrier<0>();
    load(1, s0 + 1);
    read_first(0);
  }

  for (int s = s0; s < s1; ++s) {
    const int cur = (s - s0) & 1;
    if constexpr (!EARLY) {
      wait_barrier<0>();
      if (s + 1 < s1) load(cur ^ 1, s + 1);
      read_first(cur);
    }
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      const int h = n / TP, i = n % TP, slot = n % RING;
      const bool half = HALF == 2 && n == (TP > 2 ? TP - 2 : 0), next = EARLY && n == (HALF == 2 ? STEPS - 2 : STEPS - 1);
      if (n == TURN) {
        wait_barrier<0>();
        begin(cur, s + 2);
      }
      if (n + AHEAD < STEPS) read_p(cur, n + AHEAD);
      else if (EARLY) read_p(cur ^ 1, n + AHEAD - STEPS);
      if (half) read_q(cur, 1);
      if (next && HALF == 2) read_q(cur ^ 1, 0);
#pragma unroll
      for (int j = 0; j < TQ; ++j) {
        if constexpr (ES == 1) acc[i][j] = mma8(p[slot][0], p[slot][W - 1], q[h][j][0], q[h][j][W - 1], acc[i][j]);
        else acc[i][j] = Mma<T>::run(p[slot][0], q[h][j][0], acc[i][j]);
      }
      if (next && HALF == 1) read_q(cur ^ 1, 0);
      if (EARLY || n + AHEAD < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, RP, 0);
      if (half || (next && HALF == 2)) __builtin_amdgcn_sched_group_barrier(0x100, TQ * RQ, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, TQ, 0);
      if (next && HALF == 1) __builtin_amdgcn_sched_group_barrier(0x100, TQ * RQ, 0);
      if (n >= TURN) {
        constexpr int EACH = (ALL + AHEAD - 1) / AHEAD;
#pragma unroll
        for (int k = (n - TURN) * EACH; k < (n - TURN + 1) * EACH && k < ALL; ++k) issue(k);
      }
      if constexpr (QX && PX) {
        if (own && EARLY && i == (h == 0 ? 0 : TP - 1))
#pragma unroll
          for (int j = 0; j < TQ; ++j) osum[j] = Mma<T>::run(ones, q[h][j][0], osum[j]);
      }
    }
    if constexpr (QX && PX && !EARLY) {
      if (own)
#pragma unroll
        for (int h = 0; h < HALF; ++h)
#pragma unroll
          for (int j = 0; j < TQ; ++j) osum[j] = Mma<T>::run(ones, q[h][j][0], osum[j]);
    }
  }
  wait_barrier<0>();                      // the buffers are free: each wave turns its tiles into rows of its own piece of them
  if constexpr (QX && PX) {
    if (own && (threadIdx.x & 63) < 16) {
#pragma unroll
      for (int j = 0; j < TQ; ++j) {
        const int row = q0 + wq * WQ + j * 16 + (threadIdx.x & 15);
        if (row < a.M) {
          if (a.splits == 1) ((T*)a.sums)[row] = (T)osum[j][0];
          else a.ws[(size_t)a.splits * a.M * a.ldw + (size_t)part * a.M + row] = osum[j][0];
        }
      }
    }
  }

  constexpr int PITCH = WP + 4, LPR = WP / 8, RPP = 64 / LPR;         // floats per row, lanes per row, rows per pass
  const int lane = threadIdx.x & 63;
  float* const turn = reinterpret_cast<float*>(lds) + wave * 16 * PITCH;
  const int col = p0 + wp * WP + (lane % LPR) * 8, left = a.N - col;
  constexpr bool FULL = !QX && !PX;       // the products of the backward pass are stored as they are
  float b[8], ps[8];
  if (FULL && a.splits == 1) epilogue_columns(a.e, col, left, b, ps);
#pragma unroll
  for (int j = 0; j < TQ; ++j) {
#pragma unroll
    for (int i = 0; i < TP; ++i)
      *reinterpret_cast<f32x4*>(turn + (lane & 15) * PITCH + i * 16 + (lane >> 4) * 4) = acc[i][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int k = 0; k < 16 / RPP; ++k) {
      const int r = k * RPP + lane / LPR, row = q0 + wq * WQ + j * 16 + r;
      const f32x4 v0 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + (lane % LPR) * 8);
      const f32x4 v1 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + (lane % LPR) * 8 + 4);
      if (row < a.M && left > 0) {
        const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        if (a.splits == 1) {
          if constexpr (FULL) epilogue8(a.e, v, row, col, left, b, ps);
          else plain8<T>(a.e, v, row, col, left);
        } else {
          float* const w = a.ws + ((size_t)part * a.M + row) * a.ldw + col;      // ldw is a multiple of 8
          *reinterpret_cast<f32x4*>(w) = v0;
          *reinterpret_cast<f32x4*>(w + 4) = v1;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// the parts of a divided sum, added in a fixed order, and what follows the product.  Eight neighbouring columns are one item; SL threads
// share an item's parts (few items and many parts: one thread each would be a handful of workgroups on long chains of loads)
template <int SL>
__global__ __launch_bounds__(256) void gemm_join_kernel(const GemmArgs a) {
  constexpr int ITEMS = 256 / SL;
  __shared__ float red[SL][ITEMS][9];
  const int per_row = (a.N + 7) / 8, item = threadIdx.x % ITEMS, slice = threadIdx.x / ITEMS;
  const size_t id = (size_t)blockIdx.x * ITEMS + item;
  const bool in = id < (size_t)a.M * per_row;
  const int row = in ? (int)(id / per_row) : 0, col = in ? (int)(id % per_row) * 8 : 0;
  float v[9] = {};                   // [8]: the row's own sum
  const bool own = in && a.sums && col == 0;
  if (in) {
    const size_t part = (size_t)a.M * a.ldw;
    const float* const w = a.ws + (size_t)row * a.ldw + col;
#pragma unroll 4
    for (int s = slice; s < a.splits; s += SL) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(w + s * part), y = *reinterpret_cast<const f32x4*>(w + s * part + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] += x[i]; v[4 + i] += y[i]; }
    }
    if (own)
      for (int s = slice; s < a.splits; s += SL) v[8] += a.ws[a.splits * part + (size_t)s * a.M + row];
  }
  if constexpr (SL > 1) {
#pragma unroll
    for (int i = 0; i < 9; ++i) red[slice][item][i] = v[i];
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int k = 1; k < SL; ++k)
#pragma unroll
      for (int i = 0; i < 9; ++i) v[i] += red[k][item][i];
  }
  if (!in) return;
  if (own) {
    if (a.e.dtype == 1) ((b16*)a.sums)[row] = (b16)v[8];
    else ((h16*)a.sums)[row] = (h16)v[8];
  }
  float b[8], ps[8];
  epilogue_columns(a.e, col, a.N - col, b, ps);
  epilogue8(a.e, v, row, col, a.N - col, b, ps);
}

// ---- up to 16 rows: the weight is read once, straight into registers ------------------------------------------------------
// A workgroup owns 16 columns of the output (16 rows of W); its eight waves take turns along the sum, two 64-byte pieces of each
// weight row at a time, and meet in shared memory.  1 x 4096 x 4096 bf16: 9.5 us with its launch from memory (33.6 MB: 3.5 TB/s), 7.3 where
// the last cache holds the weight; 16 rows 12.2 and 10.0; e4m3 8.1 and 7.3.
// Rows that are not whole 16-byte pieces at aligned places are read as they lie (laying the weight out first would move its bytes three times): every piece is a 16-byte access at any address, the last one of a row moved back to the row's end and shifted down.
// 16 bytes at `at` of a row of `bytes` >= 16; zeros behind its end
__device__ __forceinline__ i32x4 row16(const char* const row, const unsigned at, const unsigned bytes) {
  const unsigned from = at < bytes - 16 ? at : bytes - 16, down = (at - from) * 8;
  unsigned long long v[2];
  __builtin_memcpy(v, row + from, 16);
  unsigned long long lo = v[0], hi = v[1];
  if (down) {
    lo = down < 64 ? v[0] >> down | v[1] << (64 - down) : down < 128 ? v[1] >> (down - 64) : 0;
    hi = down < 64 ? v[1] >> down : 0;
  }
  return i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}
template <typename T, bool WHOLE>
__global__ __launch_bounds__(512) void gemv_kernel(const GemmArgs a) {
  constexpr int ES = sizeof(T), PIECE = 16 / ES, NW = 8, U = 8;       // U stages of a wave, 16 KiB, on their way at a time
  __shared__ float red[NW][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
  const int p0 = blockIdx.x * 16;
  const size_t wbytes = ((size_t)((a.N - p0 < 16 ? a.N - p0 : 16) - 1) * a.ldp + a.R) * ES, xbytes = ((size_t)(a.M - 1) * a.ldq + a.R) * ES;
  const buf_rsrc rw = make_rsrc((const char*)a.p + (size_t)p0 * a.ldp * ES, (unsigned)wbytes);
  const buf_rsrc rx = make_rsrc(a.q, (unsigned)xbytes);
  const unsigned wrow = p0 + i < a.N ? (unsigned)(i * a.ldp * ES) : BUF_OOB, xrow = i < a.M ? (unsigned)(i * a.ldq * ES) : BUF_OOB;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const char* const wr = (const char*)a.p + ((size_t)p0 + (p0 + i < a.N ? i : 0)) * a.ldp * ES;       // rows that are not there: any, nothing is made of them
  const char* const xr = (const char*)a.q + (size_t)(i < a.M ? i : 0) * a.ldq * ES;
  const int stages = (a.R + 8 * PIECE - 1) / (8 * PIECE);          // 128 bytes of a row per stage
  for (int s = wave; s < stages; s += NW * U) {
    i32x4 w[U][2], x[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int piece = (s + u * NW) * 8 + h * 4 + g;
        const bool in = piece * PIECE < a.R;
        const unsigned off = (unsigned)piece * 16;
        if constexpr (!WHOLE) {
          if (s + u * NW >= stages) {
            w[u][h] = x[u][h] = i32x4{0, 0, 0, 0};
            continue;
          }
          w[u][h] = row16(wr, off, (unsigned)a.R * ES);
          x[u][h] = row16(xr, off, (unsigned)a.R * ES);
          continue;
        }
        w[u][h] = __builtin_bit_cast(i32x4, buffer_load_b128(rw, in && wrow != BUF_OOB ? wrow + off : BUF_OOB, 0));
        x[u][h] = __builtin_bit_cast(i32x4, buffer_load_b128(rx, in && xrow != BUF_OOB ? xrow + off : BUF_OOB, 0));
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (ES == 1) {
        acc = mma8(w[u][0], w[u][1], x[u][0], x[u][1], acc);
      } else {
        acc = Mma<T>::run(w[u][0], x[u][0], acc);
        acc = Mma<T>::run(w[u][1], x[u][1], acc);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[wave][i][g * 4 + k] = acc[k];          // [row of x][column]
  __syncthreads();
  if (threadIdx.x < 32) {
    const int row = threadIdx.x >> 1, c = (threadIdx.x & 1) * 8, col = p0 + c;
    if (row < a.M && col < a.N) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float t = 0.f;
#pragma unroll
        for (int wv = 0; wv < NW; ++wv) t += red[wv][row][c + k];
        v[k] = t;
      }
      float b[8], ps[8];
      epilogue_columns(a.e, col, a.N - col, b, ps);
      epilogue8(a.e, v, row, col, a.N - col, b, ps);
    }
  }
}

// ---- narrow rows: up to 256 values in and out ----------------------------------------------------------------------------------
// Pixels' channels: a product of few columns is bound by the rows' traffic, and tiles that meet in shared memory only delay it.  Here the
// whole weight stays in shared memory, a wave takes 16 rows at a time straight from memory into the multiply's operand and back, and
// what used to be launches of their own rides along (f16, 200,704 x 64 x 64: 13.1 us, 52 MB, 3.9 TB/s; in tiles 21.6; 72,576 x 204 x 51 with its
// gradients: 24 + 21 us, and dW 10 + 7):
//   forward   x may have any pitch and offset; its rows as whole pieces (the operand of dW) are written on the way
//   backward  dz = dy act'(z) is formed in the operand's registers and written for dW
// Shared memory: the weight as [TP * 16 columns][KS * 32 places], 16 bytes between rows that keep 16 rows' pieces in different banks.
struct RowsArgs {
  const void *x, *w;
  const unsigned char* d;         // backward: derivative [rows][ldd bytes], or NULL
  float low;                      // and the derivative that a 0 bit stands for
  void* xp;                       // NULL, or the operand's rows with pitch roundup(K, 8) and zeros behind them
  size_t ldx, ldw, ldd, rows;
  int N, K;
  Epilogue e;                     // out without gaps
};
// Two neighbouring tiles' results: four consecutive columns of each per lane (columns 4 g of its tile) -> eight consecutive ones of one
// tile (g = 0, 1: the first's columns 0, 8; g = 2, 3: the second's), and back: two exchanges of 16- and 32-lane halves per register pair.
__device__ __forceinline__ u32x4 joined(const u32x2* const t) {
  u32x4 r;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const u32x2 a = __builtin_amdgcn_permlane32_swap(t[0][k], t[1][k], false, false);
    const u32x2 b = __builtin_amdgcn_permlane16_swap(a[0], a[1], false, false);
    r[k] = b[0];
    r[2 + k] = b[1];
  }
  return r;
}
__device__ __forceinline__ void apart(const u32x4 r, u32x2* const t) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const u32x2 a = __builtin_amdgcn_permlane16_swap(r[k], r[2 + k], false, false);
    const u32x2 b = __builtin_amdgcn_permlane32_swap(a[0], a[1], false, false);
    t[0][k] = b[0];
    t[1][k] = b[1];
  }
}
enum { ROWS_FWD, ROWS_FWD_KEEP, ROWS_BWD, ROWS_BWD_BITS };       // forward; and the derivative; backward with it as codes (or none), as bits
template <typename T, int KS, int MODE, int NW>
__global__ __launch_bounds__(NW * 64) void rows_kernel(const RowsArgs a) {
  constexpr bool BWD = MODE >= ROWS_BWD, BITS = MODE == ROWS_BWD_BITS, KEEP = MODE == ROWS_FWD_KEEP;
  constexpr int PITCH = KS * 64 + 16, NT = NW * 64;
  typedef T T8 __attribute__((ext_vector_type(8)));
  typedef T T4 __attribute__((ext_vector_type(4)));
  extern __shared__ __align__(16) unsigned char lds[];
  const int N = a.N, K = a.K, kp = (K + 7) & ~7, tp = (N + 15) / 16;
  float* const bias = reinterpret_cast<float*>(lds + tp * 16 * PITCH);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, q = lane & 15;

  if constexpr (!BWD) {           // w [N][K]
    for (int ch = threadIdx.x; ch < tp * 16 * KS * 4; ch += NT) {
      const int p = ch / (KS * 4), c = ch % (KS * 4) * 8;
      *reinterpret_cast<u32x4*>(lds + p * PITCH + c * 2) = raw8((const T*)a.w + p * a.ldw + c, p < N ? K - c : 0, c);
    }
  } else {                        // w [K][N]: turned; neighbouring threads take neighbouring places of the sum, whose stores share no bank
    for (int ch = threadIdx.x; ch < KS * 32 * tp * 2; ch += NT) {
      const int r = ch % (KS * 32), c = ch / (KS * 32) * 8;
      const T8 v = __builtin_bit_cast(T8, raw8((const T*)a.w + r * a.ldw + c, r < K ? N - c : 0, c));
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<T*>(lds + (c + i) * PITCH + r * 2) = v[i];
    }
  }
  for (int c = threadIdx.x; c < tp * 16; c += NT) bias[c] = !BWD && a.e.bias && c < N ? (float)((const T*)a.e.bias)[c] : 0.f;
  __syncthreads();

  const size_t tiles = (a.rows + 15) / 16;
  for (size_t t = (size_t)blockIdx.x * NW + wave; t < tiles; t += (size_t)gridDim.x * NW) {
    const size_t row0 = t * 16, row = row0 + q;
    const bool in = row < a.rows;
    i32x4 xf[KS];
    u16x8 dv[BWD && !BITS ? KS : 1];
    unsigned char db[BITS ? KS : 1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = ks * 32 + g * 8;
      xf[ks] = __builtin_bit_cast(i32x4, raw8((const T*)a.x + row * a.ldx + c, in ? K - c : 0, c));
      if constexpr (BITS) {
        db[ks] = in && c < kp ? a.d[row * a.ldd + c / 8] : (unsigned char)0;
      } else if constexpr (BWD) {
        if (a.d && in && c < kp) dv[ks] = *reinterpret_cast<const u16x8*>(a.d + row * a.ldd + c * 2);
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = ks * 32 + g * 8;
      if (BWD && a.d) {
        const T8 h = __builtin_bit_cast(T8, xf[ks]);
        T8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = (float)h[i];
          if constexpr (BITS) v = bit_slope(v, db[ks], i, a.low);             // behind row and column ends v is 0
          else v = in && c + i < K ? v * act_slope(dv[ks][i]) : 0.f;
          r[i] = (T)v;
        }
        xf[ks] = __builtin_bit_cast(i32x4, r);
      }
      if (a.xp && in && c < kp) *reinterpret_cast<i32x4*>((T*)a.xp + row * kp + c) = xf[ks];
    }
    // four tiles of 16 columns at a time: enough independent multiplies, few enough registers for 16 waves per compute unit
#pragma unroll 1
    for (int p4 = 0; p4 < tp; p4 += 4) {
      f32x4 acc[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        acc[p] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p4 + p < tp) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            acc[p] = Mma<T>::run(*reinterpret_cast<const i32x4*>(lds + ((p4 + p) * 16 + q) * PITCH + ks * 64 + g * 16), xf[ks], acc[p]);
        }
      }
#pragma unroll
      for (int pp = 0; pp < 4; pp += 2) {
        if (p4 + pp >= tp) break;
        const int col8 = (p4 + pp + (g >> 1)) * 16 + (g & 1) * 8, left = in ? N - col8 : 0;      // this lane's eight columns of the pair
        u32x2 yp[2], cp[2], rp[2];
        if (!BWD && a.e.res) apart(raw8((const T*)a.e.res + row * a.e.ldr + col8, left, col8), rp);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[4];
          if constexpr (BWD) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = acc[pp + h][i];
          } else {
            const int col = (p4 + pp + h) * 16 + g * 4;
            f32x4 b = {0.f, 0.f, 0.f, 0.f};
            if (p4 + pp + h < tp) b = *reinterpret_cast<const f32x4*>(bias + col);
            float z[4], d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = acc[pp + h][i] + b[i];
            if (KEEP && !act_bits(a.e.act)) {
              act_apply<4, true>(a.e.act, z, y, d);
              cp[h] = u32x2{act_code(d[0], z[0]) | act_code(d[1], z[1]) << 16, act_code(d[2], z[2]) | act_code(d[3], z[3]) << 16};
            } else {
              act_apply<4, false>(a.e.act, z, y, d);
              if (KEEP) cp[h] = u32x2{(z[0] > 0.f ? 1u : 0u) | (z[1] > 0.f ? 2u : 0u) | (z[2] > 0.f ? 4u : 0u) | (z[3] > 0.f ? 8u : 0u), 0u};
            }
            if (a.e.res) {
              const T4 v = __builtin_bit_cast(T4, rp[h]);
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] += (float)v[i];
            }
          }
          yp[h] = __builtin_bit_cast(u32x2, T4{(T)y[0], (T)y[1], (T)y[2], (T)y[3]});
        }
        if (KEEP) {
          const u32x4 c = joined(cp);
          unsigned char* const kept = a.e.d + row * a.e.ldd;
          if (in && left > 0) {
            if (act_bits(a.e.act)) kept[col8 / 8] = (unsigned char)(c[0] | c[2] << 4);
            else *reinterpret_cast<u32x4*>(kept + col8 * 2) = c;
          }
        }
        const u32x4 o = joined(yp);
        unsigned short* const out = (unsigned short*)a.e.out + row * N + col8;
        if (left >= 8) {
          __builtin_memcpy(out, &o, 16);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < left) out[i] = (unsigned short)(o[i / 2] >> (16 * (i & 1)));
        }
      }
    }
  }
}

// ---- rows of any width, pitch and offset, laid out again with a pitch of whole 16-byte pieces and zeros behind each row --------
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const T* const src, const size_t ld, T* const dst, const int cols, const int ldd, const size_t rows) {
  const int per = ldd * (int)sizeof(T) / 16, PIECE = 16 / (int)sizeof(T);
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= rows * per) return;
  const size_t row = id / per;
  const int c = (int)(id - row * per) * PIECE;
  T v[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) v[i] = c + i < cols ? src[row * ld + c + i] : T(0);
  __builtin_memcpy(__builtin_assume_aligned(dst + row * ldd + c, 16), v, 16);
}

// ---- dz = dy act'(z) with a pitch of whole pieces, and the column sums of each workgroup's rows (db) ----------------------------
// Bound: memory (8192 x 8192 bf16: 403 MB in 75 us, 5.4 TB/s).
struct DzArgs {
  const void* dy;
  const unsigned char* d;         // [rows][ldd bytes], or NULL: no activation
  float low;                      // what a 0 bit stands for
  void* dz;                       // or NULL: only the sums
  float* partial;                 // [gridDim.y][N] or NULL
  size_t rows, lddy, ldd, lddz;
  int N;
};
template <typename T, int L, bool WHOLE, bool BITS>
__global__ __launch_bounds__(256) void dz_kernel(const DzArgs a) {
  constexpr int G = 256 / L;
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  const int col = (blockIdx.x * L + lane) * 8, left = WHOLE ? (col < a.N ? 8 : 0) : a.N - col;       // WHOLE: N is a multiple of 8
  float sum[8] = {};
  if (left > 0) {
    constexpr int U = 4;                     // rows whose loads are in flight together
    const size_t step = (size_t)gridDim.y * G;
    for (size_t row = (size_t)blockIdx.y * G + grp; row < a.rows; row += U * step) {
      float v[U][8];
      u16x8 c[BITS ? 1 : U];
      unsigned char bits[BITS ? U : 1];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (row + k * step < a.rows) {
          load8((const T*)a.dy + (row + k * step) * a.lddy + col, left, col, v[k]);
          if constexpr (BITS) bits[k] = a.d[(row + k * step) * a.ldd + col / 8];
          else if (a.d) c[k] = *reinterpret_cast<const u16x8*>(a.d + (row + k * step) * a.ldd + col * 2);
        }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (row + k * step < a.rows) {
          if constexpr (BITS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = bit_slope(v[k][i], bits[k], i, a.low);           // 0 behind the last column
          } else if (a.d) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = i < left ? v[k][i] * act_slope(c[k][i]) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] += v[k][i];
          if (a.dz) store8((T*)a.dz + (row + k * step) * a.lddz + col, 8, v[k]);           // zeros behind the last column
        }
    }
  }
  if (!a.partial) return;
  __shared__ float red[G][L * 8 + 1];
#pragma unroll
  for (int i = 0; i < 8; ++i) red[grp][lane * 8 + i] = sum[i];
  __syncthreads();
  for (int c = threadIdx.x; c < L * 8; c += 256) {
    const int n = blockIdx.x * L * 8 + c;
    float t = 0.f;
    for (int g = 0; g < G; ++g) t += red[g][c];
    if (n < a.N) a.partial[(size_t)blockIdx.y * a.N + n] = t;
  }
}

inline int dz_lanes(const int N) { return N <= 64 ? 8 : N <= 128 ? 16 : N <= 256 ? 32 : 64; }
inline int dz_groups(const size_t rows, const int N) {
  const int L = dz_lanes(N), cols = (N + L * 8 - 1) / (L * 8);
  size_t g = (rows + 256 / L - 1) / (256 / L);
  const size_t most = 1024 / cols < 64 ? 64 : 1024 / cols;
  return (int)(g < most ? g : most);
}

// ---- which tile, and how many parts of the sum ---------------------------------------------------------------------------------
struct Plan { int tile, splits, per; };
inline Plan gemm_plan(const int M, const int N, const int R, const int es) {
  const int stages = (int)(((long)R * es + 127) / 128);
  const auto tiles = [&](const int b) { return (long)((M + b - 1) / b) * ((N + b - 1) / b); };
  Plan p{256, 1, stages};
  // Large tiles, one per compute unit at a time, where they fill the last round of the 256 units well (4096 x 4096 x 4096 in 256 of them: 106 us,
  // 113 in tiles of 128; 8192 x 4096 x 4096 in 512: 211 and 235); not where a second round would be mostly empty (5120 x 4096 x 4096 in 320: 187 us, 164
  // in tiles of 128).  From 1.5 rounds on the two differ by at most a few percent either way but for full rounds, which large tiles win.
  // What this does not weigh is how much of a tile exists: with far fewer columns or rows than a tile has, smaller ones would be quicker
  // (60,000 x 20 x 4096 in large tiles 144 us, in tiles of 64 112 and in four parts 104; 40,000 x 20 x 4096 in tiles of 128 91, of 64 69; 64 x 50,257 x 768 30, 19).
  const long large = tiles(256);
  if (large < 192 || (large > 256 && large <= 384) || stages < 4) p.tile = 128;
  // Too few tiles of 128 for the chip: tiles of 64, unless the sums are so long that reading the operands half as often pays for dividing them (f16,
  // dW of 200,704 x 512 x 512 314 us in tiles of 64, 143; of 8192 x 1024 x 1024 73, 32; below, bf16 1024 x 2048 x 2048 17 and 30) and edges waste little
  const long mid = tiles(128), small = tiles(64);
  if (p.tile == 128 && mid < 192 && (mid * stages < 8192 || 4 * mid > small + small / 4)) p.tile = 64;
  const long t = tiles(p.tile);
  // too few tiles for 256 compute units: divide the sum, at least 4 stages a part (64 x 4096 x 4096 14.4 us, undivided 35.9; 256 x 512 x 8192 16.5, 66.4)
  // and one such tile per unit leaves it half idle over a long sum (tiles of 64: 1024 x 1024 x 4096 25 us, undivided 36, but over a short one 1024 x 1024 x
  // 1024 14, 9; of 128: 2048 x 2048 x 8192 70, 88, and 2048 x 2048 x 2048 34, 30).  Exactly one: a few more already share units by themselves, and two
  // parts each are a second round (2048 x 2049 x 8192, 272 tiles: 101 us, in two parts 111; 288 tiles 105, 115; 320 105, 120; 368 112, 129)
  if (p.tile < 256 && ((t < 256 && stages > 8) || (p.tile == 64 && t < 512 && stages >= 48) || (t == 256 && stages >= 64))) {
    long s = (512 + t - 1) / t;
    if (s > stages / 4) s = stages / 4;
    if (s > 256) s = 256;
    p.splits = s < 1 ? 1 : (int)s;
  }
  p.per = (stages + p.splits - 1) / p.splits;
  if (p.per < 1) p.per = 1;
  p.splits = (stages + p.per - 1) / p.per;
  if (p.splits < 1) p.splits = 1;
  return p;
}
inline size_t up8(const size_t n) { return (n + 7) & ~(size_t)7; }
inline size_t slope_bytes(const int n, const int act) { return act_bits(act) ? up8(n) / 8 : up8(n) * 2; }      // of a row's kept derivative
inline bool slope_ok(const void* const slope, const int act) { return !slope || act_bits(act) || aligned_to(slope, 16); }
inline float slope_low(const int act) { return act == ACT_LRELU ? LRELU : 0.f; }

template <typename T, bool QX, bool PX, int BQ, int BP, int NQ, int NP>
hipError_t gemm_go(const GemmArgs& a, hipStream_t s) {
  static std::atomic<unsigned long long> optin{0};
  constexpr int stage = (BQ + BP) * 128, turn = NQ * NP * 16 * (BP / NP + 4) * 4, most = 2 * stage > turn ? 2 * stage : turn;
  const int need = a.per > 1 || BQ * BP >= 256 * 256 ? 2 * stage : stage, bytes = need > turn ? need : turn;      // one stage: one buffer, more workgroups at a time
  const void* const fn = reinterpret_cast<const void*>(&gemm_kernel<T, QX, PX, BQ, BP, NQ, NP>);
  if (const hipError_t e = lds_optin(fn, most, optin); e != hipSuccess) return e;
  const long wgs = (long)((a.M + BQ - 1) / BQ) * ((a.N + BP - 1) / BP) * a.splits;
  hipLaunchKernelGGL((gemm_kernel<T, QX, PX, BQ, BP, NQ, NP>), dim3((unsigned)wgs), dim3(NQ * NP * 64), bytes, s, a);
  return hipGetLastError();
}
template <typename T, bool QX, bool PX>
int gemm_run(GemmArgs a, hipStream_t s) {
  const Plan p = gemm_plan(a.M, a.N, a.R, sizeof(T));
  a.splits = p.splits;
  a.per = p.per;
  a.ldw = up8(a.N);
  if (p.splits > 1 && !a.ws) return SELFC_EINVAL;
  hipError_t e;
  if (p.tile == 256) e = gemm_go<T, QX, PX, 256, 256, 4, 2>(a, s);
  else if (p.tile == 128) e = gemm_go<T, QX, PX, 128, 128, 2, 2>(a, s);
  else e = gemm_go<T, QX, PX, 64, 64, 2, 2>(a, s);
  if (e != hipSuccess) return pw_rc(e);
  if (p.splits > 1) {
    const size_t n = (size_t)a.M * ((a.N + 7) / 8);
    // many parts of few columns (f16, dW of 200,704 x 128 x 64 with the rest of its layer): 88 us with 16 threads per item, 129 with one
    if (p.splits >= 16) hipLaunchKernelGGL((gemm_join_kernel<16>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((gemm_join_kernel<1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
    return pw_rc(hipGetLastError());
  }
  return SELFC_OK;
}

// ---- narrow rows: which instance, and the shared memory it takes ----------------------------------------------------------------
constexpr int ROWS_MAX = 256;
struct RowsPlan { int ks, nw, lds, per_cu; };
inline RowsPlan rows_plan(const int N, const int K) {
  RowsPlan p{};
  const int tp = (N + 15) / 16;
  p.ks = K <= 64 ? 2 : K <= 128 ? 4 : 8;
  p.lds = tp * 16 * (p.ks * 64 + 16) + tp * 64;
  // a large weight is shared by more waves (f16, 200,704 x 192 x 128: 4 waves 37.0 us, 8 32.4; 72,576 x 51 x 204: 18.4, 14.1); a small one: no difference
  p.nw = p.lds > 32 * 1024 ? 8 : 4;
  const int most = 16 / p.nw;                      // 16 waves per compute unit
  p.per_cu = 160 * 1024 / p.lds < most ? 160 * 1024 / p.lds : most;
  return p;
}
inline bool rows_ok(const int n, const int k) { return n <= ROWS_MAX && k <= ROWS_MAX; }        // 133 KiB at most: it fits
template <typename T, int MODE>
int rows_run(RowsArgs a, hipStream_t s) {
  const RowsPlan p = rows_plan(a.N, a.K);
  // workgroups that the chip holds at a time, each with its copy of the weight, or as many as there are tiles for
  const size_t need = (a.rows + p.nw * 16 - 1) / (p.nw * 16), hold = 256 * (size_t)p.per_cu;
  const dim3 grid((unsigned)(need < hold ? need : hold)), blk(p.nw * 64);
#define ROWS(KS, NW)                                                                                                              \
  {                                                                                                                               \
    static std::atomic<unsigned long long> optin{0};                                                                              \
    const void* const fn = reinterpret_cast<const void*>(&rows_kernel<T, KS, MODE, NW>);                                           \
    if (const hipError_t e = lds_optin(fn, 160 * 1024, optin); e != hipSuccess) return pw_rc(e);                                  \
    hipLaunchKernelGGL((rows_kernel<T, KS, MODE, NW>), grid, blk, p.lds, s, a);                                                    \
  }
  if (p.ks == 2 && p.nw == 4) ROWS(2, 4)
  else if (p.ks == 2) ROWS(2, 8)
  else if (p.ks == 4 && p.nw == 4) ROWS(4, 4)
  else if (p.ks == 4) ROWS(4, 8)
  else if (p.nw == 4) ROWS(8, 4)
  else ROWS(8, 8)
#undef ROWS
  return pw_rc(hipGetLastError());
}

// Few rows: a workgroup per 16 columns reads its part of the weight in one go (8192 bytes of the sum per row are on their way at once), or in
// several where there are workgroups enough and x is next to nothing.  bf16, rows x columns x sum, here and in divided tiles, from memory (and with
// the weight in the last cache):
//   1 x 2048 x 2048 7.1 us, 10.2 (7.1, 10.2);  1 x 4096 x 4096 9.5, 13.9 (7.3, 10.5);  16 x 4096 x 4096 12.2, 14.6 (10.0, 11.5);
//   1 x 4096 x 8192 17.2, 21.5 (14.3, 15.9);  16 x 16384 x 4096 40, 39 (31, 24)
// and where the tiles are taken: 1 x 1024 x 8192 12.5, 10.3 (11.4, 9.9);  16 x 2048 x 8192 19.9, 14.3 (17.1, 11.2);  8 x 8192 x 8192 34, 38 (28, 24).
// Rows as they lie, against laying them out first (f16): 16 x 1000 x 301 5.4 us, 9.5; 10 x 6832 x 1721 17, 29; 1 x 4096 x 4097 17.7, 30.0; 16 x 4096 x 4097
// 28.6, 35.4; not for longer sums (16 x 2048 x 8193 52.6, 37.1) and not below one piece.
inline bool gemv_any(const size_t rows, const int k, const size_t es) { return rows <= 16 && (size_t)k * es >= 16 && (size_t)k * es <= 8192 + 128; }
inline bool gemv_takes(const size_t rows, const int n, const int k, const size_t es) {
  return rows <= 16 && ((size_t)k * es <= 8192 || (rows <= 4 && n >= 4096));
}
// shapes whose offsets the kernels hold: 32-bit within a tile, 32-bit numbers of workgroups
inline bool lin_shape(const size_t M, const int N, const int K) {
  return M <= 0x3fffffff && N >= 1 && K >= 1 && N <= (1 << 20) && K <= (1 << 20) && (M / 64 + 1) * ((size_t)N / 64 + 1) < (1u << 28);
}
inline bool rows_fit(const void* p, const size_t ld, const size_t cols, const size_t es) {     // whole pieces at aligned places
  return aligned_to(p, 16) && (ld * es) % 16 == 0 && (cols * es) % 16 == 0 && ld < (1u << 21);
}

Epilogue make_epilogue(void* out, size_t ldo, const void* bias, const void* res, size_t ldr, int dtype, int act) {
  Epilogue e{};
  e.out = out; e.bias = bias; e.res = res; e.ldo = ldo; e.ldr = ldr; e.dtype = dtype; e.act = act;
  return e;
}

}  // namespace
}  // namespace selfc

using namespace selfc;

extern "C" {

size_t selfc_linear_ws_floats(size_t rows, int cols, int sum, int elem_bytes) {
  if (rows < 1 || rows > 0x3fffffff || cols < 1 || sum < 1) return 0;
  const Plan p = gemm_plan((int)rows, cols, sum, elem_bytes);
  return p.splits > 1 ? (size_t)p.splits * rows * up8(cols) : 0;
}

int selfc_pack_rows(const void* src, size_t ld, void* dst, size_t rows, int cols, int ldd, int elem_bytes, void* stream) {
  if (cols < 1 || ldd < cols || (elem_bytes != 1 && elem_bytes != 2) || (ldd * elem_bytes) % 16) return SELFC_EINVAL;
  if (rows == 0) return SELFC_OK;
  if (!src || !dst || !aligned_to(dst, 16)) return SELFC_EINVAL;
  const size_t n = rows * (size_t)(ldd * elem_bytes / 16);
  if (n > 0xffffff00ull) return SELFC_EINVAL;                    // a launch has fewer than 2^32 lanes
  const dim3 grid((unsigned)((n + 255) / 256)), blk(256);
  if (elem_bytes == 2) hipLaunchKernelGGL((pack_rows_kernel<unsigned short>), grid, blk, 0, (hipStream_t)stream, (const unsigned short*)src, ld, (unsigned short*)dst, cols, ldd, rows);
  else hipLaunchKernelGGL((pack_rows_kernel<unsigned char>), grid, blk, 0, (hipStream_t)stream, (const unsigned char*)src, ld, (unsigned char*)dst, cols, ldd, rows);
  return pw_rc(hipGetLastError());
}

int selfc_linear_any_layout(size_t rows, int k, int elem_bytes) { return k >= 1 && (elem_bytes == 1 || elem_bytes == 2) && gemv_any(rows, k, elem_bytes); }

int selfc_linear(const void* x, size_t ldx, const void* w, size_t ldw, const float* x_scale, const float* w_scale, const void* bias, int act,
                 const void* res, size_t ldr, void* y, void* slope, float* ws, size_t rows, int n, int k, int in_dtype, int out_dtype, void* stream) {
  if (rows == 0) return SELFC_OK;
  if (!x || !w || !y || !lin_shape(rows, n, k) || act < ACT_NONE || act > ACT_SILU || in_dtype < 1 || in_dtype > 3 || out_dtype < 0 || out_dtype > 2) return SELFC_EINVAL;
  const bool q8 = in_dtype == 3;
  if (q8 != (x_scale != nullptr) || q8 != (w_scale != nullptr) || (!q8 && in_dtype != out_dtype) || (slope && q8) || !slope_ok(slope, act)) return SELFC_EINVAL;
  const size_t es = q8 ? 1 : 2;
  const bool whole = rows_fit(x, ldx, k, es) && rows_fit(w, ldw, k, es);
  if (!whole && !(gemv_any(rows, k, es) && aligned_to(x, es) && aligned_to(w, es))) return SELFC_EINVAL;      // selfc_pack_rows first
  if ((rows > 1 && ldx < (size_t)k) || (n > 1 && ldw < (size_t)k) || (res && rows > 1 && ldr < (size_t)n)) return SELFC_EINVAL;
  GemmArgs a{};
  a.q = x; a.p = w; a.ldq = ldx; a.ldp = ldw; a.M = (int)rows; a.N = n; a.R = k; a.ws = ws;
  a.e = make_epilogue(y, n, bias, res, ldr, out_dtype, act);
  a.e.qs = x_scale; a.e.ps = w_scale; a.e.d = (unsigned char*)slope; a.e.ldd = slope_bytes(n, act);
  hipStream_t s = (hipStream_t)stream;
  if (!whole || gemv_takes(rows, n, k, es)) {
    a.splits = 1;
    const dim3 grid((n + 15) / 16), blk(512);
#define GEMV(T_)                                                                            \
  if (whole) hipLaunchKernelGGL((gemv_kernel<T_, true>), grid, blk, 0, s, a);               \
  else hipLaunchKernelGGL((gemv_kernel<T_, false>), grid, blk, 0, s, a)
    if (q8) { GEMV(unsigned char); }
    else if (in_dtype == 1) { GEMV(b16); }
    else { GEMV(h16); }
#undef GEMV
    return pw_rc(hipGetLastError());
  }
  if (q8) return gemm_run<unsigned char, false, false>(a, s);
  return in_dtype == 1 ? gemm_run<b16, false, false>(a, s) : gemm_run<h16, false, false>(a, s);
}

size_t selfc_linear_dz_floats(size_t rows, int n) { return n < 1 ? 1 : (size_t)(dz_groups(rows, n) + 1) * n; }

int selfc_linear_dz(const void* dy, size_t lddy, const void* slope, int act, void* dz, size_t lddz, void* db, float* partial, size_t rows, int n, int dtype, void* stream) {
  if (!dy || n < 1 || (dtype != 1 && dtype != 2) || (db && !partial) || (!dz && !db) || rows > 0x3fffffff) return SELFC_EINVAL;
  if (dz && (!aligned_to(dz, 16) || lddz % 8 || lddz < up8(n))) return SELFC_EINVAL;
  if (act < ACT_NONE || act > ACT_SILU || !slope_ok(slope, act)) return SELFC_EINVAL;
  const bool bits = slope && act_bits(act);
  DzArgs a{};
  a.dy = dy; a.d = (const unsigned char*)slope; a.dz = dz; a.partial = db ? partial : nullptr; a.rows = rows; a.lddy = lddy; a.lddz = lddz; a.N = n;
  a.ldd = slope_bytes(n, act); a.low = slope_low(act);
  hipStream_t s = (hipStream_t)stream;
  const int L = dz_lanes(n), groups = dz_groups(rows, n);
  if (groups) {
    const dim3 grid((n + L * 8 - 1) / (L * 8), groups), blk(256);
#define DZ2(T_, L_)                                                                                             \
  {                                                                                                            \
    if (n % 8 == 0 && bits) hipLaunchKernelGGL((dz_kernel<T_, L_, true, true>), grid, blk, 0, s, a);           \
    else if (n % 8 == 0) hipLaunchKernelGGL((dz_kernel<T_, L_, true, false>), grid, blk, 0, s, a);             \
    else if (bits) hipLaunchKernelGGL((dz_kernel<T_, L_, false, true>), grid, blk, 0, s, a);                   \
    else hipLaunchKernelGGL((dz_kernel<T_, L_, false, false>), grid, blk, 0, s, a);                            \
  }
#define DZ(L_) if (dtype == 1) DZ2(b16, L_) else DZ2(h16, L_)
    if (L == 8) { DZ(8); }
    else if (L == 16) { DZ(16); }
    else if (L == 32) { DZ(32); }
    else { DZ(64); }
#undef DZ
#undef DZ2
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return pw_rc(e);
  }
  return db ? pw_colsum(partial, groups, n, dtype, db, s) : SELFC_OK;
}

int selfc_linear_dx(const void* dz, size_t lddz, const void* w, size_t ldw, void* dx, float* ws, size_t rows, int n, int k, int dtype, void* stream) {
  if (rows == 0) return SELFC_OK;
  if (!dz || !w || !dx || !lin_shape(rows, k, n) || (dtype != 1 && dtype != 2)) return SELFC_EINVAL;
  if (!rows_fit(dz, lddz, up8(n), 2) || lddz < up8(n) || !rows_fit(w, ldw, up8(k), 2) || ldw < up8(k)) return SELFC_EINVAL;
  GemmArgs a{};
  a.q = dz; a.p = w; a.ldq = lddz; a.ldp = ldw; a.M = (int)rows; a.N = k; a.R = n; a.px = (int)up8(k); a.ws = ws;
  a.e = make_epilogue(dx, k, nullptr, nullptr, 0, dtype, ACT_NONE);
  return dtype == 1 ? gemm_run<b16, false, true>(a, (hipStream_t)stream) : gemm_run<h16, false, true>(a, (hipStream_t)stream);
}

size_t selfc_linear_dw_floats(size_t rows, int n, int k) {
  if (rows < 1 || rows > 0x3fffffff || n < 1 || k < 1) return 0;
  const Plan p = gemm_plan(n, k, (int)rows, 2);
  return p.splits > 1 ? (size_t)p.splits * n * (up8(k) + 1) : 0;
}

int selfc_linear_dw(const void* dz, size_t lddz, const void* x, size_t ldx, void* dw, void* db, float* ws, size_t rows, int n, int k, int dtype, void* stream) {
  if (!dz || !x || !dw || !lin_shape(n, k, 1) || rows < 1 || rows > 0x3fffffff || (dtype != 1 && dtype != 2)) return SELFC_EINVAL;
  if (!rows_fit(dz, lddz, up8(n), 2) || lddz < up8(n) || !rows_fit(x, ldx, up8(k), 2) || ldx < up8(k)) return SELFC_EINVAL;
  GemmArgs a{};
  a.q = dz; a.p = x; a.ldq = lddz; a.ldp = ldx; a.M = n; a.N = k; a.R = (int)rows; a.qx = (int)up8(n); a.px = (int)up8(k); a.ws = ws; a.sums = db;
  a.e = make_epilogue(dw, k, nullptr, nullptr, 0, dtype, ACT_NONE);
  return dtype == 1 ? gemm_run<b16, true, true>(a, (hipStream_t)stream) : gemm_run<h16, true, true>(a, (hipStream_t)stream);
}

int selfc_linear_rows_ok(int n, int k) { return n >= 1 && k >= 1 && rows_ok(n, k); }

int selfc_linear_rows(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, int act, const void* res, size_t ldr, void* y,
                      void* slope, void* xp, size_t rows, int n, int k, int dtype, void* stream) {
  if (rows == 0) return SELFC_OK;
  if (!x || !w || !y || n < 1 || k < 1 || !rows_ok(n, k) || rows > 0x3fffffff || act < ACT_NONE || act > ACT_SILU || (dtype != 1 && dtype != 2)) return SELFC_EINVAL;
  if ((rows > 1 && ldx < (size_t)k) || (n > 1 && ldw < (size_t)k) || (res && rows > 1 && ldr < (size_t)n)) return SELFC_EINVAL;
  if (!aligned_to(y, 16) || !slope_ok(slope, act) || (xp && !aligned_to(xp, 16))) return SELFC_EINVAL;
  RowsArgs a{};
  a.x = x; a.w = w; a.xp = xp; a.ldx = ldx; a.ldw = ldw; a.rows = rows; a.N = n; a.K = k;
  a.e.out = y; a.e.bias = bias; a.e.res = res; a.e.ldr = ldr; a.e.act = act; a.e.d = (unsigned char*)slope; a.e.ldd = slope_bytes(n, act);
  hipStream_t s = (hipStream_t)stream;
  if (slope) return dtype == 1 ? rows_run<b16, ROWS_FWD_KEEP>(a, s) : rows_run<h16, ROWS_FWD_KEEP>(a, s);
  return dtype == 1 ? rows_run<b16, ROWS_FWD>(a, s) : rows_run<h16, ROWS_FWD>(a, s);
}

int selfc_linear_rows_bwd(const void* dy, size_t lddy, const void* slope, int act, const void* w, size_t ldw, void* dx, void* dz,
                          size_t rows, int n, int k, int dtype, void* stream) {
  if (rows < 1 || !dy || !w || !dx || n < 1 || k < 1 || !rows_ok(n, k) || rows > 0x3fffffff || (dtype != 1 && dtype != 2)) return SELFC_EINVAL;
  if ((rows > 1 && lddy < (size_t)n) || (n > 1 && ldw < (size_t)k)) return SELFC_EINVAL;
  if (act < ACT_NONE || act > ACT_SILU || !aligned_to(dx, 16) || !slope_ok(slope, act) || (dz && !aligned_to(dz, 16))) return SELFC_EINVAL;
  RowsArgs a{};
  a.x = dy; a.w = w; a.d = (const unsigned char*)slope; a.low = slope_low(act); a.xp = dz;
  a.ldx = lddy; a.ldw = ldw; a.ldd = slope_bytes(n, act); a.rows = rows; a.N = k; a.K = n;
  a.e.out = dx;
  hipStream_t s = (hipStream_t)stream;
  if (slope && act_bits(act)) return dtype == 1 ? rows_run<b16, ROWS_BWD_BITS>(a, s) : rows_run<h16, ROWS_BWD_BITS>(a, s);
  return dtype == 1 ? rows_run<b16, ROWS_BWD>(a, s) : rows_run<h16, ROWS_BWD>(a, s);
}

}  // extern "C"
