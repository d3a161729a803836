// Root-mean-square norm over the last axis with the residual's addition in front of it:
//   h = x + r (rounded to the rows' type: it is an output, the stream that the layers add to)
//   y = h rstd w,   rstd = 1 / sqrt(mean(h^2) + eps)
// as rows of the input's type or as e4m3 with one scale per row (largest |y| of the row = 448 steps), and its gradient
//   dx = dr = rstd (dy w - n c) + dh,   n = h rstd,  c = mean(dy w n),      dw = sum over rows of dy n.
// The norm is that of the ROUNDED h, so the backward pass needs h alone and recomputes rstd from the row it holds anyway.
//
// Bound: memory.  A row is read once into registers, eight values per lane and load, and everything that is summed over it is a
// butterfly over the lanes that share it: the smallest power of two of lanes (8..64) that covers the row, so narrow rows (64
// channels: 8 lanes) leave no lane idle, up to 2,048 values; a workgroup of 256 up to 16,384.  The backward pass holds two rows
// (h and dy), the next ones' and dw's sums as well, so its rows go to a workgroup from 1,024 values on (256, 512, 1,024 lanes: more lanes, not
// more values per lane, which would spill; from 8,193 values on 1,024 lanes have 128 registers each, and 16-bit rows spill after all: 4 registers for whole
// rows, 50 to 56 for widths that are not a multiple of 8).  dw: a workgroup keeps its columns' sums in registers over all of its rows and writes
// one row of partial sums; a second launch adds them in a fixed order (no atomics: the same bits every time).
// Measured (a large copy: 5.15 TB/s): 8,192 rows of 4,096 in bf16 with residual, forward 44 us (268 MB, 6.1 TB/s: part of the input is still in the
// last cache), backward 63 us (268 MB and 17 MB of partial sums) + 5 for their sum; 200,704 rows of 64 in f16, 21, 23.5 and 4 us (103 MB each way).
// Forward and backward from a graph, with an fp32 weight (what memory takes at a large copy's rate): 8,192 x 4,096 fp32 214 us (209), 200,704 x 64 fp32 79
// (80); bf16 4,096 x 8,192 131 (104), 2,048 x 16,384 144 (104), 2,048 x 16,380 215 (104): the last two pay for their spills.
#include "pointwise.hpp"

namespace selfc {
namespace {

constexpr int RN_MAX = 16384;
constexpr float E4M3_MAX = 448.f;
#define LEFT(c) (WHOLE ? ((c) < C ? 8 : 0) : C - (c))

// sum / max over a row's lanes.  L <= 64: a butterfly; more: the workgroup, through one LDS word per wave (callers use two sets in
// turn, so that one barrier per reduction is enough)
template <int L, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* const red) {
  v = MAX ? lanes_max<(L < 64 ? L : 64)>(v) : lanes_sum<(L < 64 ? L : 64)>(v);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < L / 64; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

struct RnArgs {
  const void *x, *r, *w;
  void *h, *y;
  float* scale;
  size_t rows, ldx, ldr;
  int C, w_f32;
  float eps;
};

// L lanes per row, NV vectors of 8 values per lane.  WHOLE: C is a multiple of 8, so that no vector is cut by the row's end
template <typename T, int L, int NV, bool Q8, bool WHOLE>
__global__ __launch_bounds__(256) void rmsnorm_kernel(const RnArgs a) {
  __shared__ float red[8];
  const int lane = threadIdx.x & (L - 1);
  const size_t row = (size_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= a.rows) return;                 // L = 256: the whole workgroup, so no barrier is left behind
  const T* const x = (const T*)a.x + row * a.ldx;
  const T* const r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const int C = a.C;
  float h[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * L + lane) * 8;
    load8(x + c, LEFT(c), c, h[j]);
  }
  if (r) {
    float t[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      load8(r + c, LEFT(c), c, t[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = (float)(T)(h[j][i] + t[j][i]);
      if (c < C) store8((T*)a.h + row * C + c, LEFT(c), h[j]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += h[j][i] * h[j][i];
  ss = row_reduce<L, false>(ss, red);
  const float rstd = 1.f / sqrtf(ss / (float)C + a.eps);
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * L + lane) * 8;
    float w[8];
    if (a.w_f32) load8((const float*)a.w + c, LEFT(c), c, w);
    else load8((const T*)a.w + c, LEFT(c), c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[j][i] = h[j][i] * rstd * w[i];
      if constexpr (Q8) most = fmaxf(most, fabsf(h[j][i]));
    }
    if constexpr (!Q8) {
      if (c < C) store8((T*)a.y + row * C + c, LEFT(c), h[j]);
    }
  }
  if constexpr (Q8) {
    most = row_reduce<L, true>(most, red + 4);
    // a row of zeros: scale 1; a row whose largest value is below 448 steps of 2^-126: that step, so that its reciprocal is finite
    const float scale = most > 0.f ? fmaxf(most / E4M3_MAX, 0x1p-126f) : 1.f;
    const float inv = 1.f / scale;            // (a product with it differs from a division by up to a last bit: a value at a tie may take the neighbouring code)
    if (lane == 0) a.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      if (c < C) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[j][0] * inv, h[j][1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[j][2] * inv, h[j][3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[j][4] * inv, h[j][5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[j][6] * inv, h[j][7] * inv, hi, true);
        unsigned char* const q = (unsigned char*)a.y + row * C + c;
        const int two[2] = {lo, hi};
        if (c + 8 <= C) {
          __builtin_memcpy(q, two, 8);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < C) q[i] = (unsigned char)((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
      }
    }
  }
}

struct RnBwdArgs {
  const void *h, *w, *dy, *dh;
  void* dx;
  float* partial;             // [gridDim.x][C]
  size_t rows, ldh;
  int C, w_f32, want_dx;
  float eps;
};

// The next row's values are on their way while a row is worked on: they stay as they are stored until their turn (the widest rows'
// workgroups have no registers left for that).
template <typename T, int L, int NV, bool WHOLE>
__global__ __launch_bounds__(L > 256 ? L : 256) void rmsnorm_bwd_kernel(const RnBwdArgs a) {
  constexpr int NT = L > 256 ? L : 256, G = NT / L;                // rows at a time
  constexpr bool AHEAD = L < 1024;
  __shared__ float red[2][2][L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  const int C = a.C;
  const size_t step = (size_t)gridDim.x * G;
  float dw[NV][8] = {};
  Raw8<T> nh[NV], ny[NV], nd[NV];
  const auto fetch = [&](const size_t row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      nh[j].load((const T*)a.h + row * a.ldh + c, LEFT(c), c);
      ny[j].load((const T*)a.dy + row * C + c, LEFT(c), c);
      if (a.dh) nd[j].load((const T*)a.dh + row * C + c, LEFT(c), c);
    }
  };
  size_t row = (size_t)blockIdx.x * G + grp;
  if (AHEAD && row < a.rows) fetch(row);
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    if (!AHEAD) fetch(row);
    Raw8<T> rh[NV], ry[NV], rd[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) { rh[j] = nh[j]; ry[j] = ny[j]; rd[j] = nd[j]; }
    if (AHEAD && row + step < a.rows) fetch(row + step);
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      float h[8], dy[8], w[8];
      rh[j].expand(h);
      ry[j].expand(dy);
      if (a.w_f32) load8((const float*)a.w + c, LEFT(c), c, w);
      else load8((const T*)a.w + c, LEFT(c), c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += h[i] * h[i];
        dot += dy[i] * w[i] * h[i];
      }
    }
    ss = row_reduce<L, false>(ss, red[turn][0]);
    dot = row_reduce<L, false>(dot, red[turn][1]);
    const float rstd = 1.f / sqrtf(ss / (float)C + a.eps);
    const float c2 = dot * rstd / (float)C;                      // mean(dy w n)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      float h[8], dy[8], w[8], add[8], out[8];
      rh[j].expand(h);
      ry[j].expand(dy);
      if (a.dh) rd[j].expand(add);
      if (a.w_f32) load8((const float*)a.w + c, LEFT(c), c, w);
      else load8((const T*)a.w + c, LEFT(c), c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = h[i] * rstd;
        dw[j][i] += dy[i] * n;
        out[i] = rstd * (dy[i] * w[i] - n * c2);
        if (a.dh) out[i] += add[i];
      }
      if (a.want_dx && c < C) store8((T*)a.dx + row * C + c, LEFT(c), out);
    }
  }
  if (!a.partial) return;
  if constexpr (L < 64) {                    // lanes that hold the same columns
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] += __shfl_xor(dw[j][i], o);
  }
  if constexpr (L <= 64) {
    __shared__ float sum[4][L * NV * 8];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < L) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[wave][(j * L + lane) * 8 + i] = dw[j][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) a.partial[(size_t)blockIdx.x * C + c] = (sum[0][c] + sum[1][c]) + (sum[2][c] + sum[3][c]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) a.partial[(size_t)blockIdx.x * C + c + i] = dw[j][i];
    }
  }
}

// out[c] = sum over g of partial[g][c], in a fixed order: 16 columns x 64 slices per workgroup
template <typename T>
__global__ __launch_bounds__(1024) void colsum_kernel(const float* const partial, const int rows, const int C, T* const out) {
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
  float acc = 0.f;
  if (col < C)
    for (int g = slice; g < rows; g += 512) {          // eight loads in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = g + k * 64 < rows ? partial[(size_t)(g + k * 64) * C + col] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc += v[k];
    }
  __shared__ float red[64][17];
  red[slice][threadIdx.x & 15] = acc;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (slice < o) red[slice][threadIdx.x & 15] += red[slice + o][threadIdx.x & 15];
    __syncthreads();
  }
  if (slice == 0 && col < C) out[col] = (T)red[0][threadIdx.x & 15];
}

// workgroups of the backward pass: two to four per compute unit; a workgroup's partial sums are C values to write and read again
inline int rn_bwd_groups(const size_t rows, const int C) {
  const int at_a_time = C <= 64 ? 32 : C <= 128 ? 16 : C <= 256 ? 8 : C <= 1024 ? 4 : 1;
  const size_t need = (rows + at_a_time - 1) / at_a_time, most = C <= 2048 ? 1024 : 512;
  return (int)(need < most ? need : most);
}

}  // namespace

int pw_colsum(const float* partial, int rows, int C, int dtype, void* out, hipStream_t s) {
  const dim3 grid((C + 15) / 16), blk(1024);
  if (dtype == 0) hipLaunchKernelGGL((colsum_kernel<float>), grid, blk, 0, s, partial, rows, C, (float*)out);
  else if (dtype == 1) hipLaunchKernelGGL((colsum_kernel<b16>), grid, blk, 0, s, partial, rows, C, (b16*)out);
  else hipLaunchKernelGGL((colsum_kernel<h16>), grid, blk, 0, s, partial, rows, C, (h16*)out);
  return pw_rc(hipGetLastError());
}

}  // namespace selfc

using namespace selfc;

namespace {

// the kernel for a row of C values: lanes per row and vectors per lane
template <typename T, bool Q8>
void rn_launch(const RnArgs& a, hipStream_t s) {
#define RN(L, NV)                                                                                                            \
  do {                                                                                                                        \
    const dim3 grid((unsigned)((a.rows + 256 / L - 1) / (256 / L)));                                                          \
    if (C % 8 == 0) hipLaunchKernelGGL((rmsnorm_kernel<T, L, NV, Q8, true>), grid, dim3(256), 0, s, a);                       \
    else hipLaunchKernelGGL((rmsnorm_kernel<T, L, NV, Q8, false>), grid, dim3(256), 0, s, a);                                 \
  } while (0)
  const int C = a.C;
  if (C <= 64) RN(8, 1);
  else if (C <= 128) RN(16, 1);
  else if (C <= 256) RN(32, 1);
  else if (C <= 512) RN(64, 1);
  else if (C <= 1024) RN(64, 2);
  else if (C <= 2048) RN(64, 4);
  else if (C <= 4096) RN(256, 2);
  else if (C <= 8192) RN(256, 4);
  else RN(256, 8);
#undef RN
}
template <typename T>
void rn_bwd_launch(const RnBwdArgs& a, const int groups, hipStream_t s) {
#define RN(L, NV)                                                                                                            \
  do {                                                                                                                        \
    const dim3 grid((unsigned)groups), blk(L > 256 ? L : 256);                                                                \
    if (C % 8 == 0) hipLaunchKernelGGL((rmsnorm_bwd_kernel<T, L, NV, true>), grid, blk, 0, s, a);                             \
    else hipLaunchKernelGGL((rmsnorm_bwd_kernel<T, L, NV, false>), grid, blk, 0, s, a);                                       \
  } while (0)
  const int C = a.C;
  if (C <= 64) RN(8, 1);
  else if (C <= 128) RN(16, 1);
  else if (C <= 256) RN(32, 1);
  else if (C <= 512) RN(64, 1);
  else if (C <= 1024) RN(64, 2);
  else if (C <= 2048) RN(256, 1);
  else if (C <= 4096) RN(256, 2);
  else if (C <= 8192) RN(512, 2);
  else RN(1024, 2);
#undef RN
}

// rows: a launch has fewer than 2^32 lanes, and the forward pass takes 8 (C <= 64) to 256 of them for a row
bool rn_shape(const size_t rows, const int C, const int dtype) {
  if (C < 1 || C > RN_MAX || dtype < 0 || dtype > 2) return false;
  const size_t lanes = C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 2048 ? 64 : 256;
  return rows <= 0x7fffffffull && rows <= 0xffffff00ull / lanes;
}

}  // namespace

extern "C" {

int selfc_rmsnorm(const void* x, size_t ldx, const void* r, size_t ldr, const void* w, int w_f32, void* h, void* y, float* q8_scale,
                  size_t rows, int C, int dtype, float eps, void* stream) {
  if (!rn_shape(rows, C, dtype) || !x || !w || !y || (r != nullptr) != (h != nullptr) || !(eps >= 0.f)) return SELFC_EINVAL;
  if (rows > 1 && (ldx < (size_t)C || (r && ldr < (size_t)C))) return SELFC_EINVAL;
  if (rows == 0) return SELFC_OK;
  RnArgs a{};
  a.x = x; a.r = r; a.w = w; a.h = h; a.y = y; a.scale = q8_scale; a.rows = rows; a.ldx = ldx; a.ldr = ldr; a.C = C; a.w_f32 = w_f32; a.eps = eps;
  hipStream_t s = (hipStream_t)stream;
  if (q8_scale) {
    if (dtype == 0) rn_launch<float, true>(a, s);
    else if (dtype == 1) rn_launch<b16, true>(a, s);
    else rn_launch<h16, true>(a, s);
  } else {
    if (dtype == 0) rn_launch<float, false>(a, s);
    else if (dtype == 1) rn_launch<b16, false>(a, s);
    else rn_launch<h16, false>(a, s);
  }
  return pw_rc(hipGetLastError());
}

size_t selfc_rmsnorm_bwd_floats(size_t rows, int C) { return C < 1 ? 1 : (size_t)(rn_bwd_groups(rows, C) + 1) * (size_t)C; }

int selfc_rmsnorm_bwd(const void* h, size_t ldh, const void* w, int w_f32, const void* dy, const void* dh, void* dx, void* dw,
                      float* partial, size_t rows, int C, int dtype, float eps, void* stream) {
  if (!rn_shape(rows, C, dtype) || !h || !w || !dy || (!dx && !dw) || (dw && !partial) || !(eps >= 0.f)) return SELFC_EINVAL;
  if (rows > 1 && ldh < (size_t)C) return SELFC_EINVAL;
  RnBwdArgs a{};
  a.h = h; a.w = w; a.dy = dy; a.dh = dh; a.dx = dx; a.partial = dw ? partial : nullptr; a.rows = rows; a.ldh = ldh; a.C = C; a.w_f32 = w_f32;
  a.want_dx = dx != nullptr; a.eps = eps;
  hipStream_t s = (hipStream_t)stream;
  const int groups = rn_bwd_groups(rows, C);
  if (groups) {
    if (dtype == 0) rn_bwd_launch<float>(a, groups, s);
    else if (dtype == 1) rn_bwd_launch<b16>(a, groups, s);
    else rn_bwd_launch<h16>(a, groups, s);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return pw_rc(e);
  }
  if (!dw) return SELFC_OK;
  return pw_colsum(partial, groups, C, w_f32 ? 0 : dtype, dw, s);            // no rows: zeros
}

}  // extern "C"
