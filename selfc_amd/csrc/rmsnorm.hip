// Root-mean-square norm over the last axis with the residual's addition in front of it:
//   h = x + r (rounded to the rows' type: it is an output, the stream that the layers add to)
//   y = h rstd w,   rstd = 1 / sqrt(mean(h^2) + eps)
// as rows of the input's type or as e4m3 with one scale per row (largest |y| of the row = 448 steps), and its gradient
//   dx = dr = rstd (dy w - n c) + dh,   n = h rstd,  c = mean(dy w n),      dw = sum over rows of dy n.
// The norm is that of the ROUNDED h, so the backward pass needs h alone and recomputes rstd from the row it holds anyway.
//
// Bound: memory.  A row is read once into registers, eight values per lane and load, and everything that is summed over it is a
// butterfly over the lanes that share it: the smallest power of two of lanes (8..64) that covers the row, so narrow rows (64
// channels: 8 lanes) leave no lane idle, up to 2,048 values; a workgroup of 256 up to 16,384.  dw: a workgroup keeps its columns'
// sums in registers over all of its rows and writes one row of partial sums; a second launch adds them in a fixed order (no
// atomics: the same bits every time).
#include "pointwise.hpp"
#include "prof.hpp"

namespace selfc {
namespace {

constexpr int RN_MAX = 16384;
constexpr float E4M3_MAX = 448.f;

// sum / max over a row's lanes.  L <= 64: a butterfly; L = 256: the workgroup, through four LDS words (two sets, used in turn, so
// that one barrier per reduction is enough)
template <int L, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* const red) {
  v = MAX ? lanes_max<(L < 64 ? L : 64)>(v) : lanes_sum<(L < 64 ? L : 64)>(v);
  if constexpr (L == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

struct RnArgs {
  const void *x, *r, *w;
  void *h, *y;
  float* scale;
  size_t rows, ldx, ldr;
  int C, w_f32, run;          // run: values per load and store (8, 4, 2 or 1)
  float eps;
};

// L lanes per row, NV vectors of 8 values per lane
template <typename T, int L, int NV, bool Q8, bool RUN8>
__global__ __launch_bounds__(256) void rmsnorm_kernel(const RnArgs a) {
  __shared__ float red[8];
  const int lane = threadIdx.x & (L - 1);
  const size_t row = (size_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= a.rows) return;                 // L = 256: the whole workgroup, so no barrier is left behind
  const T* const x = (const T*)a.x + row * a.ldx;
  const T* const r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const int C = a.C;
  const int run = RUN8 ? 8 : a.run;           // whole 16-byte pieces: no other loads are compiled in
  float h[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * L + lane) * 8;
    load8(x + c, C - c, run, h[j]);
  }
  if (r) {
    float t[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      load8(r + c, C - c, run, t[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = (float)(T)(h[j][i] + t[j][i]);
      if (c < C) store8((T*)a.h + row * C + c, C - c, run, h[j]);
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
    if (a.w_f32) load8((const float*)a.w + c, C - c, run, w);
    else load8((const T*)a.w + c, C - c, run, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[j][i] = h[j][i] * rstd * w[i];
      if constexpr (Q8) most = fmaxf(most, fabsf(h[j][i]));
    }
    if constexpr (!Q8) {
      if (c < C) store8((T*)a.y + row * C + c, C - c, run, h[j]);
    }
  }
  if constexpr (Q8) {
    most = row_reduce<L, true>(most, red + 4);
    // a row of zeros: scale 1; a row whose largest value is below 448 steps of 2^-126: that step, so that its reciprocal is finite
    const float scale = most > 0.f ? fmaxf(most / E4M3_MAX, 0x1p-126f) : 1.f;
    const float inv = 1.f / scale;
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
        if (run == 8) {
          *reinterpret_cast<u32x2*>(q) = u32x2{(unsigned)lo, (unsigned)hi};
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
  int C, w_f32, run, want_dx;
  float eps;
};

template <typename T, int L, int NV, bool RUN8>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(const RnBwdArgs a) {
  __shared__ float red[2][8];
  constexpr int G = 256 / L;                 // rows at a time
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  const int C = a.C;
  const int run = RUN8 ? 8 : a.run;           // whole 16-byte pieces: no other loads are compiled in
  float dw[NV][8] = {};
  int turn = 0;
  for (size_t row = (size_t)blockIdx.x * G + grp; row < a.rows; row += (size_t)gridDim.x * G, turn ^= 1) {
    float h[NV][8], dy[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      load8((const T*)a.h + row * a.ldh + c, C - c, run, h[j]);
      load8((const T*)a.dy + row * C + c, C - c, run, dy[j]);
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      float w[8];
      if (a.w_f32) load8((const float*)a.w + c, C - c, run, w);
      else load8((const T*)a.w + c, C - c, run, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += h[j][i] * h[j][i];
        dot += dy[j][i] * w[i] * h[j][i];
      }
    }
    ss = row_reduce<L, false>(ss, red[turn]);
    dot = row_reduce<L, false>(dot, red[turn] + 4);
    const float rstd = 1.f / sqrtf(ss / (float)C + a.eps);
    const float c2 = dot * rstd / (float)C;                      // mean(dy w n)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * 8;
      float w[8], add[8], out[8];
      if (a.w_f32) load8((const float*)a.w + c, C - c, run, w);
      else load8((const T*)a.w + c, C - c, run, w);
      if (a.dh) load8((const T*)a.dh + row * C + c, C - c, run, add);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = h[j][i] * rstd;
        dw[j][i] += dy[j][i] * n;
        out[i] = rstd * (dy[j][i] * w[i] - n * c2);
        if (a.dh) out[i] += add[i];
      }
      if (a.want_dx && c < C) store8((T*)a.dx + row * C + c, C - c, run, out);
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
    for (int g = slice; g < rows; g += 64) acc += partial[(size_t)g * C + col];
  __shared__ float red[64][17];
  red[slice][threadIdx.x & 15] = acc;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (slice < o) red[slice][threadIdx.x & 15] += red[slice + o][threadIdx.x & 15];
    __syncthreads();
  }
  if (slice == 0 && col < C) out[col] = (T)red[0][threadIdx.x & 15];
}

// workgroups of the backward pass: enough to fill the chip several times, few enough that the partial sums stay small beside the rows
inline int rn_bwd_groups(const size_t rows, const int C) {
  const int L = C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 2048 ? 64 : 256;
  const size_t need = (rows + 256 / L - 1) / (256 / L);
  return (int)(need < 1024 ? need : 1024);
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
    if (a.run == 8) hipLaunchKernelGGL((rmsnorm_kernel<T, L, NV, Q8, true>), grid, dim3(256), 0, s, a);                       \
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
    if (a.run == 8) hipLaunchKernelGGL((rmsnorm_bwd_kernel<T, L, NV, true>), dim3((unsigned)groups), dim3(256), 0, s, a);     \
    else hipLaunchKernelGGL((rmsnorm_bwd_kernel<T, L, NV, false>), dim3((unsigned)groups), dim3(256), 0, s, a);               \
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

bool rn_shape(const size_t rows, const int C, const int dtype) {
  return C >= 1 && C <= RN_MAX && rows <= 0x7fffffffull && dtype >= 0 && dtype <= 2;
}

}  // namespace

extern "C" {

int selfc_rmsnorm(const void* x, size_t ldx, const void* r, size_t ldr, const void* w, int w_f32, void* h, void* y, float* q8_scale,
                  size_t rows, int C, int dtype, float eps, void* stream) {
  if (!rn_shape(rows, C, dtype) || !x || !w || !y || (r != nullptr) != (h != nullptr) || !(eps >= 0.f)) return SELFC_EINVAL;
  if (rows > 1 && (ldx < (size_t)C || (r && ldr < (size_t)C))) return SELFC_EINVAL;
  if (rows == 0) return SELFC_OK;
  const size_t es = dtype ? 2 : 4;
  RnArgs a{};
  a.x = x; a.r = r; a.w = w; a.h = h; a.y = y; a.scale = q8_scale; a.rows = rows; a.ldx = ldx; a.ldr = ldr; a.C = C; a.w_f32 = w_f32; a.eps = eps;
  const auto least = [](const int p, const int q) { return p < q ? p : q; };
  a.run = least(row_run(x, rows > 1 ? ldx : C, C, es), least(row_run(w, C, C, w_f32 ? 4 : es), row_run(y, C, C, q8_scale ? 1 : es)));
  if (r) a.run = least(a.run, least(row_run(r, rows > 1 ? ldr : C, C, es), row_run(h, C, C, es)));
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
  const size_t es = dtype ? 2 : 4;
  RnBwdArgs a{};
  a.h = h; a.w = w; a.dy = dy; a.dh = dh; a.dx = dx; a.partial = dw ? partial : nullptr; a.rows = rows; a.ldh = ldh; a.C = C; a.w_f32 = w_f32;
  a.want_dx = dx != nullptr; a.eps = eps;
  const auto least = [](const int p, const int q) { return p < q ? p : q; };
  a.run = least(row_run(h, rows > 1 ? ldh : C, C, es), least(row_run(w, C, C, w_f32 ? 4 : es), row_run(dy, C, C, es)));
  if (dh) a.run = least(a.run, row_run(dh, C, C, es));
  if (dx) a.run = least(a.run, row_run(dx, C, C, es));
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
