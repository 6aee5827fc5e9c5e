// Layer norm over the rows of [m][d]: y = (x - mu) rstd scale + bias, mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), and its gradients
//   dx = rstd (h - mean(h) - xh mean(h xh)),  h = dy scale,  xh = (x - mu) rstd;     dscale = sum_rows dy xh;     dbias = sum_rows dy.
// Bound by memory: x read and y written once; the backward reads x and dy and writes dx once.  A row lives in the registers of LPR lanes (8 .. 64 of one
// wave, or the 256 of a workgroup), NG granules of 8 elements each, so mean and variance are two passes over registers, not over memory - the
// variance is a sum of squared deviations, never a difference of squares.  The column sums of the backward stay in registers while a persistent
// workgroup walks over its rows; each workgroup leaves one partial and a second kernel adds them in a fixed order.
// Measured: 524288 x 256 in bf16 109 us forward and 153 backward (4.9 and 5.3 TB/s), 16384 x 4096 in f16 57 and 106 (4.7 and 3.8; the wide rows' column sums
// hold the registers that would keep a second row's loads in flight), 10007 x 1023 in float32 20 and 27 (4.0 and 4.6), one row of 256 2.7.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "operators.h"
#include "operators_dev.h"

namespace nerfds_ops {

namespace {

constexpr int THREADS = 256;

// sum over the LPR lanes of a row (LPR == 256: over the workgroup, through LDS); every lane of the row gets it
template <int LPR> OPS_DEV float row_sum(float v, float* red) {
#pragma unroll
  for (int d = (LPR < 64 ? LPR : 64) / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (LPR == THREADS) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0] + red[1] + red[2] + red[3];
  }
  return v;
}

// lane `l` of a row holds granules l, l + LPR, ...
template <typename T, int LPR, int NG>
__global__ __launch_bounds__(THREADS) void k_norm_fwd(const NormFwd A) {
  __shared__ float red[4];
  constexpr int ROWS = THREADS / LPR;
  const int l = threadIdx.x % LPR, d = A.d;
  const float inv_d = 1.f / (float)d;
  for (long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LPR; row - threadIdx.x / LPR < A.m; row += (long long)gridDim.x * ROWS) {
    const bool live = row < A.m;
    const T* x = static_cast<const T*>(A.x) + row * A.ldx;
    float v[NG][8];
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int c = 8 * (l + g * LPR);
      const Gran<T> r = gran_load<T>(x + c, live ? d - c : 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) { v[g][j] = gran_get<T>(r, j); s += v[g][j]; }
    }
    const float mu = row_sum<LPR>(s, red) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[g][j] = 8 * (l + g * LPR) + j < d ? v[g][j] - mu : 0.f;
        q += v[g][j] * v[g][j];
      }
    const float rstd = 1.f / sqrtf(row_sum<LPR>(q, red) * inv_d + A.eps);
    if (!live) continue;
    if (A.stats != nullptr && l == 0) { A.stats[2 * row] = mu; A.stats[2 * row + 1] = rstd; }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int c = 8 * (l + g * LPR);
      if (c >= d) continue;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[g][j] * rstd;
      if (A.scale != nullptr) {
        const Gran<T> w = gran_load<T>(static_cast<const T*>(A.scale) + c, d - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] *= gran_get<T>(w, j);
      }
      if (A.bias != nullptr) {
        const Gran<T> w = gran_load<T>(static_cast<const T*>(A.bias) + c, d - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += gran_get<T>(w, j);
      }
      gran_store<T>(static_cast<T*>(A.y) + row * A.ldy + c, gran_pack<T>(o), d - c);
    }
  }
}

// part: [grid][2][d rounded up to 4] - column sums of dy xh, of dy
template <typename T, int LPR, int NG>
__global__ __launch_bounds__(THREADS) void k_norm_bwd(const NormBwd A, float* __restrict__ part) {
  constexpr int ROWS = THREADS / LPR;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float cols[LPR == THREADS ? 1 : THREADS * 8];
  const int l = threadIdx.x % LPR, d = A.d;
  const float inv_d = 1.f / (float)d;
  float w[NG][8], ds[NG][8], db[NG][8];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int c = 8 * (l + g * LPR);
    const Gran<T> r = A.scale != nullptr ? gran_load<T>(static_cast<const T*>(A.scale) + c, d - c) : gran_zero<T>();
#pragma unroll
    for (int j = 0; j < 8; ++j) { w[g][j] = A.scale != nullptr ? gran_get<T>(r, j) : 1.f; ds[g][j] = 0.f; db[g][j] = 0.f; }
  }
  for (long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LPR; row - threadIdx.x / LPR < A.m; row += (long long)gridDim.x * ROWS) {
    const bool live = row < A.m;
    const float mu = live ? A.stats[2 * row] : 0.f, rstd = live ? A.stats[2 * row + 1] : 0.f;
    float xh[NG][8], h[NG][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int c = 8 * (l + g * LPR);
      const Gran<T> rx = gran_load<T>(static_cast<const T*>(A.x) + row * A.ldx + c, live ? d - c : 0);
      const Gran<T> ry = gran_load<T>(static_cast<const T*>(A.dy) + row * A.lddy + c, live ? d - c : 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dy = gran_get<T>(ry, j);
        xh[g][j] = c + j < d ? (gran_get<T>(rx, j) - mu) * rstd : 0.f;
        ds[g][j] += dy * xh[g][j];
        db[g][j] += dy;
        h[g][j] = dy * w[g][j];
        s1 += h[g][j];
        s2 += h[g][j] * xh[g][j];
      }
    }
    if (A.dx == nullptr) continue;
    const float m1 = row_sum<LPR>(s1, red) * inv_d, m2 = row_sum<LPR>(s2, red) * inv_d;
    if (!live) continue;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int c = 8 * (l + g * LPR);
      if (c >= d) continue;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = rstd * (h[g][j] - m1 - xh[g][j] * m2);
      gran_store<T>(static_cast<T*>(A.dx) + row * A.lddx + c, gran_pack<T>(o), d - c);
    }
  }
  if (part == nullptr) return;
  const int dp = (d + 3) & ~3;
  float* out = part + (size_t)blockIdx.x * 2 * dp;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if constexpr (LPR == THREADS) {
        const int c = 8 * (l + g * LPR);
#pragma unroll
        for (int j = 0; j < 8; ++j) if (c + j < d) out[k * dp + c + j] = k == 0 ? ds[g][j] : db[g][j];
      } else {      // the rows side by side in this workgroup: added through LDS, in the order of their number
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) cols[threadIdx.x * 8 + j] = k == 0 ? ds[g][j] : db[g][j];
        __syncthreads();
        for (int e = threadIdx.x; e < 8 * LPR; e += THREADS) {
          float s = 0.f;
          for (int r = 0; r < ROWS; ++r) s += cols[r * LPR * 8 + e];
          const int c = 8 * g * LPR + e;
          if (c < d) out[k * dp + c] = s;
        }
      }
    }
}

// Rows too long for the registers of a workgroup: the row is read again for each of the passes (mean, deviations, output), which L2 serves.
template <typename T> __global__ __launch_bounds__(THREADS) void k_norm_fwd_long(const NormFwd A) {
  __shared__ float red[4];
  const int d = A.d;
  for (long long row = blockIdx.x; row < A.m; row += gridDim.x) {
    const T* x = static_cast<const T*>(A.x) + row * A.ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < d; c += THREADS) s += to_f32<T>(x[c]);
    const float mu = row_sum<THREADS>(s, red) / (float)d;
    float q = 0.f;
    for (int c = threadIdx.x; c < d; c += THREADS) { const float v = to_f32<T>(x[c]) - mu; q += v * v; }
    const float rstd = 1.f / sqrtf(row_sum<THREADS>(q, red) / (float)d + A.eps);
    if (A.stats != nullptr && threadIdx.x == 0) { A.stats[2 * row] = mu; A.stats[2 * row + 1] = rstd; }
    for (int c = threadIdx.x; c < d; c += THREADS) {
      float v = (to_f32<T>(x[c]) - mu) * rstd;
      if (A.scale != nullptr) v *= to_f32<T>(static_cast<const T*>(A.scale)[c]);
      if (A.bias != nullptr) v += to_f32<T>(static_cast<const T*>(A.bias)[c]);
      static_cast<T*>(A.y)[row * A.ldy + c] = from_f32<T>(v);
    }
  }
}
// (the column sums of a workgroup accumulate in its own partial: thread t owns the columns t + 256 i)
template <typename T> __global__ __launch_bounds__(THREADS) void k_norm_bwd_long(const NormBwd A, float* __restrict__ part) {
  __shared__ float red[4];
  const int d = A.d, dp = (d + 3) & ~3;
  float* out = part + (size_t)blockIdx.x * 2 * dp;
  if (part != nullptr)
    for (int c = threadIdx.x; c < d; c += THREADS) { out[c] = 0.f; out[dp + c] = 0.f; }
  for (long long row = blockIdx.x; row < A.m; row += gridDim.x) {
    const T* x = static_cast<const T*>(A.x) + row * A.ldx;
    const T* gy = static_cast<const T*>(A.dy) + row * A.lddy;
    const float mu = A.stats[2 * row], rstd = A.stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < d; c += THREADS) {
      const float dy = to_f32<T>(gy[c]), xh = (to_f32<T>(x[c]) - mu) * rstd, h = A.scale != nullptr ? dy * to_f32<T>(static_cast<const T*>(A.scale)[c]) : dy;
      if (part != nullptr) { out[c] += dy * xh; out[dp + c] += dy; }
      s1 += h;
      s2 += h * xh;
    }
    if (A.dx == nullptr) continue;
    const float m1 = row_sum<THREADS>(s1, red) / (float)d, m2 = row_sum<THREADS>(s2, red) / (float)d;
    for (int c = threadIdx.x; c < d; c += THREADS) {
      const float dy = to_f32<T>(gy[c]), xh = (to_f32<T>(x[c]) - mu) * rstd, h = A.scale != nullptr ? dy * to_f32<T>(static_cast<const T*>(A.scale)[c]) : dy;
      static_cast<T*>(A.dx)[row * A.lddx + c] = from_f32<T>(rstd * (h - m1 - xh * m2));
    }
  }
}

long long up(long long a, long long b) { return (a + b - 1) / b; }
long long up4(long long a) { return (a + 3) & ~3LL; }

// lanes per row and granules per lane: the fewest lanes that hold a row in 2 granules each, then whole waves of 4, then the workgroup; 0 = longer than that
struct RowShape { int lpr, ng; };
RowShape row_shape(int d) {
  if (d <= 64) return {8, 1};
  if (d <= 128) return {16, 1};
  if (d <= 256) return {32, 1};
  if (d <= 512) return {64, 1};
  if (d <= 1024) return {64, 2};
  if (d <= 2048) return {256, 1};
  if (d <= 4096) return {256, 2};
  if (d <= 8192) return {256, 4};
  return {0, 0};
}
int bwd_grid(long long m, int d, int num_cus) {
  const RowShape s = row_shape(d);
  const long long groups = s.lpr ? up(m, THREADS / s.lpr) : m, most = 4LL * num_cus;
  return (int)(groups < most ? groups : most);
}

#define NORM_SHAPES(X) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(64, 2) X(256, 1) X(256, 2) X(256, 4)

template <typename T> void fwd_t(hipStream_t st, const NormFwd& a, int num_cus) {
  const RowShape s = row_shape(a.d);
  const long long groups = s.lpr ? up(a.m, THREADS / s.lpr) : a.m, most = 32LL * num_cus;
  const dim3 grid((unsigned)(groups < most ? groups : most));
#define X(L, G) if (s.lpr == L && s.ng == G) { hipLaunchKernelGGL((k_norm_fwd<T, L, G>), grid, dim3(THREADS), 0, st, a); return; }
  NORM_SHAPES(X)
#undef X
  hipLaunchKernelGGL((k_norm_fwd_long<T>), grid, dim3(THREADS), 0, st, a);
}
template <typename T> void bwd_t(hipStream_t st, const NormBwd& a, int num_cus) {
  if (a.m == 0) {      // an empty sum is zero
    sum_splits<T>(st, SplitSum{nullptr, 0, a.d, a.dscale}, SplitSum{nullptr, 0, a.d, a.dbias}, 0);
    return;
  }
  const RowShape s = row_shape(a.d);
  const int grid = bwd_grid(a.m, a.d, num_cus);
  float* part = a.dscale != nullptr || a.dbias != nullptr ? a.ws : nullptr;
  bool done = false;
#define X(L, G) if (s.lpr == L && s.ng == G) { hipLaunchKernelGGL((k_norm_bwd<T, L, G>), dim3(grid), dim3(THREADS), 0, st, a, part); done = true; }
  NORM_SHAPES(X)
#undef X
  if (!done) hipLaunchKernelGGL((k_norm_bwd_long<T>), dim3(grid), dim3(THREADS), 0, st, a, part);
  if (part != nullptr) sum_splits<T>(st, SplitSum{part, 2 * up4(a.d), a.d, a.dscale}, SplitSum{part + up4(a.d), 2 * up4(a.d), a.d, a.dbias}, grid);
}

}  // namespace

size_t norm_bwd_ws(const NormBwd& a, int num_cus) {
  return a.dscale != nullptr || a.dbias != nullptr ? (size_t)bwd_grid(a.m, a.d, num_cus) * 2 * up4(a.d) * sizeof(float) : 0;
}
void norm_forward(hipStream_t st, const NormFwd& a, int num_cus) {
  if (a.dtype == F32) fwd_t<float>(st, a, num_cus);
  else if (a.dtype == F16) fwd_t<f16_t>(st, a, num_cus);
  else fwd_t<bf16_t>(st, a, num_cus);
}
void norm_backward(hipStream_t st, const NormBwd& a, int num_cus) {
  if (a.dtype == F32) bwd_t<float>(st, a, num_cus);
  else if (a.dtype == F16) bwd_t<f16_t>(st, a, num_cus);
  else bwd_t<bf16_t>(st, a, num_cus);
}

}  // namespace nerfds_ops
