// Orthogonalised updates: X0 = U / |U|_F, then `steps` times  A = X X^T,  B = b A + c A A,  X <- a X + B X  - the odd quintic a s + b s^3 + c s^5 on
// every singular value s of X, which carries all of (0, 1] into about [0.7, 1.2].  With (a, b, c) as below it keeps [0, 1.2025] inside itself, so every
// element of X, A and B is bounded (1.21, 1.45, 2.81) whatever U was.  U is taken with its short side as rows (a tall U is transposed on the way in
// and out), so A and B are the smaller Gram matrices.
//
// Arithmetic: matrices live between the products as two f16 planes, hi + lo = value * 2^15 (B: 2^14), 22 significand bits; a product is three MFMAs
// (hi hi + hi lo + lo hi) with float32 accumulation.  The bounds above keep the planes inside f16's range, and what is dropped (lo lo) is 2^-24 of
// a product: measured against 64 bits it is as exact as float32 products (6e-7 after five steps at 256 x 256), at three times their rate.  One f16 plane
// alone costs 2e-3 ... 5e-3, more than a bf16 result may be off.
//
// Any number of matrices of any shapes runs in one launch per product (up to 64 per launch; the list rides in the kernel arguments, so a captured
// graph needs no other memory than the workspace).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "operators.h"
#include "operators_dev.h"

namespace nerfds_ops {

namespace {

constexpr int THREADS = 256, TILE = 64, BK = 64, MAX_BATCH = 64;
constexpr int SUM_ELEMS = 16384;                        // elements of U per workgroup of the norm
constexpr float CA = 3.4445f, CB = -4.7750f, CC = 2.0315f;
constexpr float SX = 32768.f, SB = 16384.f;             // plane scales of X and A; of B
constexpr double TINY = 1e-30;                          // |U| below this divides as this: a zero matrix gives zero

struct Mat {
  const void* u; void* o;
  long long ldu, ldo;
  long long ws;             // byte offset of its workspace
  int rows, cols;
  int first;                // first workgroup of this launch that works on it
  int pad;
};
struct Batch { int count, total; char* ws; Mat m[MAX_BATCH]; };
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

// workspace of one matrix: planes of X twice (read one, write the other), A, B, the partial sums of the norm
struct Layout {
  int n, m, np, mp, sums;   // short and long side, both rounded up to whole tiles
  long long x[2], a, b, part, bytes;
  __host__ __device__ Layout(int rows, int cols) {
    n = rows < cols ? rows : cols; m = rows < cols ? cols : rows;
    np = (n + TILE - 1) / TILE * TILE; mp = (m + TILE - 1) / TILE * TILE;
    sums = (int)(((long long)rows * cols + SUM_ELEMS - 1) / SUM_ELEMS);
    const long long xb = 4LL * np * mp, ab = 4LL * np * np;
    x[0] = 0; x[1] = xb; a = 2 * xb; b = a + ab; part = b + ab; bytes = (part + 8LL * sums + 255) & ~255LL;
  }
};

OPS_DEV const Mat& find(const Batch& B, int wg) {
  int i = 0;
  while (i + 1 < B.count && wg >= B.m[i + 1].first) ++i;
  return B.m[i];
}

// partial sums of squares in 64 bits: no overflow or underflow for any float32 U
template <typename T> __global__ __launch_bounds__(THREADS) void k_sumsq(const Batch B) {
  __shared__ double red[THREADS];
  const Mat& M = find(B, blockIdx.x);
  const Layout L(M.rows, M.cols);
  const int part = blockIdx.x - M.first;
  const long long count = (long long)M.rows * M.cols, e0 = (long long)part * SUM_ELEMS, e1 = e0 + SUM_ELEMS < count ? e0 + SUM_ELEMS : count;
  double s = 0.0;
  for (long long e = e0 + threadIdx.x; e < e1; e += THREADS) {
    const double v = to_f32<T>(static_cast<const T*>(M.u)[e / M.cols * M.ldu + e % M.cols]);
    s += v * v;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int d = THREADS / 2; d >= 1; d >>= 1) {
    if (threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) reinterpret_cast<double*>(B.ws + M.ws + L.part)[part] = red[0];
}

OPS_DEV void split2(float v, _Float16& hi, _Float16& lo) { hi = (_Float16)v; lo = (_Float16)(v - (float)hi); }

// X0's planes, one 64 x 64 tile per workgroup
template <typename T> __global__ __launch_bounds__(THREADS) void k_prepare(const Batch B) {
  __shared__ double red[THREADS];
  __shared__ float tile[TILE][TILE + 1];
  const Mat& M = find(B, blockIdx.x);
  const Layout L(M.rows, M.cols);
  const int t = blockIdx.x - M.first, i0 = t / (L.mp / TILE) * TILE, j0 = t % (L.mp / TILE) * TILE;
  const bool tall = M.rows > M.cols;
  double s = 0.0;
  for (int p = threadIdx.x; p < L.sums; p += THREADS) s += reinterpret_cast<const double*>(B.ws + M.ws + L.part)[p];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int d = THREADS / 2; d >= 1; d >>= 1) {
    if (threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
    __syncthreads();
  }
  const double inv = (double)SX / (red[0] > TINY * TINY || red[0] != red[0] ? sqrt(red[0]) : TINY);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // read along U's rows, write along X's
  for (int q = w; q < TILE; q += THREADS / 64) {
    const int r = tall ? j0 + q : i0 + q, c = tall ? i0 + lane : j0 + lane;
    const float v = r < M.rows && c < M.cols ? (float)(inv * (double)to_f32<T>(static_cast<const T*>(M.u)[r * M.ldu + c])) : 0.f;
    if (tall) tile[lane][q] = v; else tile[q][lane] = v;
  }
  __syncthreads();
  _Float16* x = reinterpret_cast<_Float16*>(B.ws + M.ws + L.x[0]);
  const long long plane = (long long)L.np * L.mp;
  for (int q = w; q < TILE; q += THREADS / 64) {
    _Float16 hi, lo;
    split2(tile[q][lane], hi, lo);
    const long long at = (long long)(i0 + q) * L.mp + j0 + lane;
    x[at] = hi;
    x[plane + at] = lo;
  }
}

OPS_DEV f32x16 mma16(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// LDS tiles [64][64] f16, 8 granules a row; "strided" (the contraction across the rows) is read transposed
template <bool CONT> OPS_DEV int tile_at(int row, int g) { return row * 128 + ((g ^ (CONT ? row & 7 : ((row >> 1) & 1) << 2)) << 4); }
template <bool CONT> OPS_DEV u32x4 tile_frag(const char* lds, int t, int ks) {
  const int lane = threadIdx.x & 63;
  if constexpr (CONT) return *reinterpret_cast<const u32x4*>(lds + tile_at<true>(32 * t + (lane & 31), 2 * ks + (lane >> 5)));
  else {
    const int i = lane & 15, row = 16 * ks + 8 * (lane >> 5) + (i >> 2), g = 4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + tile_at<false>(row, g) + (i & 1) * 8)));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + tile_at<false>(row + 4, g) + (i & 1) * 8)));
    return u32x4{a[0], a[1], b[0], b[1]};
  }
}

enum { GRAM = 0, POLY = 1, UPDATE = 2, UPDATE_OUT = 3 };

// One 64 x 64 tile of a product; GRAM and POLY are symmetric: tiles i <= j only, written twice
template <int STEP, typename T> __global__ __launch_bounds__(THREADS) void k_product(const Batch B, int cur) {
  __shared__ __attribute__((aligned(16))) char lds[4 * TILE * BK * 2];
  const Mat& M = find(B, blockIdx.x);
  const Layout L(M.rows, M.cols);
  int t = blockIdx.x - M.first, ti, tj;
  constexpr bool SYM = STEP == GRAM || STEP == POLY;
  if constexpr (SYM) {
    const int tn = L.np / TILE;
    ti = 0;
    while (t >= tn - ti) { t -= tn - ti; ++ti; }
    tj = ti + t;
  } else { ti = t / (L.mp / TILE); tj = t % (L.mp / TILE); }
  const int i0 = ti * TILE, j0 = tj * TILE;
  char* ws = B.ws + M.ws;
  const long long xplane = (long long)L.np * L.mp, aplane = (long long)L.np * L.np;
  _Float16* X = reinterpret_cast<_Float16*>(ws + L.x[cur]);
  _Float16* A = reinterpret_cast<_Float16*>(ws + L.a);
  _Float16* P = reinterpret_cast<_Float16*>(ws + L.b);
  const _Float16* lhs = STEP == GRAM ? X : STEP == POLY ? A : P;
  const _Float16* rhs = STEP == GRAM ? X : STEP == POLY ? A : X;
  const int ldl = STEP == GRAM ? L.mp : L.np, ldr = STEP == POLY ? L.np : L.mp, K = STEP == GRAM ? L.mp : L.np;
  const long long pl = STEP == GRAM ? xplane : aplane, pr = STEP == POLY ? aplane : xplane;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
  u32x4 rl[2][2], rr[2][2];
  auto fetch = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int idx = threadIdx.x + THREADS * q, row = idx / 8, g = idx % 8;
      const long long al = (long long)(i0 + row) * ldl + k + 8 * g;
      const long long ar = SYM ? (long long)(j0 + row) * ldr + k + 8 * g : (long long)(k + row) * ldr + j0 + 8 * g;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        rl[q][p] = *reinterpret_cast<const u32x4*>(lhs + p * pl + al);
        rr[q][p] = *reinterpret_cast<const u32x4*>(rhs + p * pr + ar);
      }
    }
  };
  f32x16 acc = {};
  fetch(0);
  for (int k = 0; k < K; k += BK) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int idx = threadIdx.x + THREADS * q, row = idx / 8, g = idx % 8;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        *reinterpret_cast<u32x4*>(lds + p * 8192 + tile_at<true>(row, g)) = rl[q][p];
        *reinterpret_cast<u32x4*>(lds + 16384 + p * 8192 + tile_at<SYM>(row, g)) = rr[q][p];
      }
    }
    __syncthreads();
    if (k + BK < K) fetch(k + BK);
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      const u32x4 lh = tile_frag<true>(lds, wi, ks), ll = tile_frag<true>(lds + 8192, wi, ks);
      const u32x4 rh = tile_frag<SYM>(lds + 16384, wj, ks), rlo = tile_frag<SYM>(lds + 24576, wj, ks);
      // (the right operand first: lane l then holds row l & 31 of the tile and 4 consecutive columns per register quad)
      acc = mma16(rlo, lh, acc);
      acc = mma16(rh, ll, acc);
      acc = mma16(rh, lh, acc);
    }
  }

  const int i = i0 + 32 * wi + (lane & 31);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int j = j0 + 32 * wj + 8 * q + 4 * (lane >> 5);
    float v[4];
    if constexpr (STEP == GRAM) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[4 * q + e] * (1.f / SX);                       // A 2^15
    } else {
      const _Float16* old = STEP == POLY ? A + (long long)i * L.np + j : X + (long long)i * L.mp + j;
      const long long plane = STEP == POLY ? aplane : xplane;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float o = (float)old[e] + (float)old[plane + e];
        if constexpr (STEP == POLY) v[e] = (CB * o + CC * (acc[4 * q + e] * (1.f / SX))) * (SB / SX);      // B 2^14
        else v[e] = CA * o + acc[4 * q + e] * (1.f / SB);                                                // X 2^15
      }
    }
    if constexpr (STEP == UPDATE_OUT) {
      const bool tall = M.rows > M.cols;
      T* o = static_cast<T*>(M.o);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i < L.n && j + e < L.m) o[tall ? (j + e) * M.ldo + i : i * M.ldo + j + e] = from_f32<T>(v[e] * (1.f / SX));
    } else {
      _Float16* out = STEP == GRAM ? A : STEP == POLY ? P : reinterpret_cast<_Float16*>(ws + L.x[cur ^ 1]);
      const int ld = SYM ? L.np : L.mp;
      const long long plane = SYM ? aplane : xplane;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        _Float16 hi, lo;
        split2(v[e], hi, lo);
        out[(long long)i * ld + j + e] = hi;
        out[plane + (long long)i * ld + j + e] = lo;
        if (SYM && ti != tj) {
          out[(long long)(j + e) * ld + i] = hi;
          out[plane + (long long)(j + e) * ld + i] = lo;
        }
      }
    }
  }
}

template <typename T> void run(hipStream_t st, const OrthoMat* mats, int count, int steps, char* ws) {
  for (int at = 0; at < count; at += MAX_BATCH) {
    Batch B{};
    B.count = std::min(MAX_BATCH, count - at);
    B.ws = ws;
    long long off = 0;
    for (int i = 0; i < B.count; ++i) {
      const OrthoMat& s = mats[at + i];
      B.m[i] = Mat{s.u, s.o, s.ldu, s.ldo, off, s.rows, s.cols, 0, 0};
      off += Layout(s.rows, s.cols).bytes;
    }
    ws += off;
    // workgroups of a launch: f(layout) per matrix
    auto spread = [&](auto f) {
      int total = 0;
      for (int i = 0; i < B.count; ++i) { B.m[i].first = total; total += f(Layout(B.m[i].rows, B.m[i].cols)); }
      return dim3((unsigned)total);
    };
    auto sums = [](const Layout& L) { return L.sums; };
    auto full = [](const Layout& L) { return (L.np / TILE) * (L.mp / TILE); };
    auto sym = [](const Layout& L) { const int t = L.np / TILE; return t * (t + 1) / 2; };
    const dim3 block(THREADS);
    dim3 grid = spread(sums);
    hipLaunchKernelGGL((k_sumsq<T>), grid, block, 0, st, B);
    grid = spread(full);
    hipLaunchKernelGGL((k_prepare<T>), grid, block, 0, st, B);
    for (int s = 0; s < steps; ++s) {
      grid = spread(sym);
      hipLaunchKernelGGL((k_product<GRAM, T>), grid, block, 0, st, B, s & 1);
      hipLaunchKernelGGL((k_product<POLY, T>), grid, block, 0, st, B, s & 1);
      grid = spread(full);
      if (s + 1 < steps) hipLaunchKernelGGL((k_product<UPDATE, T>), grid, block, 0, st, B, s & 1);
      else hipLaunchKernelGGL((k_product<UPDATE_OUT, T>), grid, block, 0, st, B, s & 1);
    }
  }
}

}  // namespace

size_t ortho_ws(const OrthoMat* mats, int count) {
  size_t b = 0;
  for (int i = 0; i < count; ++i) b += Layout(mats[i].rows, mats[i].cols).bytes;
  return b;
}
void orthogonalize(hipStream_t st, int dtype, const OrthoMat* mats, int count, int steps, void* ws) {
  if (dtype == F32) run<float>(st, mats, count, steps, static_cast<char*>(ws));
  else if (dtype == F16) run<f16_t>(st, mats, count, steps, static_cast<char*>(ws));
  else run<bf16_t>(st, mats, count, steps, static_cast<char*>(ws));
}

}  // namespace nerfds_ops
