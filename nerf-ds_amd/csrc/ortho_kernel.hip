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
// Measured: 256 x 256 and smaller, the 40 kernels of the field in float32: norm 9, preparation 15, then per step 9 + 8 + 12 us for the three products, each of which waits
// for memory once or twice, not for its arithmetic; three of 1024 x 4096 and one of 2000 x 2047 in bf16: 20, 40 and 112 + 62 + 176 (UPDATE: 126 GFLOP of products of planes,
// 716 TFLOP/s; GRAM waits for its longest contraction, 4096, in a single round of workgroups).
//
// Three ways through the same arithmetic, by size:
//   whole   short side <= 64, long side <= 384: ONE workgroup takes the matrix through all steps in LDS (64 x 64: one launch, against 17)
//   64      tiles of 64 x 64, one launch per product over all such matrices: bound by latency (a product of 256 x 256 is 10 - 16 workgroups of 4 steps)
//   128     tiles of 128 x 128, where the matrices have enough of them to fill the card: bound by the matrix pipe
// A list of up to 64 matrices rides in the kernel arguments of each launch, so a captured graph needs no other memory than the workspace.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>

#include "lds_attr.h"
#include "operators.h"
#include "operators_dev.h"

namespace nerfds_ops {

namespace {

constexpr int THREADS = 256, WAVES8 = 512, TILE = 64, MAX_BATCH = 64;      // threads of the norm and the preparation, of the products
constexpr unsigned CUS = 256;                           // of the card
constexpr int WHOLE_N = 64, WHOLE_M = 384;             // sides of a matrix that one workgroup takes whole
constexpr int SUM_ELEMS = 8192;                         // elements of U per workgroup of the norm, at the most
constexpr float CA = 3.4445f, CB = -4.7750f, CC = 2.0315f;
constexpr float SX = 32768.f, SB = 16384.f;             // plane scales of X and A; of B
constexpr double TINY = 1e-30;                          // |U| below this divides as this: a zero matrix gives zero

struct Mat {
  const void* u; void* o;
  long long ldu, ldo;
  long long ws;             // byte offset of its workspace
  int rows, cols;
};
struct Batch { char* ws; int tile; int first[MAX_BATCH]; Mat m[MAX_BATCH]; };      // first: the matrix's first workgroup in this launch (unused entries: INT_MAX)
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

// workspace of one matrix: planes of X and of its transpose, twice (read one, write the other), of A and B, and the partial sums of the norm
struct Layout {
  int n, m, np, mp;                    // short and long side, and rounded up to whole tiles
  int sum_rows, sum_cols, sums;        // rows of a partial sum, partial sums along a row, in all
  long long xbytes, a, b, part, bytes;
  __host__ __device__ long long x(int cur) const { return 2 * cur * xbytes; }              // [2][np][mp]
  __host__ __device__ long long xt(int cur) const { return (2 * cur + 1) * xbytes; }       // [2][mp][np]
  __host__ __device__ Layout(int rows, int cols, int tile) {
    n = rows < cols ? rows : cols; m = rows < cols ? cols : rows;
    np = (n + tile - 1) / tile * tile; mp = (m + tile - 1) / tile * tile;
    sum_cols = (cols + SUM_ELEMS - 1) / SUM_ELEMS;
    sum_rows = sum_cols > 1 || cols * 2 > SUM_ELEMS ? 1 : SUM_ELEMS / cols;
    sums = (rows + sum_rows - 1) / sum_rows * sum_cols;
    const long long ab = 4LL * np * np;
    xbytes = 4LL * np * mp; a = 4 * xbytes; b = a + ab; part = b + ab; bytes = (part + 8LL * sums + 255) & ~255LL;
  }
};

// the matrix of a workgroup: one lane per entry compares, so a list of 64 costs one load
struct Found { int i, local; };
OPS_DEV Found find(const Batch& B, int wg) {
  const int mine = B.first[threadIdx.x & 63];
  const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine <= wg)) - 1);
  return {i, wg - B.first[i]};
}

// the sum over the first 256 threads, in a fixed order; every thread gets it
OPS_DEV double tree_sum(double v, double* red) {
  __syncthreads();
  if (threadIdx.x < THREADS) red[threadIdx.x] = v;
  __syncthreads();
  for (int d = THREADS / 2; d >= 1; d >>= 1) {
    if (threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
    __syncthreads();
  }
  return red[0];
}

// Partial sum `part` of the squares, each element's in 64 bits: no overflow or underflow for any float32 U.  A part is whole rows (or, of a longer row,
// SUM_ELEMS columns), 4 elements per lane and step.  All ways through this file add in the same order - a matrix's result is the same bits
// whatever else is in the call.
template <typename T> OPS_DEV double sum_part(const Mat& M, const Layout& L, int part, double* red) {
  const int r0 = part / L.sum_cols * L.sum_rows, c0 = part % L.sum_cols * SUM_ELEMS;
  const int rows = min(L.sum_rows, M.rows - r0), cols = min(SUM_ELEMS, M.cols - c0), quads = (cols + 3) / 4;
  double s = 0.0;
#pragma unroll 4
  for (int e = threadIdx.x; e < rows * quads && threadIdx.x < THREADS; e += THREADS) {
    const int r = (unsigned)e / (unsigned)quads, c = (e - r * quads) * 4;
    const T* p = static_cast<const T*>(M.u) + (r0 + r) * M.ldu + c0 + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double v = c + j < cols ? to_f32<T>(p[j]) : 0.f;
      s = fma(v, v, s);
    }
  }
  return tree_sum(s, red);
}
// X0 = U * this
OPS_DEV double scale_of(const double* parts, int sums, double* red) {
  double s = 0.0;
  for (int p = threadIdx.x; p < sums && threadIdx.x < THREADS; p += THREADS) s += parts[p];
  s = tree_sum(s, red);
  return (double)SX / (s > TINY * TINY || s != s ? sqrt(s) : TINY);
}

template <typename T> __global__ __launch_bounds__(THREADS) void k_sumsq(const Batch B) {
  __shared__ double red[THREADS];
  const Found at = find(B, blockIdx.x);
  const Mat& M = B.m[at.i];
  const Layout L(M.rows, M.cols, B.tile);
  const double s = sum_part<T>(M, L, at.local, red);
  if (threadIdx.x == 0) reinterpret_cast<double*>(B.ws + M.ws + L.part)[at.local] = s;
}

// (v is pinned as a float32 first: an instruction that multiplies, adds and rounds to f16 in one would give other bits, and not in every kernel)
OPS_DEV void split2(float v, _Float16& hi, _Float16& lo) {
  asm("" : "+v"(v));
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

OPS_DEV _Float16 half_of(const u32x2& v, int e) { return __builtin_bit_cast(_Float16, (uint16_t)(v[e >> 1] >> (16 * (e & 1)))); }
OPS_DEV float f16_of(const u32x2& v, int e) { return (float)half_of(v, e); }
OPS_DEV void split4(const float (&v)[4], u32x2 (&out)[2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    _Float16 hi, lo;
    split2(v[e], hi, lo);
    const unsigned h = __builtin_bit_cast(uint16_t, hi), l = __builtin_bit_cast(uint16_t, lo);
    if (e & 1) { out[0][e >> 1] |= h << 16; out[1][e >> 1] |= l << 16; } else { out[0][e >> 1] = h; out[1][e >> 1] = l; }
  }
}

// X0's planes, one 64 x 64 tile per workgroup
template <typename T> __global__ __launch_bounds__(THREADS) void k_prepare(const Batch B) {
  __shared__ double red[THREADS];
  __shared__ float tile[TILE][TILE + 1];
  const Found at = find(B, blockIdx.x);
  const Mat& M = B.m[at.i];
  const Layout L(M.rows, M.cols, B.tile);
  const int t = at.local, i0 = t / (L.mp / TILE) * TILE, j0 = t % (L.mp / TILE) * TILE;
  const bool tall = M.rows > M.cols;
  const double inv = scale_of(reinterpret_cast<const double*>(B.ws + M.ws + L.part), L.sums, red);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // read along U's rows, write along X's
  for (int q = w; q < TILE; q += THREADS / 64) {
    const int r = tall ? j0 + q : i0 + q, c = tall ? i0 + lane : j0 + lane;
    const float v = r < M.rows && c < M.cols ? (float)(inv * (double)to_f32<T>(static_cast<const T*>(M.u)[r * M.ldu + c])) : 0.f;
    if (tall) tile[lane][q] = v; else tile[q][lane] = v;
  }
  __syncthreads();
  _Float16* x = reinterpret_cast<_Float16*>(B.ws + M.ws + L.x(0));
  _Float16* xt = reinterpret_cast<_Float16*>(B.ws + M.ws + L.xt(0));
  const long long plane = (long long)L.np * L.mp;
  // 8 elements of a row of X and of its transpose at a time (columns of 65 floats: 8 rows x 8 granules fall on all banks either way)
  for (int e = threadIdx.x; e < TILE * 8; e += THREADS) {
    const int q = e >> 3, g = 8 * (e & 7);
    const long long at[2] = {(long long)(i0 + q) * L.mp + j0 + g, (long long)(j0 + q) * L.np + i0 + g};
#pragma unroll
    for (int turned = 0; turned < 2; ++turned) {
      u32x4 plane_of[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = turned ? tile[g + 4 * h + k][q] : tile[q][g + 4 * h + k];
        u32x2 pack[2];
        split4(v, pack);
#pragma unroll
        for (int p = 0; p < 2; ++p) { plane_of[p][2 * h] = pack[p][0]; plane_of[p][2 * h + 1] = pack[p][1]; }
      }
      _Float16* out = (turned ? xt : x) + at[turned];
      *reinterpret_cast<u32x4*>(out) = plane_of[0];
      *reinterpret_cast<u32x4*>(out + plane) = plane_of[1];
    }
  }
}

// from the accumulators (products of scaled planes) and the old value, at its own scale, to the new one (fused by hand: the compiler's choice could differ
// between the kernels)
OPS_DEV float gram_of(float acc) { return acc * (1.f / SX); }                                                        // A 2^15
OPS_DEV float poly_of(float a, float acc) { return fmaf(CC, acc * (1.f / SX), CB * a) * (SB / SX); }                // B 2^14
OPS_DEV float update_of(float x, float acc) { return fmaf(CA, x, acc * (1.f / SB)); }                               // X 2^15

OPS_DEV f32x16 mma16(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// LDS tiles of f16: a row is one line's BK contraction steps.  Granules of 16 bytes are swizzled so that the rows one read touches together fall on different
// banks.  (Every product has the contraction along the rows of both operands - X X^T, A A^T = A A, B (X^T)^T - because X is kept beside its
// transpose: a transposed read of LDS makes the compiler wait for every DMA in flight.)
template <int ROWB> OPS_DEV int swizzle(int row) { return ROWB == 128 ? row >> 1 & 7 : row >> 2 & 3; }
template <int ROWB> OPS_DEV u32x4 tile_frag(const char* lds, int t, int ks) {
  const int lane = threadIdx.x & 63, row = 32 * t + (lane & 31), g = 2 * ks + (lane >> 5);
  return *reinterpret_cast<const u32x4*>(lds + row * ROWB + ((g ^ swizzle<ROWB>(row)) << 4));
}

enum { GRAM = 0, POLY = 1, UPDATE = 2, UPDATE_OUT = 3 };

extern __shared__ __attribute__((aligned(16))) char g_lds[];

// all but the newest N loads have arrived, and this wave's LDS reads too: past the barrier that follows, the stage they came from may be overwritten
template <int N> OPS_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// One TS x TS tile of a product; GRAM and POLY are symmetric: tiles i <= j only, written twice.  Operand tiles arrive by LDS-DMA, up to 128 KiB of them under way
// or in use (128-byte rows: a request then is a whole cache line, half as many as with rows of 64; updates of 1024-wide matrices 183 -> 173 us), one barrier a stage.
// 8 waves: four of (TS / 2) x (TS / 2) take the even, four the odd contraction steps of 16, and their sums are added - two waves per SIMD, so that one's LDS reads
// run under the other's MFMAs, without reading any fragment more often.
template <int TS, int COUNT_> struct Ring {
  static constexpr int BK = 64, PLANE = TS * BK * 2, STAGE = 4 * PLANE, COUNT = COUNT_, IPW = STAGE / 1024 / 8, EACH = IPW / 4;      // DMA instructions per wave: of a stage, of a plane
  // afterwards: the tile in float32, and its two planes transposed (rows padded against bank conflicts)
  static constexpr int ROWF = TS + 4, ROWT = TS + 8, OUTF = TS * ROWF * 4, OUTT = TS * ROWT * 2;
  static constexpr int LDS = COUNT * STAGE > OUTF + 2 * OUTT ? COUNT * STAGE : OUTF + 2 * OUTT;
  static_assert(IPW == 4 * EACH, "whole instructions per wave and plane");
};
template <int STEP, typename T, int TS, int COUNT> __global__ __launch_bounds__(WAVES8) void k_product(const Batch B, int cur) {
  typedef Ring<TS, COUNT> R;
  constexpr int BK = R::BK, W = TS / 64;      // 32 x 32 tiles per wave and side
  constexpr bool SYM = STEP == GRAM || STEP == POLY;
  constexpr int ROWB = BK * 2;
  const Found at = find(B, blockIdx.x);
  const Mat& M = B.m[at.i];
  const Layout L(M.rows, M.cols, TS);
  int t = at.local, ti, tj;
  if constexpr (SYM) {
    const int tn = L.np / TS;
    ti = 0;
    while (t >= tn - ti) { t -= tn - ti; ++ti; }
    tj = ti + t;
  } else {      // bands of 8 tile rows, down the band first, a stretch of them per XCD: the 32 tiles in flight there are 8 x 4 and share operands both ways
    t = (int)xcd_order(t, (L.np / TS) * (L.mp / TS));
    const int tn = L.np / TS, tm = L.mp / TS, band = t / (8 * tm), rows = min(8, tn - 8 * band), r = t - band * 8 * tm;
    ti = 8 * band + r % rows;
    tj = r / rows;
  }
  const int i0 = ti * TS, j0 = tj * TS;
  char* ws = B.ws + M.ws;
  const long long xplane = (long long)L.np * L.mp, aplane = (long long)L.np * L.np;
  _Float16* X = reinterpret_cast<_Float16*>(ws + L.x(cur));
  _Float16* A = reinterpret_cast<_Float16*>(ws + L.a);
  _Float16* P = reinterpret_cast<_Float16*>(ws + L.b);
  const _Float16* lhs = STEP == GRAM ? X : STEP == POLY ? A : P;
  const _Float16* rhs = STEP == GRAM ? X : STEP == POLY ? A : reinterpret_cast<_Float16*>(ws + L.xt(cur));
  const int K = STEP == GRAM ? L.mp : L.np;      // row length of both operands
  const long long pl = STEP == GRAM ? xplane : aplane, pr = STEP == POLY ? aplane : xplane;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave >> 1 & 1, wj = wave & 1, odd = wave >> 2;

  // DMA: instruction u of wave w fills bytes 1024 (w + 8 u) .. of each plane, planes in the order left hi, left lo, right hi, right lo
  const _Float16* src[2][R::EACH];
#pragma unroll
  for (int u = 0; u < R::EACH; ++u) {
    const int slot = (wave + 8 * u) * 64 + lane, row = slot / (ROWB / 16), g = (slot % (ROWB / 16)) ^ swizzle<ROWB>(row);
    src[0][u] = lhs + (long long)(i0 + row) * K + 8 * g;
    src[1][u] = rhs + (long long)(j0 + row) * K + 8 * g;
  }
  const int steps = K / BK;
  auto issue = [&](int s, int slot) __attribute__((always_inline)) {
    s = s < steps ? s : steps - 1;      // (past the end: the last one again, into a slot nobody reads any more, so that the waits can count)
#pragma unroll
    for (int u = 0; u < R::IPW; ++u) {
      const int plane = u / R::EACH, e = u % R::EACH;
      const _Float16* g = src[plane >> 1][e] + s * BK + (plane & 1 ? (plane >> 1 ? pr : pl) : 0);
      const int off = __builtin_amdgcn_readfirstlane(slot * R::STAGE + plane * R::PLANE + (wave + 8 * e) * 1024);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)(g_lds + off), 16, 0, 0);
    }
  };
  f32x16 acc[W][W] = {};
#pragma unroll
  for (int s = 0; s < R::COUNT - 1; ++s) issue(s, s);
  for (int s = 0; s < steps; ++s) {
    wait_loads<(R::COUNT - 2) * R::IPW>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue(s + R::COUNT - 1, (s + R::COUNT - 1) % R::COUNT);
    __builtin_amdgcn_sched_barrier(0);
    const char* st = g_lds + (s % R::COUNT) * R::STAGE;
#pragma unroll
    for (int half = 0; half < BK / 32; ++half) {
      const int ks = 2 * half + odd;
      u32x4 l[W][2], r[W][2];
#pragma unroll
      for (int a = 0; a < W; ++a)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          l[a][p] = tile_frag<ROWB>(st + p * R::PLANE, W * wi + a, ks);
          r[a][p] = tile_frag<ROWB>(st + (2 + p) * R::PLANE, W * wj + a, ks);
        }
      // (the right operand first: lane l then holds row l & 31 of the tile and 4 consecutive columns per register quad)
#pragma unroll
      for (int a = 0; a < W; ++a)
#pragma unroll
        for (int b = 0; b < W; ++b) {
          acc[a][b] = mma16(r[b][1], l[a][0], acc[a][b]);
          acc[a][b] = mma16(r[b][0], l[a][1], acc[a][b]);
          acc[a][b] = mma16(r[b][0], l[a][0], acc[a][b]);
        }
    }
  }
  wait_loads<0>();      // no DMA may be on its way into LDS that is no longer this workgroup's

  // The tile goes through LDS so that memory sees whole rows, of the result and of its transpose.  What the product is added to is asked for now.
  constexpr int GR = TS / 8, EACH = TS * GR / WAVES8;      // granules of a row, granules of a thread
  const _Float16* add = STEP == POLY ? A : X;
  const int ld = SYM ? L.np : L.mp;
  const long long plane = SYM ? aplane : xplane;
  // a wave takes 16 rows x 4 granules: 64 bytes of a row in memory, and 32 of a column in the transposed planes (2 waves' worth of banks)
  auto mine = [&](int u, int& r, int& c) __attribute__((always_inline)) {
    const int b = (threadIdx.x >> 6) + 8 * u;
    r = 16 * (b % (TS / 16)) + (lane >> 2);
    c = 8 * (4 * (b / (TS / 16)) + (lane & 3));
  };
  Gran<f16_t> old[EACH][2];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    int r, c;
    mine(u, r, c);
    const _Float16* at = add + (long long)(i0 + r) * ld + j0 + c;
    if constexpr (STEP != GRAM) { old[u][0].v = *reinterpret_cast<const u32x4*>(at); old[u][1].v = *reinterpret_cast<const u32x4*>(at + plane); }
  }
  // 1. float32, the even and the odd steps' sums
  float* tile = reinterpret_cast<float*>(g_lds);
  _Float16* turned = reinterpret_cast<_Float16*>(g_lds + R::OUTF);      // [2][TS][ROWT]
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    __syncthreads();
    if (odd == turn) {
#pragma unroll
      for (int a = 0; a < W; ++a)
#pragma unroll
        for (int b = 0; b < W; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4* at = reinterpret_cast<f32x4*>(tile + (32 * (W * wi + a) + (lane & 31)) * R::ROWF + 32 * (W * wj + b) + 8 * q + 4 * (lane >> 5));
            const f32x4 v = {acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
            *at = turn == 0 ? v : *at + v;
          }
    }
  }
  __syncthreads();
  // 2. 8 elements of a row per thread: with what the product is added to, out along the rows, and back into LDS across them
  _Float16* out = STEP == GRAM ? A : STEP == POLY ? P : reinterpret_cast<_Float16*>(ws + L.x(cur ^ 1));
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    int r, c;
    mine(u, r, c);
    const int i = i0 + r, j = j0 + c;
    if (SYM && W == 2 && ti == tj && r >= 64 && c < 64) continue;      // (the mirror image of the block above the diagonal: written in 3.)
    const long long at = (long long)i * ld + j;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = tile[r * R::ROWF + c + k], o = STEP == GRAM ? 0.f : gran_get<f16_t>(old[u][0], k) + gran_get<f16_t>(old[u][1], k);
      v[k] = STEP == GRAM ? gram_of(x) : STEP == POLY ? poly_of(o, x) : update_of(o, x);
    }
    if constexpr (STEP == UPDATE_OUT) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= 1.f / SX;
      if (M.rows <= M.cols) {
        if (i < L.n) gran_store<T>(static_cast<T*>(M.o) + i * M.ldo + j, gran_pack<T>(v), L.m - j);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) tile[r * R::ROWF + c + k] = v[k];
      }
    } else {
      u32x2 p[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float w[4] = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
        split4(w, p[h]);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        *reinterpret_cast<u32x4*>(out + s * plane + at) = u32x4{p[0][s][0], p[0][s][1], p[1][s][0], p[1][s][1]};
        _Float16* col = turned + s * (R::OUTT / 2) + c * R::ROWT + r;
#pragma unroll
        for (int k = 0; k < 8; ++k) col[k * R::ROWT] = half_of(p[k >> 2][s], k & 3);
      }
    }
  }
  // 3. the transpose: X's own, or the other half of a symmetric result (what lies below the diagonal's 64 x 64 blocks is a copy of what lies above, whatever
  // the tile: a product and its mirror image round differently, the cross terms come in the other order)
  const bool copy = !SYM || ti != tj;
  if (STEP == UPDATE_OUT ? M.rows > M.cols : copy || W == 2) {
    __syncthreads();
    _Float16* mirror = SYM ? out : reinterpret_cast<_Float16*>(ws + L.xt(cur ^ 1));
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int e = threadIdx.x + WAVES8 * u, c = e / GR, r = e % GR * 8;
      if constexpr (STEP == UPDATE_OUT) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tile[(r + k) * R::ROWF + c];
        if (j0 + c < L.m) gran_store<T>(static_cast<T*>(M.o) + (j0 + c) * M.ldo + i0 + r, gran_pack<T>(v), L.n - i0 - r);
      } else {
        if (!copy && !(c >= 64 && r < 64)) continue;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          *reinterpret_cast<u32x4*>(mirror + s * plane + (long long)(j0 + c) * L.np + i0 + r) = *reinterpret_cast<const u32x4*>(turned + s * (R::OUTT / 2) + c * R::ROWT + r);
      }
    }
  }
}

// A matrix of at most 64 x 384 (either way round) in one workgroup: X, A and B stay in LDS as planes, rows of 64 (A, B) and mp (X) elements.
// 45 matrices of this size in one launch are 45 workgroups side by side; the chain of 15 products costs barriers where the launches cost microseconds.
constexpr int WHOLE_LDS = 2 * 2 * WHOLE_N * WHOLE_M + 2 * 2 * 2 * WHOLE_N * WHOLE_N + 16 * 1024;
template <typename T> __global__ __launch_bounds__(WAVES8) void k_whole(const Batch B, int steps) {
  const Mat& M = B.m[blockIdx.x];
  const Layout L(M.rows, M.cols, TILE);
  const bool tall = M.rows > M.cols;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rowx = L.mp * 2, xplane = WHOLE_N * rowx;
  char* X = g_lds;                              // [2][64][mp]
  char* A = g_lds + 2 * xplane;
  char* P = A + 2 * 8192;
  f32x4* sums = reinterpret_cast<f32x4*>(P + 2 * 8192);      // [4 tiles][4 quads][64 lanes]: what two waves of a tile give each other
  // X is read along its rows (16 lines, one granule) and across them (4 rows, 4 granules, transposed): the swizzle sends both to the 16 granules that the banks
  // span, in rows of 128 bytes (modulo 256) and of 256
  auto turn8 = [](int r) __attribute__((always_inline)) { return (r << 1 & 4) | (r >> 2 & 3); };
  auto xat = [&](int r, int g) __attribute__((always_inline)) { return r * rowx + ((g ^ (rowx & 128 ? turn8(r) : (r << 2 & 12) | (r >> 2 & 3))) << 4); };
  auto aat = [&](int r, int g) __attribute__((always_inline)) { return r * 128 + ((g ^ turn8(r)) << 4); };

  double* red = reinterpret_cast<double*>(g_lds);
  double* parts = red + THREADS;
  for (int p = 0; p < L.sums; ++p) {
    const double s = sum_part<T>(M, L, p, red);
    if (threadIdx.x == 0) parts[p] = s;
  }
  __syncthreads();
  const double inv = scale_of(parts, L.sums, red);
  __syncthreads();
  // (along the rows of U: for a tall U that scatters 2-byte elements over LDS, once)
#pragma unroll 8
  for (int e = threadIdx.x; e < WHOLE_N * L.mp; e += WAVES8) {
    const int i = tall ? e % WHOLE_N : (unsigned)e / (unsigned)L.mp, j = tall ? e / WHOLE_N : (unsigned)e % (unsigned)L.mp, r = tall ? j : i, c = tall ? i : j;
    const float v = r < M.rows && c < M.cols ? (float)(inv * (double)to_f32<T>(static_cast<const T*>(M.u)[r * M.ldu + c])) : 0.f;
    _Float16 hi, lo;
    split2(v, hi, lo);
    const int at = xat(i, j >> 3) + (j & 7) * 2;
    *reinterpret_cast<_Float16*>(X + at) = hi;
    *reinterpret_cast<_Float16*>(X + xplane + at) = lo;
  }
  __syncthreads();

  // fragments: line 32 t + (l & 31), contraction steps 16 ks + 8 (l >> 5) ..
  auto along = [&](const char* base, auto place, int t, int ks) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(base + place(32 * t + (lane & 31), 2 * ks + (lane >> 5)));
  };
  auto across = [&](const char* base, int t, int ks) __attribute__((always_inline)) {
    const int i = lane & 15, row = 16 * ks + 8 * (lane >> 5) + (i >> 2), g = 4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(base + xat(row, g) + (i & 1) * 8)));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(base + xat(row + 4, g) + (i & 1) * 8)));
    return u32x4{a[0], a[1], b[0], b[1]};
  };
  // GRAM: A = X X^T; POLY: P = b A + c A A; UPDATE: X <- a X + P X (in place: X is read by all before it is written).  Waves (wi, wj) have the 32 x 32
  // tile (wi, wj), one the even and one the odd contraction steps of 16 as in k_product; each gives the other half of its sums and finishes the other half
  // (64 x 64, one call: 23 us; 29 where the odd wave finishes all and two waves of eight make the update).
  const int wi = wave >> 1 & 1, wj = wave & 1, odd = wave >> 2;
  f32x4* const box = sums + (wave & 3) * 256 + lane;
  for (int step = 0; step < steps; ++step) {
#pragma unroll
    for (int kind = GRAM; kind <= UPDATE; ++kind) {
      if (kind == UPDATE && L.mp > 64) break;
      f32x16 acc = {};
      const int K = kind == GRAM ? L.mp : WHOLE_N;
#pragma unroll 4
      for (int ks = odd; ks < K / 16; ks += 2) {
        u32x4 l[2], r[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          l[p] = kind == GRAM ? along(X + p * xplane, xat, wi, ks) : along((kind == POLY ? A : P) + p * 8192, aat, wi, ks);
          r[p] = kind == GRAM ? along(X + p * xplane, xat, wj, ks) : kind == POLY ? along(A + p * 8192, aat, wj, ks) : across(X + p * xplane, wj, ks);
        }
        acc = mma16(r[1], l[0], acc);
        acc = mma16(r[0], l[1], acc);
        acc = mma16(r[0], l[0], acc);
      }
      f32x4 own[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 low = {acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]}, high = {acc[4 * h + 8], acc[4 * h + 9], acc[4 * h + 10], acc[4 * h + 11]};
        own[h] = odd ? high : low;
        box[64 * (2 * (1 - odd) + h)] = odd ? low : high;
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = 2 * odd + h, row = 32 * wi + (lane & 31), col = 32 * wj + 8 * q + 4 * (lane >> 5);
        const f32x4 given = box[64 * q];
        const int at = (kind == UPDATE ? xat(row, col >> 3) : aat(row, col >> 3)) + 8 * (lane >> 5);
        char* const from = kind == UPDATE ? X : A;
        const int plane = kind == UPDATE ? xplane : 8192;
        u32x2 oh = {}, ol = {};
        if (kind != GRAM) { oh = *reinterpret_cast<const u32x2*>(from + at); ol = *reinterpret_cast<const u32x2*>(from + plane + at); }
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = given[e] + own[h][e], o = f16_of(oh, e) + f16_of(ol, e);
          v[e] = kind == GRAM ? gram_of(x) : kind == POLY ? poly_of(o, x) : update_of(o, x);
        }
        if (kind == UPDATE && step + 1 == steps) {
          T* o = static_cast<T*>(M.o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (row < L.n && col + e < L.m) o[tall ? (col + e) * M.ldo + row : row * M.ldo + col + e] = from_f32<T>(v[e] * (1.f / SX));
        } else {
          char* const out = kind == GRAM ? A : kind == POLY ? P : X;
          u32x2 pack[2];
          split4(v, pack);
          *reinterpret_cast<u32x2*>(out + at) = pack[0];
          *reinterpret_cast<u32x2*>(out + plane + at) = pack[1];
        }
      }
      __syncthreads();
    }
    if (L.mp == 64) continue;
    // UPDATE of a longer X: a wave takes 32 columns whole (both row tiles), reads them, and writes them back in place (64 x 384: 70 us; 81 by the way above, which
    // needs two barriers for each 64 columns)
    for (int t = wave; t < L.mp / 32; t += 8) {
      f32x16 acc[2][2] = {};      // [row tile][even, odd]
#pragma unroll
      for (int ks = 0; ks < WHOLE_N / 16; ++ks) {
        const u32x4 rh = across(X, t, ks), rl = across(X + xplane, t, ks);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u32x4 lh = along(P, aat, a, ks), ll = along(P + 8192, aat, a, ks);
          acc[a][ks & 1] = mma16(rl, lh, acc[a][ks & 1]);
          acc[a][ks & 1] = mma16(rh, ll, acc[a][ks & 1]);
          acc[a][ks & 1] = mma16(rh, lh, acc[a][ks & 1]);
        }
      }
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = 32 * a + (lane & 31), j = 32 * t + 8 * q + 4 * (lane >> 5), at = xat(i, 4 * t + q) + 8 * (lane >> 5);
          const u32x2 oh = *reinterpret_cast<const u32x2*>(X + at), ol = *reinterpret_cast<const u32x2*>(X + xplane + at);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = update_of(f16_of(oh, e) + f16_of(ol, e), acc[a][0][4 * q + e] + acc[a][1][4 * q + e]);
          if (step + 1 < steps) {
            u32x2 pack[2];
            split4(v, pack);
            *reinterpret_cast<u32x2*>(X + at) = pack[0];
            *reinterpret_cast<u32x2*>(X + xplane + at) = pack[1];
          } else {
            T* o = static_cast<T*>(M.o);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i < L.n && j + e < L.m) o[tall ? (j + e) * M.ldo + i : i * M.ldo + j + e] = from_f32<T>(v[e] * (1.f / SX));
          }
        }
    }
    __syncthreads();
  }
}

// How the matrices of a call are taken.  Whole if all of them are that small (next to larger ones, whose launches happen anyway, they go along in those:
// alone they would hold the others up).  Through 128 x 128 tiles those with a short side of 256 and more, if these tiles are at least two per CU of the card -
// an update then keeps it busy at the larger tile's rate -, else, and the shorter ones always, through 64 x 64 tiles, of which there are four times as many.
enum Way { WHOLE, TILES_64, TILES_128 };
struct Ways {
  bool whole = true, large;
  Ways(const OrthoMat* mats, int count) {
    long long tiles = 0;
    for (int i = 0; i < count; ++i) {
      const int n = std::min(mats[i].rows, mats[i].cols), m = std::max(mats[i].rows, mats[i].cols);
      whole = whole && n <= WHOLE_N && m <= WHOLE_M;
      if (n >= 256) tiles += ((n + 127) / 128) * (long long)((m + 127) / 128);
    }
    large = tiles >= 2 * CUS;
  }
  Way of(const OrthoMat& m) const { return whole ? WHOLE : large && std::min(m.rows, m.cols) >= 256 ? TILES_128 : TILES_64; }
};
Layout layout_of(const OrthoMat& m, Way w) { return Layout(m.rows, m.cols, w == TILES_128 ? 128 : TILE); }

template <int STEP, typename T, int TS, int COUNT> void product_of(hipStream_t st, dim3 grid, const Batch& B, int cur) {
  typedef Ring<TS, COUNT> R;
  nerfds::allow_dynamic_lds(reinterpret_cast<const void*>(&k_product<STEP, T, TS, COUNT>), R::LDS);
  hipLaunchKernelGGL((k_product<STEP, T, TS, COUNT>), grid, dim3(WAVES8), R::LDS, st, B, cur);
}
// 64 x 64 tiles: four stages of 32 KiB, or two where the launch has more workgroups than the card has CUs, so that two of them share one (20 matrices of
// 256 x 256: 148 us instead of 165; one of them 97 instead of 93, 768 x 3000 368 instead of 319).  128 x 128 tiles: two stages fill LDS as they are.
template <int STEP, typename T, int TS> void product(hipStream_t st, dim3 grid, const Batch& B, int cur) {
  if (TS == 128 || grid.x > CUS) product_of<STEP, T, TS, 2>(st, grid, B, cur); else product_of<STEP, T, TS, TS == 128 ? 2 : 4>(st, grid, B, cur);
}

template <typename T, int TS> void products(hipStream_t st, Batch& B, int count, int steps) {
  // workgroups of a launch: f(layout) per matrix
  auto spread = [&](auto f) {
    int total = 0;
    for (int i = 0; i < count; ++i) { B.first[i] = total; total += f(Layout(B.m[i].rows, B.m[i].cols, TS)); }
    return dim3((unsigned)total);
  };
  auto full = [](const Layout& L) { return (L.np / TS) * (L.mp / TS); };
  auto sym = [](const Layout& L) { const int t = L.np / TS; return t * (t + 1) / 2; };
  const dim3 block(THREADS);
  dim3 grid = spread([](const Layout& L) { return L.sums; });
  hipLaunchKernelGGL((k_sumsq<T>), grid, block, 0, st, B);
  grid = spread([](const Layout& L) { return (L.np / TILE) * (L.mp / TILE); });
  hipLaunchKernelGGL((k_prepare<T>), grid, block, 0, st, B);
  for (int s = 0; s < steps; ++s) {
    grid = spread(sym);
    product<GRAM, T, TS>(st, grid, B, s & 1);
    product<POLY, T, TS>(st, grid, B, s & 1);
    grid = spread(full);
    if (s + 1 < steps) product<UPDATE, T, TS>(st, grid, B, s & 1); else product<UPDATE_OUT, T, TS>(st, grid, B, s & 1);
  }
}

template <typename T> void run(hipStream_t st, const OrthoMat* mats, int count, int steps, char* ws) {
  const Ways ways(mats, count);
  // (the longest contractions first in each batch: what is left at a launch's end is then short)
  for (const Way way : {WHOLE, TILES_64, TILES_128}) {
    for (int at = 0; at < count;) {
      Batch B{};
      B.ws = ws;
      B.tile = way == TILES_128 ? 128 : TILE;
      std::fill(B.first, B.first + MAX_BATCH, INT_MAX);
      int n = 0;
      long long off = 0;
      for (; at < count && n < MAX_BATCH; ++at) {
        const OrthoMat& s = mats[at];
        if (ways.of(s) != way) continue;
        B.m[n++] = Mat{s.u, s.o, s.ldu, s.ldo, off, s.rows, s.cols};
        if (way != WHOLE) off += layout_of(s, way).bytes;
      }
      ws += off;
      if (n == 0) break;
      if (way != WHOLE) std::stable_sort(B.m, B.m + n, [](const Mat& a, const Mat& b) { return std::min(a.rows, a.cols) > std::min(b.rows, b.cols); });
      if (way == WHOLE) {
        nerfds::allow_dynamic_lds(reinterpret_cast<const void*>(&k_whole<T>), WHOLE_LDS);
        hipLaunchKernelGGL((k_whole<T>), dim3((unsigned)n), dim3(WAVES8), WHOLE_LDS, st, B, steps);
      } else if (way == TILES_64) products<T, 64>(st, B, n, steps);
      else products<T, 128>(st, B, n, steps);
    }
  }
}

}  // namespace

size_t ortho_ws(const OrthoMat* mats, int count) {
  const Ways ways(mats, count);
  size_t b = 0;
  for (int i = 0; i < count; ++i) {
    const Way w = ways.of(mats[i]);
    if (w != WHOLE) b += layout_of(mats[i], w).bytes;
  }
  return b;
}
void orthogonalize(hipStream_t st, int dtype, const OrthoMat* mats, int count, int steps, void* ws) {
  if (dtype == F32) run<float>(st, mats, count, steps, static_cast<char*>(ws));
  else if (dtype == F16) run<f16_t>(st, mats, count, steps, static_cast<char*>(ws));
  else run<bf16_t>(st, mats, count, steps, static_cast<char*>(ws));
}

}  // namespace nerfds_ops
