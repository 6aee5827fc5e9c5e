// y = act(x kernel + bias) + residual with its gradients, for any sizes, three element types.  The three matrix products are one tile kernel:
//   forward   y  [m x n] = x  [m x k] . kernel [k x n]       contraction over k
//   data      dx [m x k] = dz [m x n] . kernel^T             contraction over n
//   weights   dk [k x n] = x^T        . dz [m x n]           contraction over m, split over workgroups and summed in a second kernel
// dz = dy act'(z).  Each operand is stored with the contraction either along its rows ("contiguous") or across them ("strided"); a strided tile is
// transposed on its way from LDS to the registers (ds_read_b64_tr_b16), so no operand is ever transposed in memory.
// k_gemm below takes everything (a few rows' long contraction in pieces that k_join adds); dense_resident.h, dense_tile.h and dense_backward.h the 16-bit products that stream past a small kernel, that are large, and both
// gradients of a narrow layer.  65536 x 256 -> 256 in float32 with softplus: forward 71 us, dz 35, dx 59, the weight gradient 54 - 60 and its sum 7 (six products of
// parts each, 52 GFLOP: 46 us at the rate of a large 16-bit product, 720 - 960 TFLOP/s reached).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "lds_attr.h"
#include "operators.h"
#include "operators_dev.h"

namespace nerfds_ops {

namespace {

constexpr int BM = 128, BN = 128, THREADS = 256;

struct GemmArgs {
  const void* a; long long lda;       // contiguous: [M][C], strided: [C][M]
  const void* b; long long ldb;       // contiguous: [N][C], strided: [C][N]
  long long M, N, C;
  const unsigned char* mask; long long ldm;      // relu bits of the operand that is dz, or nullptr
  const void* bias; const void* residual; long long ldr;
  void* y; long long ldy;
  void* save; long long lds; int act;
  float* part; float* colpart; int splits; long long cps;      // weights: [splits][M][N], [splits][N], contraction per split (a multiple of BK)
  int tiles_n; long long tiles;
  long long lo;      // k_gemm: elements from dz to its second part, 0: it has one (data: operand a, weights: operand b)
  bool large;        // weights: k_tile takes it
  void* dbias;       // weights: the column sums of b, by the one split there is (with more: colpart)
};

template <typename T> struct Shape;
// float32 operands go to the matrix pipe as three bf16 parts (8 + 8 + 8 significand bits, cut off, so their sum IS the float) and six products: all
// those of 2^-16 and above.  What is dropped is below 2^-23 of a product - float32's own rounding - at 2.6 times the rate of the float32 MFMA.
template <> struct Shape<float> { static constexpr int BK = 32, P = 3; };
template <> struct Shape<f16_t> { static constexpr int BK = 64, P = 1; };
template <> struct Shape<bf16_t> { static constexpr int BK = 64, P = 1; };

OPS_DEV f32x16 mma(const u32x4& a, const u32x4& b, const f32x16& c, f16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T> OPS_DEV f32x16 mma(const u32x4& a, const u32x4& b, const f32x16& c, T) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 8 floats -> three planes of 8 bf16, each the upper half of what is left
OPS_DEV void split3(const f32x4 (&v)[2], u32x4 (&out)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = v[i >> 1][2 * (i & 1)], h = v[i >> 1][2 * (i & 1) + 1];      // (a bit cast of a vector ELEMENT reads element 0)
    unsigned a = __builtin_bit_cast(unsigned, f), b = __builtin_bit_cast(unsigned, h);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      out[p][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      if (p < 2) {
        a = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, a) - __builtin_bit_cast(float, a & 0xffff0000u));
        b = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, b) - __builtin_bit_cast(float, b & 0xffff0000u));
      }
    }
  }
}

// zero where the relu bit is 0
template <typename T> OPS_DEV void gran_mask(Gran<T>& g, unsigned bits) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (!(bits >> i & 1u)) g.v[i >> 2][i & 3] = 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) g.v[i] &= ((bits >> (2 * i) & 1u) ? 0xffffu : 0u) | ((bits >> (2 * i + 1) & 1u) ? 0xffff0000u : 0u);
  }
}

// One operand's tile: 128 lines of BK contraction steps.
//   contiguous: LDS row = line (BK elements), granule g of row r at g ^ sw(r): the 16 rows that are read together fall on all 16 granules' banks
//   strided:    LDS row = contraction step (128 elements), granule g of row r at g ^ ((r & 3) << 2), likewise for the 4 x 16 blocks of the transposed read
template <typename T, bool CONT> struct Tile {
  static constexpr int BK = Shape<T>::BK, P = Shape<T>::P, PLANE = 128 * BK * 2, BYTES = P * PLANE;
  static constexpr int NG = 128 * BK / 8 / THREADS;        // granules of a thread
  static OPS_DEV void place(int i, int& row, int& g) {
    const int idx = threadIdx.x + THREADS * i;
    if constexpr (CONT) { row = idx / (BK / 8); g = idx % (BK / 8); } else { row = idx / 16; g = idx % 16; }
  }
  static OPS_DEV int offset(int row, int g) {
    if constexpr (CONT) return row * (BK * 2) + ((g ^ (BK == 64 ? row >> 1 & 7 : row >> 2 & 3)) << 4);
    else return row * 256 + ((g ^ ((row & 3) << 2)) << 4);
  }
  // lines from `line`, contraction [c, c1)
  static OPS_DEV void load(Gran<T> (&r)[NG], const void* p, long long ld, long long line, long long lines, long long c, long long c1) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      int row, g;
      place(i, row, g);
      const long long rr = (CONT ? line : c) + row, cc = (CONT ? c : line) + 8 * g, rows = CONT ? lines : c1, cols = CONT ? c1 : lines;
      r[i] = gran_load<T>(static_cast<const T*>(p) + rr * ld + cc, rr < rows ? cols - cc : 0);
    }
  }
  static OPS_DEV void mask(Gran<T> (&r)[NG], const unsigned char* p, long long ld, long long line, long long lines, long long c, long long c1) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      int row, g;
      place(i, row, g);
      const long long rr = (CONT ? line : c) + row, cc = (CONT ? c : line) + 8 * g, rows = CONT ? lines : c1, cols = CONT ? c1 : lines;
      gran_mask<T>(r[i], rr < rows && cc < cols ? p[rr * ld + (cc >> 3)] : 0u);
    }
  }
  static OPS_DEV void stage(const Gran<T> (&r)[NG], char* lds) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      int row, g;
      place(i, row, g);
      char* at = lds + offset(row, g);
      if constexpr (P == 3) {
        u32x4 s[3];
        split3(r[i].v, s);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>(at + p * PLANE) = s[p];
      } else *reinterpret_cast<u32x4*>(at) = r[i].v;
    }
  }
  // the fragment of lines 32 t .. 32 t + 31, contraction steps 16 ks .. 16 ks + 15: lane l holds line l & 31, steps 8 (l >> 5) ..
  static OPS_DEV u32x4 frag(const char* lds, int plane, int t, int ks) {
    const int lane = threadIdx.x & 63;
    if constexpr (CONT) return *reinterpret_cast<const u32x4*>(lds + plane * PLANE + offset(32 * t + (lane & 31), 2 * ks + (lane >> 5)));
    else {
      // a 16-lane group reads the block [4 steps][16 lines]: lane i supplies the 8-byte piece (step i / 4, lines 4 (i % 4) ..) and receives line i
      const int i = lane & 15, row = 16 * ks + 8 * (lane >> 5) + (i >> 2), g = 4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
      const char* at = lds + plane * PLANE + offset(row, g) + (i & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 4 * 256));
      u32x4 f;
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
      return f;
    }
  }
};

// Activations on the hardware's exp2, log2 and reciprocal (1 ulp each).  For float32 results exp's argument carries the rounding of x log2(e) along, and
// log(1 + e) is e log(u) / (u - 1) with u = 1 + e rounded, which cancels the rounding of u: 2 - 3 ulp, where the library's expf and log1pf are 60
// instructions (33 of 103 us for 65536 x 256 outputs).  16-bit results need neither.  erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + p x), is Abramowitz &
// Stegun 7.1.26 (absolute error 1.5e-7), for 16-bit results; the library's erfcf is 100 instructions, 85 us of 33 million outputs.
template <typename T> OPS_DEV float exp_(float x) {
  const float t = x * 1.44269504f, e = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(T) == 2) return e;
  const float r = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -t));      // what t lost, in units of log2: log2(e) = 1.44269504 + 1.926e-8
  return fabsf(t) < 126.f ? fmaf(e * 0.69314718f, r, e) : e;
}
template <typename T> OPS_DEV float sigmoid_(float z) { return __builtin_amdgcn_rcpf(1.f + exp_<T>(-z)); }
template <typename T> OPS_DEV float log1p_exp_(float z) {      // log(1 + exp(z)), z <= 0
  const float e = exp_<T>(z), u = 1.f + e, d = u - 1.f, l = 0.69314718f * __builtin_amdgcn_logf(u);      // (v_log_f32: base 2)
  return d == 0.f ? e : l * e * __builtin_amdgcn_rcpf(d);
}
template <typename T> OPS_DEV float cdf_(float z) {            // of the normal distribution
  if constexpr (sizeof(T) == 4) return 0.5f * erfcf(-0.70710678f * z);      // (erfc: 1 + erf cancels for negative z)
  else {
    const float x = 0.70710678f * fabsf(z), t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
    const float q = 0.5f * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f)))) * exp_<T>(-x * x);
    return z < 0.f ? q : 1.f - q;
  }
}
template <typename T, int ACT> OPS_DEV float act_value(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;      // (NaN stays)
  if constexpr (ACT == ACT_SIGMOID) return sigmoid_<T>(z);
  if constexpr (ACT == ACT_SOFTPLUS) return fmaxf(z, 0.f) + log1p_exp_<T>(-fabsf(z));
  if constexpr (ACT == ACT_SILU) return z * sigmoid_<T>(z);
  if constexpr (ACT == ACT_GELU) return z * cdf_<T>(z);
  return z;
}
template <typename T, int ACT> OPS_DEV float act_slope(float z) {
  if constexpr (ACT == ACT_SIGMOID) { const float s = sigmoid_<T>(z); return s * (1.f - s); }
  if constexpr (ACT == ACT_SOFTPLUS) return sigmoid_<T>(z);
  if constexpr (ACT == ACT_SILU) { const float s = sigmoid_<T>(z); return s * (1.f + z * (1.f - s)); }
  if constexpr (ACT == ACT_GELU) return cdf_<T>(z) + z * exp_<T>(-0.5f * z * z) * 0.39894228f;
  return 1.f;
}
// The switch stands around 8 elements, and the loops that come here are not unrolled: a copy of every activation for every element of a tile is
// 150 KB of code that a wave jumps through, and the tile then waits for its instructions (524288 x 256 x 256 through k_gemm: 382 us instead of 250).
template <typename T> OPS_DEV void act_values(float (&v)[8], int act) {
  switch (act) {
#define CASE(A) case A: _Pragma("unroll") for (int j = 0; j < 8; ++j) v[j] = act_value<T, A>(v[j]); break;
    CASE(ACT_RELU) CASE(ACT_SIGMOID) CASE(ACT_SOFTPLUS) CASE(ACT_SILU) CASE(ACT_GELU)
#undef CASE
    default: break;
  }
}
template <typename T> OPS_DEV void act_slopes(float (&v)[8], int act) {
  switch (act) {
#define CASE(A) case A: _Pragma("unroll") for (int j = 0; j < 8; ++j) v[j] = act_slope<T, A>(v[j]); break;
    CASE(ACT_SIGMOID) CASE(ACT_SOFTPLUS) CASE(ACT_SILU) CASE(ACT_GELU)
#undef CASE
    default: break;
  }
}

// bit j: v[j] > 0 (one compare and one add with carry each)
OPS_DEV unsigned relu_bits(const float (&v)[8]) {
  unsigned bits = 0;
#pragma unroll
  for (int j = 7; j >= 0; --j) bits = bits + bits + (v[j] > 0.f ? 1u : 0u);
  return bits;
}

// The end of the forward for 8 elements of row m, columns n ..: what the backward needs, activation, residual, the one rounding
template <typename T> OPS_DEV void finish(float (&v)[8], long long m, long long n, long long valid, int act, void* save, long long lds, const void* residual, long long ldr, void* y,
                                          long long ldy) {
  if (save != nullptr) {
    if (act == ACT_RELU) {
      static_cast<unsigned char*>(save)[m * lds + (n >> 3)] = (unsigned char)relu_bits(v);
    } else if (act != ACT_NONE) gran_store<T>(static_cast<T*>(save) + m * lds + n, gran_pack<T>(v), valid);
  }
  act_values<T>(v, act);
  if (residual != nullptr) {
    const Gran<T> g = gran_load<T>(static_cast<const T*>(residual) + m * ldr + n, valid);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += gran_get<T>(g, j);
  }
  gran_store<T>(static_cast<T*>(y) + m * ldy + n, gran_pack<T>(v), valid);
}

enum { OUT_FORWARD = 0, OUT_PLAIN = 1, OUT_WEIGHTS = 2 };      // weights: partial sums of a split (part), or the result (y) where one split does it

template <typename T, bool AC, bool BC, int OUT, int MASK /* 0, or the operand (1 = a, 2 = b) the relu bits belong to */>
__global__ __launch_bounds__(THREADS, 2) void k_gemm(const GemmArgs G) {
  typedef Tile<T, AC> TA;
  typedef Tile<T, BC> TB;
  constexpr int BK = Shape<T>::BK, P = Shape<T>::P;
  constexpr int STAGE = TA::BYTES + TB::BYTES, EPI = 4 * 32 * 68 * 4;
  __shared__ __attribute__((aligned(16))) char lds[STAGE > EPI ? STAGE : EPI];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const long long order = xcd_order(blockIdx.x, G.tiles);
  const long long m0 = order / G.tiles_n * BM, n0 = order % G.tiles_n * BN;
  const long long c0 = blockIdx.y * G.cps, c1 = c0 + G.cps < G.C ? c0 + G.cps : G.C;

  f32x16 acc[2][2] = {};
  Gran<T> ra[TA::NG], rb[TB::NG];
  float cs[8] = {};
  const bool sums = OUT == OUT_WEIGHTS && (G.colpart != nullptr || G.dbias != nullptr) && m0 == 0;
  const T* pa = static_cast<const T*>(G.a);
  const T* pb = static_cast<const T*>(G.b);
  bool more = OUT != OUT_FORWARD && !MASK && sizeof(T) == 2 && G.lo != 0;
  auto fetch = [&](long long c) __attribute__((always_inline)) {
    TA::load(ra, pa, G.lda, m0, G.M, c, c1);
    TB::load(rb, pb, G.ldb, n0, G.N, c, c1);
    if constexpr (MASK == 1) TA::mask(ra, G.mask, G.ldm, m0, G.M, c, c1);
    if constexpr (MASK == 2) TB::mask(rb, G.mask, G.ldm, n0, G.N, c, c1);
  };
  fetch(c0);
  for (long long c = c0; c < c1;) {
    __syncthreads();
    TA::stage(ra, lds);
    TB::stage(rb, lds + TA::BYTES);
    if constexpr (OUT == OUT_WEIGHTS) {
      if (sums) {
#pragma unroll
        for (int i = 0; i < TB::NG; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) cs[j] += gran_get<T>(rb[i], j);
      }
    }
    __syncthreads();
    c += BK;
    if (c >= c1 && more) {      // the whole contraction again with the second part of dz
      more = false;
      c = c0;
      (OUT == OUT_WEIGHTS ? pb : pa) += G.lo;
    }
    if (c < c1) fetch(c);
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      u32x4 fa[2][P], fb[2][P];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) { fa[i][p] = TA::frag(lds, p, 2 * wm + i, ks); fb[i][p] = TB::frag(lds + TA::BYTES, p, 2 * wn + i, ks); }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (P == 3) {      // smallest first
            acc[i][j] = mma(fa[i][2], fb[j][0], acc[i][j], T{});
            acc[i][j] = mma(fa[i][0], fb[j][2], acc[i][j], T{});
            acc[i][j] = mma(fa[i][1], fb[j][1], acc[i][j], T{});
            acc[i][j] = mma(fa[i][1], fb[j][0], acc[i][j], T{});
            acc[i][j] = mma(fa[i][0], fb[j][1], acc[i][j], T{});
          }
          acc[i][j] = mma(fa[i][0], fb[j][0], acc[i][j], T{});
        }
    }
  }

  if (G.part != nullptr) {
    float* out = G.part + blockIdx.y * ((G.M * G.N + 3) & ~3LL);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const long long n = n0 + 64 * wn + 32 * j + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const long long m = m0 + 64 * wm + 32 * i + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
          if (m < G.M && n < G.N) out[m * G.N + n] = acc[i][j][r];
        }
      }
  }
  if constexpr (OUT == OUT_WEIGHTS) {
    if (sums) {      // thread t holds the sums of columns 8 (t & 15) .. over its rows: 16 threads per column group
      float* red = reinterpret_cast<float*>(lds);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) red[(threadIdx.x >> 4) * 128 + 8 * (threadIdx.x & 15) + j] = cs[j];
      __syncthreads();
      if (threadIdx.x < 128 && n0 + threadIdx.x < G.N) {
        float s = 0.f;
        for (int q = 0; q < 16; ++q) s += red[q * 128 + threadIdx.x];
        if (G.dbias != nullptr) static_cast<T*>(G.dbias)[n0 + threadIdx.x] = from_f32<T>(s);
        else G.colpart[blockIdx.y * ((G.N + 3) & ~3LL) + n0 + threadIdx.x] = s;
      }
    }
  }
  if (G.part == nullptr && (OUT != OUT_WEIGHTS || G.y != nullptr)) {
    // the wave's 64 x 64 block through LDS, 32 rows at a time, so that every lane finishes 8 consecutive elements of a row
    float* buf = reinterpret_cast<float*>(lds) + wave * 32 * 68;
    const long long n = n0 + 64 * wn + 8 * (lane & 7), valid = G.N - n;
    float bias[8] = {};
    if (OUT == OUT_FORWARD && G.bias != nullptr && valid > 0) {
      const Gran<T> g = gran_load<T>(static_cast<const T*>(G.bias) + n, valid);
#pragma unroll
      for (int j = 0; j < 8; ++j) bias[j] = gran_get<T>(g, j);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) buf[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * 68 + 32 * j + (lane & 31)] = acc[i][j][r];
      __syncthreads();
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        const int row = 8 * q + (lane >> 3);
        const long long m = m0 + 64 * wm + 32 * i + row;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = buf[row * 68 + 8 * (lane & 7) + j];
        if (m >= G.M || valid <= 0) continue;
        if constexpr (OUT == OUT_FORWARD) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += bias[j];
          finish<T>(v, m, n, valid, G.act, G.save, G.lds, G.residual, G.ldr, G.y, G.ldy);
        } else gran_store<T>(static_cast<T*>(G.y) + m * G.ldy + n, gran_pack<T>(v), valid);
      }
    }
  }
}

// The end of a product whose contraction was split: a thread adds the parts of 8 elements in their order
template <typename T, int OUT> __global__ __launch_bounds__(256) void k_join(const GemmArgs G) {
  const long long gn = (G.N + 7) / 8, stride = (G.M * G.N + 3) & ~3LL, i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= G.M * gn) return;
  const long long m = i / gn, n = i % gn * 8, valid = G.N - n;
  float v[8] = {};
#pragma unroll 4
  for (int p = 0; p < G.splits; ++p) {
    const Gran<float> g = gran_load<float>(G.part + p * stride + m * G.N + n, valid);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += gran_get<float>(g, j);
  }
  if constexpr (OUT == OUT_FORWARD) {
    if (G.bias != nullptr) {
      const Gran<T> g = gran_load<T>(static_cast<const T*>(G.bias) + n, valid);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += gran_get<T>(g, j);
    }
    finish<T>(v, m, n, valid, G.act, G.save, G.lds, G.residual, G.ldr, G.y, G.ldy);
  } else gran_store<T>(static_cast<T*>(G.y) + m * G.ldy + n, gran_pack<T>(v), valid);
}

#include "dense_tile.h"
#include "dense_resident.h"
#include "dense_backward.h"

// The forward of a few rows (m <= 8: one frame's embedding, one token): bound by reading the kernel once, so by how many loads are in flight.  A workgroup
// takes 32 columns - a cache line's worth of every kernel row - and all of k: thread (slice, granule) multiplies 8 rows of 8 columns at a time, and
// the 64 slices are added over shuffles and LDS.  float32 multiply-adds: the matrix pipe would run 32-row tiles with 31 of them empty
// (1 x 1024 x 1024 in bf16: 5.8 us with gelu against 29 us through the tile kernel, whose 16 steps each wait for memory; the 2 MB alone would take 0.4).
template <typename T, int M> __global__ __launch_bounds__(256) void k_rows(const DenseFwd A) {
  __shared__ float red[4][M][32];
  const int g = threadIdx.x & 3, slice = threadIdx.x >> 2;
  const long long n = blockIdx.x * 32LL + 8 * g, valid = A.n - n;
  float acc[M][8] = {};
  for (int k = slice * 8; k < A.k; k += 512) {
    Gran<T> x[M], w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) w[r] = gran_load<T>(static_cast<const T*>(A.kernel) + (k + r) * A.ldk + n, k + r < A.k ? valid : 0);
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = gran_load<T>(static_cast<const T*>(A.x) + m * A.ldx + k, m < A.m ? A.k - k : 0);
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m) acc[m][j] = fmaf(gran_get<T>(x[m], r), gran_get<T>(w[r], j), acc[m][j]);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = acc[m][j];
#pragma unroll
      for (int d = 4; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
      if ((threadIdx.x & 63) < 4) red[threadIdx.x >> 6][m][8 * g + j] = v;
    }
  __syncthreads();
  const int m = threadIdx.x >> 2;
  if (m >= M || m >= A.m || valid <= 0) return;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = red[0][m][8 * g + j] + red[1][m][8 * g + j] + red[2][m][8 * g + j] + red[3][m][8 * g + j];
  if (A.bias != nullptr) {
    const Gran<T> b = gran_load<T>(static_cast<const T*>(A.bias) + n, valid);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += gran_get<T>(b, j);
  }
  finish<T>(v, m, n, valid, A.act, A.save, A.act == ACT_RELU ? (A.n + 7) / 8 : A.n, A.residual, A.ldr, A.y, A.ldy);
}

// dz = dy act'(z), once, for the activations whose slope costs more than a bit test (the products below read dz once per tile of their other axis), and for relu
// (z: its bits) where those tiles are many.  dz is rounded to the tensors' type: the matrix pipe takes it in no other.  Small layers (two_parts) get what
// that rounding lost as a second array lo elements on.
template <typename T, bool RELU> __global__ __launch_bounds__(256) void k_dz(const T* __restrict__ dy, long long lddy, const void* __restrict__ z, T* __restrict__ dz, long long m, int n, int act, long long lo) {
  const int gn = (n + 7) / 8;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < m * gn; i += gridDim.x * 256LL) {
    const long long row = i / gn;
    const int c = (int)(i % gn) * 8;
    Gran<T> a = gran_load<T>(dy + row * lddy + c, n - c);
    if constexpr (RELU) gran_mask<T>(a, static_cast<const unsigned char*>(z)[i]);
    else {
      const Gran<T> b = gran_load<T>(static_cast<const T*>(z) + row * n + c, n - c);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = gran_get<T>(b, j);
      act_slopes<T>(v, act);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= gran_get<T>(a, j);
      a = gran_pack<T>(v);
      if (lo != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float high = gran_get<T>(a, j);
          v[j] = fabsf(high) < __builtin_huge_valf() ? v[j] - high : 0.f;
        }
        gran_store<T>(dz + lo + row * n + c, gran_pack<T>(v), n - c);
      }
    }
    gran_store<T>(dz + row * n + c, a, n - c);
  }
}

long long up(long long a, long long b) { return (a + b - 1) / b; }
size_t aligned(size_t b) { return (b + 255) & ~(size_t)255; }

bool whole_granules(const void* p, long long ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }
// Whether dz is written to the workspace before the products.  Relu: where they run on large tiles, of which every column (k / 256) tests the bits of the same
// dy again (8192 x 2048 -> 4096: 170 + 207 us for dx and dkernel, and 20 + 132 + 151 with a stored dz; at k = 512 the two ways cost the same).
bool stores_dz(const DenseBwd& w) {
  if (w.act == ACT_NONE || w.act == ACT_RELU) return w.act == ACT_RELU && w.dtype != F32 && w.k > (w.dx && w.dkernel ? 512 : 1024) && w.k % 8 == 0 && w.n % 8 == 0 && whole_granules(w.x, w.ldx);
  return true;
}
// Whether dz keeps its float32 value in two parts, which the products take one after the other: 16-bit layers so small that their time is latency, where the
// rounding of dz would be the larger half of the gradients' error (45% more than the rounding of the results alone, and for the few results of a
// narrow layer by chance more) and costs 1.5 us (k_both, 64 x 64 at 4096 rows: 12.1 instead of 11.0) to 5 (256 x 256 at 1024 rows: 24 instead of 19) to avoid.
bool two_parts(const DenseBwd& w) { return w.dtype != F32 && w.act != ACT_NONE && w.act != ACT_RELU && w.m <= (1 << 18) / w.n; }
// Whether the operands of the weight gradient suit the tiles that come by DMA: whole, aligned granules, relu bits in whole dwords (a dz in the workspace is)
bool weight_dma(const DenseBwd& w) {
  if (w.dtype == F32 || w.k % 8 || w.n % 8 || !whole_granules(w.x, w.ldx)) return false;
  if (stores_dz(w)) return true;
  return whole_granules(w.dy, w.lddy) && (w.act != ACT_RELU || (w.n % 32 == 0 && reinterpret_cast<uintptr_t>(w.save) % 4 == 0));
}
// Whether the weight gradient takes the large tiles: from 2^34 multiply-adds on, or where the rows are so many that memory is the bound.  (k_gemm has more
// workgroups in flight, k_tile the higher rate: 512 x 512 in bf16 at 32768 rows 41 us by k_gemm and 44 by k_tile, at 65536 rows 68 and 60; 1024 x 1024 at 8192
// rows 38 and 42, at 32768 rows 106 and 91; 256 x 256 at 4096 rows 13 and 21)
bool weight_tiles_large(const DenseBwd& w) { return weight_dma(w) && !two_parts(w) && (w.m >= 131072 || w.m >= (1LL << 34) / ((long long)w.k * w.n)); }

// Whether both gradients come from one pass (k_both): a narrow layer in 16 bits, both wanted.  Up to 128 x 256 at any number of rows (128 x 128 in bf16: 9.7 us
// instead of 6.1 + 8.5 at 512 rows, 20.5 instead of 11 + 21 at 65536), the larger ones where their parts of dkernel have rows enough behind them (256 x 256: 32
// instead of 8.5 + 17 at 8192 rows, 40 instead of 15 + 24 at 32768, 47 instead of 23 + 33 at 65536, 213 instead of 119 + 130 at 524288).
bool both_at_once(const DenseBwd& w) {
  return w.dx != nullptr && w.dkernel != nullptr && w.k <= 256 && w.n <= 256 && ((w.k <= 128 || w.n <= 128) || (w.m >= 32768 && !two_parts(w))) && weight_dma(w);
}

// Whether k_both makes dz itself, from dy and z in LDS, instead of reading what k_dz wrote (524288 x 256 x 256 in bf16: 250 us instead of 331 with softplus, 297 instead
// of 345 with gelu, whose erf is the bound then; 8192 x 128 x 128: 15 instead of 17)
bool slopes_in_both(const DenseBwd& w) {
  return w.act != ACT_NONE && w.act != ACT_RELU && both_at_once(w) && !two_parts(w) && whole_granules(w.dy, w.lddy) && whole_granules(w.save, w.n);
}

constexpr int RESIDENT_M = 16384;
// The large tiles pay where they fill the card; with fewer the 128 x 128 tiles of k_gemm spread the work over more CUs
bool large_tiles_fill(long long m, long long n, int num_cus) { return up(m, 256) * up(n, 128) >= num_cus / 2; }

struct Splits { int count; long long cps; };
// The weight gradient has few output tiles (1 for 256 x 256) and a long contraction: as many splits as fill the card - one workgroup per CU of the large tiles,
// two of the small ones.  A fraction of a round more is no gain: splits are rounded down there.  Few rows are cut short too, for each split is one chain of loads
// and products: into 64 rows while all parts together stay under 8 MB, else 128 (256 x 256 in float32 at 512 rows: 11 us with 64, 15 with 128, 22 with 256; in
// bf16 at 4096 rows, where 64 would make 16 MB: 25, 23 and 26).  k_both, which makes dx too, takes 64 (8192 rows in bf16: 37 us with 32, 32 with 64, 33 with 128).
Splits weight_splits(const DenseBwd& w, int num_cus) {
  const long long steps = up(w.m, 64);
  if (both_at_once(w)) return {(int)(steps < num_cus ? steps : num_cus), 0};
  const bool large = weight_tiles_large(w);
  const long long tiles = large ? up(w.k, 256) * up(w.n, w.n > 128 ? 256 : 128) : up(w.k, BM) * up(w.n, BN), slots = large ? num_cus : 2LL * num_cus;
  long long want = tiles >= slots ? 1 : slots / tiles;
  const long long most = steps <= (2 << 20) / ((long long)w.k * w.n) ? steps : up(steps, 2);
  if (want > most) want = most;
  const long long cps = up(steps, want) * 64;
  return {(int)up(w.m, cps), cps};
}

// Few output tiles over a long contraction (few rows): the forward's and dx's products by k_gemm are split as well and joined by k_join, where the chain of steps
// they save (a step of 64 elements takes about 1.1 us in 16 bits, 4 in float32, whatever else runs) is longer than the join, which grows with the tiles.  Pieces are
// two steps and more, all parts within 32 MB.  Whole and split: 9 x 4096 -> 64 in bf16 130 and 14 us, in float32 295 and 19; 512 x 2048 -> 2048 (64 tiles) in bf16 36 and
// 22, but from k = 768 19 and 21; in float32 118 and 39, from k = 256 26 and 21.
Splits row_splits(int dtype, long long m, long long n, long long c, int num_cus) {
  const long long step = dtype == F32 ? 32 : 64, tiles = up(m, BM) * up(n, BN);
  if (m <= 8 || tiles >= num_cus || c < (dtype == F32 ? 128 + 2 * tiles : 256 + 12 * tiles)) return {1, c};
  if (dtype != F32 && (m >= RESIDENT_M || large_tiles_fill(m, n, num_cus))) return {1, c};      // (other kernels' work, whole)
  long long want = 2LL * num_cus / tiles;
  if (want > (1 << 23) / (m * n)) want = (1 << 23) / (m * n);
  if (want > c / (2 * step)) want = c / (2 * step);
  if (want <= 1) return {1, c};
  const long long cps = up(c, want * step) * step;
  return {(int)up(c, cps), cps};
}
size_t row_part_bytes(const Splits& s, long long m, long long n) { return s.count > 1 ? aligned((size_t)s.count * up(m * n, 4) * 16) : 0; }

size_t dz_bytes(const DenseBwd& w) { return stores_dz(w) && !slopes_in_both(w) ? aligned((size_t)up(w.m * w.n, 8) * 8 * dtype_bytes(w.dtype) * (two_parts(w) ? 2 : 1)) : 0; }
size_t weight_part_bytes(const DenseBwd& w, int splits) {      // (one split of the weight gradient alone writes the result itself)
  return splits > 1 || both_at_once(w) ? aligned((size_t)splits * up((long long)w.k * w.n, 4) * 16) : 0;
}

// Whether k_tile can take the product: rows of whole, aligned granules on both sides (M, N and C too where they run along rows), relu bits in whole dwords
template <bool AC, bool BC, int MASK> bool tile_fits(const GemmArgs& G) {
  return G.lo == 0 && whole_granules(G.a, G.lda) && whole_granules(G.b, G.ldb) && G.N % 8 == 0 && ((!AC && !BC) || G.C % 8 == 0) && (AC || G.M % 8 == 0) &&
         (!MASK || (G.ldm % 4 == 0 && reinterpret_cast<uintptr_t>(G.mask) % 4 == 0));
}
template <typename T, typename GR, bool AC, bool BC, int OUT, int MASK, int ACT = ACT_NONE> void launch_tile(hipStream_t st, GemmArgs& G, int num_cus) {
  if constexpr (OUT == OUT_FORWARD && ACT + 1 < ACT_COUNT) {
    if (G.act != ACT) { launch_tile<T, GR, AC, BC, OUT, MASK, ACT + 1>(st, G, num_cus); return; }
  }
  auto kern = k_tile<T, GR, AC, BC, OUT, MASK, ACT>;
  constexpr int lds = GR::RING * (GR::BM * 64 + GR::BN * 64 + (MASK == 1 ? GR::BM * 4 : MASK == 2 ? GR::BN * 4 : 0)), slots_per_cu = 8 / GR::WAVES;
  nerfds::allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds);
  G.tiles_n = (int)up(G.N, GR::BN);
  G.tiles = up(G.M, GR::BM) * G.tiles_n;
  const long long items = G.tiles * G.splits;
  const long long slots = (long long)num_cus * slots_per_cu;
  hipLaunchKernelGGL(kern, dim3((unsigned)(items < slots ? items : slots)), dim3(64 * GR::WAVES), lds, st, G);
}

constexpr int LDS_BYTES = 160 * 1024, RESIDENT_N = 256;
template <typename T, bool BC, int NP, int OUT, bool MASK, int ACT = ACT_NONE> void launch_resident(hipStream_t st, GemmArgs& G, int num_cus) {
  if constexpr (OUT == OUT_FORWARD && ACT + 1 < ACT_COUNT) {
    if (G.act != ACT) { launch_resident<T, BC, NP, OUT, MASK, ACT + 1>(st, G, num_cus); return; }
  }
  auto kern = k_resident<T, BC, NP, OUT, MASK, ACT>;
  nerfds::allow_dynamic_lds(reinterpret_cast<const void*>(kern), LDS_BYTES);
  const long long want = up(G.M, 128);
  hipLaunchKernelGGL(kern, dim3((unsigned)(want < num_cus ? want : num_cus)), dim3(512), Resident::bytes((int)G.N, (int)G.C + (G.bias != nullptr)), st, G);
}

template <typename T, bool AC, bool BC, int OUT, int MASK> void launch(hipStream_t st, GemmArgs& G, int num_cus) {
  if constexpr (sizeof(T) == 2 && AC && OUT != OUT_WEIGHTS && MASK < 2) {
    // Many rows past a kernel that fits LDS.  RESIDENT_M: every workgroup fills 128 KiB of LDS first (3 us), which wants some 100 rows behind it
    if (G.lo == 0 && G.M >= RESIDENT_M && G.N <= RESIDENT_N && G.C <= 4096 && Resident::bytes((int)G.N, (int)G.C + (G.bias != nullptr)) <= LDS_BYTES) {
      if (G.N <= 64) launch_resident<T, BC, 2, OUT, MASK == 1>(st, G, num_cus);
      else if (G.N <= 128) launch_resident<T, BC, 4, OUT, MASK == 1>(st, G, num_cus);
      else launch_resident<T, BC, 8, OUT, MASK == 1>(st, G, num_cus);
      return;
    }
  }
  if constexpr (sizeof(T) == 2) {
    if (tile_fits<AC, BC, MASK>(G) && (OUT == OUT_WEIGHTS ? G.large : large_tiles_fill(G.M, G.N, num_cus))) {
      if constexpr (OUT != OUT_WEIGHTS) {
        // Two workgroups per CU on half the tile where the whole ones leave CUs idle: 4096 x 1024 -> 1024 (64 tiles) 38 -> 29 us, 16384 x 512 -> 512 (128 tiles)
        // 27 -> 22; 8192 x 4096 -> 2048 (256 tiles) would go from 136 to 141
        if (G.N > 128 && up(G.M, 256) * up(G.N, 256) < num_cus) {
          launch_tile<T, GridPair, AC, BC, OUT, MASK>(st, G, num_cus);
          return;
        }
      }
      if (G.N > 128) launch_tile<T, Grid256, AC, BC, OUT, MASK>(st, G, num_cus);
      else launch_tile<T, Grid128, AC, BC, OUT, MASK>(st, G, num_cus);
      return;
    }
  }
  G.tiles_n = (int)up(G.N, BN);
  G.tiles = up(G.M, BM) * G.tiles_n;
  hipLaunchKernelGGL((k_gemm<T, AC, BC, OUT, MASK>), dim3((unsigned)G.tiles, G.splits), dim3(THREADS), 0, st, G);
  if constexpr (OUT != OUT_WEIGHTS) {
    if (G.part != nullptr) hipLaunchKernelGGL((k_join<T, OUT>), dim3((unsigned)up(G.M * up(G.N, 8), 256)), dim3(256), 0, st, G);
  }
}

template <typename T> void forward_t(hipStream_t st, const DenseFwd& f, int num_cus) {
  if (f.m <= 8) {
    const dim3 grid((unsigned)up(f.n, 32));
    if (f.m == 1) hipLaunchKernelGGL((k_rows<T, 1>), grid, dim3(256), 0, st, f);
    else if (f.m <= 2) hipLaunchKernelGGL((k_rows<T, 2>), grid, dim3(256), 0, st, f);
    else if (f.m <= 4) hipLaunchKernelGGL((k_rows<T, 4>), grid, dim3(256), 0, st, f);
    else hipLaunchKernelGGL((k_rows<T, 8>), grid, dim3(256), 0, st, f);
    return;
  }
  GemmArgs G{};
  G.a = f.x; G.lda = f.ldx; G.b = f.kernel; G.ldb = f.ldk; G.M = f.m; G.N = f.n; G.C = f.k;
  G.bias = f.bias; G.residual = f.residual; G.ldr = f.ldr; G.y = f.y; G.ldy = f.ldy; G.act = f.act;
  G.save = f.save; G.lds = f.act == ACT_RELU ? up(f.n, 8) : f.n;
  const Splits s = f.ws != nullptr ? row_splits(f.dtype, f.m, f.n, f.k, num_cus) : Splits{1, f.k};
  G.splits = s.count; G.cps = s.cps;
  if (s.count > 1) G.part = static_cast<float*>(f.ws);
  launch<T, true, false, OUT_FORWARD, 0>(st, G, num_cus);
}

template <typename T, int KP, int NP, int MODE, bool LO> void launch_both(hipStream_t st, const BothArgs& G, int grid) {
  auto kern = k_both<T, KP, NP, MODE, LO>;
  nerfds::allow_dynamic_lds(reinterpret_cast<const void*>(kern), Both<KP, NP, MODE>::LDS);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(512), (Both<KP, NP, MODE>::LDS), st, G);
}
template <typename T, int MODE, bool LO> void launch_both_of(hipStream_t st, const BothArgs& G, int grid) {
  if (G.k > 128 && G.n > 128) {
    if constexpr (!LO) launch_both<T, 256, 256, MODE, LO>(st, G, grid);      // (two parts: never of this size)
  } else if (G.k > 128) launch_both<T, 256, 128, MODE, LO>(st, G, grid);
  else if (G.n > 128) launch_both<T, 128, 256, MODE, LO>(st, G, grid);
  else launch_both<T, 128, 128, MODE, LO>(st, G, grid);
}

template <typename T> void backward_t(hipStream_t st, const DenseBwd& w, int num_cus) {
  char* ws = static_cast<char*>(w.ws);
  const void* dz = w.dy;
  long long lddz = w.lddy;
  const bool stored = stores_dz(w) && !slopes_in_both(w);
  const long long lo = two_parts(w) ? up(w.m * w.n, 8) * 8 : 0;
  if (stored) {
    const long long grans = w.m * up(w.n, 8), want = up(grans, 256);
    hipLaunchKernelGGL((w.act == ACT_RELU ? k_dz<T, true> : k_dz<T, false>), dim3((unsigned)(want < 16LL * num_cus ? want : 16LL * num_cus)), dim3(256), 0, st,
                       static_cast<const T*>(w.dy), w.lddy, w.save, reinterpret_cast<T*>(ws), w.m, w.n, w.act, lo);
    dz = ws; lddz = w.n;
    ws += dz_bytes(w);
  }
  const unsigned char* bits = w.act == ACT_RELU && !stored ? static_cast<const unsigned char*>(w.save) : nullptr;
  if constexpr (sizeof(T) == 2) {
    if (both_at_once(w)) {
      const int grid = weight_splits(w, num_cus).count;
      const long long kn = (long long)w.k * w.n;
      float* part = reinterpret_cast<float*>(ws);
      float* col = reinterpret_cast<float*>(ws + weight_part_bytes(w, grid));
      const BothArgs G{w.x, w.ldx, dz, lddz, w.kernel, w.ldk, w.save, w.act == ACT_RELU ? up(w.n, 8) : w.n, w.act, w.dx, w.lddx, part, w.dbias ? col : nullptr, w.m, w.k, w.n, lo};
      if (bits) launch_both_of<T, BOTH_RELU, false>(st, G, grid);
      else if (slopes_in_both(w)) launch_both_of<T, BOTH_SLOPE, false>(st, G, grid);
      else if (lo != 0) launch_both_of<T, BOTH_PLAIN, true>(st, G, grid);
      else launch_both_of<T, BOTH_PLAIN, false>(st, G, grid);
      sum_splits<T>(st, SplitSum{part, up(kn, 4) * 4, kn, w.dkernel}, SplitSum{col, up(w.n, 4) * 4, w.n, w.dbias}, grid);
      return;
    }
  }
  if (w.dx != nullptr) {
    GemmArgs G{};
    G.a = dz; G.lda = lddz; G.b = w.kernel; G.ldb = w.ldk; G.M = w.m; G.N = w.k; G.C = w.n;
    G.lo = lo; G.mask = bits; G.ldm = up(w.n, 8); G.y = w.dx; G.ldy = w.lddx;
    const Splits s = row_splits(w.dtype, w.m, w.k, w.n, num_cus);
    G.splits = s.count; G.cps = s.cps;
    if (s.count > 1) G.part = reinterpret_cast<float*>(ws);      // (joined before the weight gradient's parts come here)
    if (bits) launch<T, true, true, OUT_PLAIN, 1>(st, G, num_cus); else launch<T, true, true, OUT_PLAIN, 0>(st, G, num_cus);
  }
  if (w.dkernel != nullptr || w.dbias != nullptr) {
    const Splits s = weight_splits(w, num_cus);
    GemmArgs G{};
    G.a = w.x; G.lda = w.ldx; G.b = dz; G.ldb = lddz; G.N = w.n; G.C = w.m;
    G.M = w.dkernel ? w.k : 1;      // (the bias gradient alone: it rides on the first tile of the kernel's rows)
    G.lo = lo; G.mask = bits; G.ldm = up(w.n, 8); G.splits = s.count; G.cps = s.cps; G.large = weight_tiles_large(w);
    const long long kn = (long long)w.k * w.n;
    const size_t part_bytes = weight_part_bytes(w, s.count);
    G.part = w.dkernel && s.count > 1 ? reinterpret_cast<float*>(ws) : nullptr;
    float* col = reinterpret_cast<float*>(ws + part_bytes);
    if (s.count == 1) { G.y = w.dkernel; G.ldy = w.n; G.dbias = w.dbias; }
    else G.colpart = w.dbias ? col : nullptr;
    if (bits) launch<T, false, false, OUT_WEIGHTS, 2>(st, G, num_cus); else launch<T, false, false, OUT_WEIGHTS, 0>(st, G, num_cus);
    if (s.count > 1) sum_splits<T>(st, SplitSum{G.part, up(kn, 4) * 4, kn, w.dkernel}, SplitSum{col, up(w.n, 4) * 4, w.n, w.dbias}, s.count);
  }
}

}  // namespace

size_t dense_save_bytes(int dtype, int act, long long m, int n) {
  return act == ACT_NONE ? 0 : act == ACT_RELU ? (size_t)m * up(n, 8) : (size_t)m * n * dtype_bytes(dtype);
}
size_t dense_fwd_ws(const DenseFwd& a, int num_cus) { return row_part_bytes(row_splits(a.dtype, a.m, a.n, a.k, num_cus), a.m, a.n); }
size_t dense_bwd_ws(const DenseBwd& a, int num_cus) {
  const Splits s = weight_splits(a, num_cus);
  const size_t weights = a.dkernel != nullptr || a.dbias != nullptr ? weight_part_bytes(a, s.count) + (s.count > 1 || both_at_once(a) ? aligned((size_t)s.count * up(a.n, 4) * 16) : 0) : 0;
  const size_t rows = a.dx != nullptr && !both_at_once(a) ? row_part_bytes(row_splits(a.dtype, a.m, a.k, a.n, num_cus), a.m, a.k) : 0;
  return dz_bytes(a) + (weights > rows ? weights : rows);
}
void dense_forward(hipStream_t st, const DenseFwd& a, int num_cus) {
  if (a.dtype == F32) forward_t<float>(st, a, num_cus);
  else if (a.dtype == F16) forward_t<f16_t>(st, a, num_cus);
  else forward_t<bf16_t>(st, a, num_cus);
}
void dense_backward(hipStream_t st, const DenseBwd& a, int num_cus) {
  if (a.m == 0) {      // an empty sum is zero
    const long long kn = (long long)a.k * a.n;
#define CLEAR(T) sum_splits<T>(st, SplitSum{nullptr, 0, kn, a.dkernel}, SplitSum{nullptr, 0, a.n, a.dbias}, 0)
    if (a.dtype == F32) CLEAR(float); else if (a.dtype == F16) CLEAR(f16_t); else CLEAR(bf16_t);
#undef CLEAR
    return;
  }
  if (a.dtype == F32) backward_t<float>(st, a, num_cus);
  else if (a.dtype == F16) backward_t<f16_t>(st, a, num_cus);
  else backward_t<bf16_t>(st, a, num_cus);
}

}  // namespace nerfds_ops
