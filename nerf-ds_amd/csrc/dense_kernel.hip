// y = act(x kernel + bias) + residual with its gradients, for any sizes, three element types.  The three matrix products are one tile kernel:
//   forward   y  [m x n] = x  [m x k] . kernel [k x n]       contraction over k
//   data      dx [m x k] = dz [m x n] . kernel^T             contraction over n
//   weights   dk [k x n] = x^T        . dz [m x n]           contraction over m, split over workgroups and summed in a second kernel
// dz = dy act'(z).  Each operand is stored with the contraction either along its rows ("contiguous") or across them ("strided"); a strided tile is
// transposed on its way from LDS to the registers (ds_read_b64_tr_b16), so no operand is ever transposed in memory.
#include <hip/hip_runtime.h>
#include <stdint.h>

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
//   contiguous: LDS row = line (BK elements), granule g of row r at g ^ sw(r): the 8 rows a quarter wave reads together fall on 8 different bank groups
//   strided:    LDS row = contraction step (128 elements), granule g of row r at g ^ ((r & 3) << 2), likewise for the 4 x 16 blocks of the transposed read
template <typename T, bool CONT> struct Tile {
  static constexpr int BK = Shape<T>::BK, P = Shape<T>::P, PLANE = 128 * BK * 2, BYTES = P * PLANE;
  static constexpr int NG = 128 * BK / 8 / THREADS;        // granules of a thread
  static OPS_DEV void place(int i, int& row, int& g) {
    const int idx = threadIdx.x + THREADS * i;
    if constexpr (CONT) { row = idx / (BK / 8); g = idx % (BK / 8); } else { row = idx / 16; g = idx % 16; }
  }
  static OPS_DEV int offset(int row, int g) {
    if constexpr (CONT) return row * (BK * 2) + ((g ^ (BK == 64 ? row & 7 : (row >> 1) & 3)) << 4);
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

OPS_DEV float sigmoid_(float z) { return 1.f / (1.f + expf(-z)); }
OPS_DEV float act_value(float z, int act) {
  switch (act) {
    case ACT_RELU: return z > 0.f || z != z ? z : 0.f;
    case ACT_SIGMOID: return sigmoid_(z);
    case ACT_SOFTPLUS: return fmaxf(z, 0.f) + log1pf(expf(-fabsf(z)));
    case ACT_SILU: return z * sigmoid_(z);
    case ACT_GELU: return 0.5f * z * erfcf(-0.70710678f * z);      // (erfc: 1 + erf cancels for negative z)
    default: return z;
  }
}
OPS_DEV float act_slope(float z, int act) {
  switch (act) {
    case ACT_SIGMOID: { const float s = sigmoid_(z); return s * (1.f - s); }
    case ACT_SOFTPLUS: return sigmoid_(z);
    case ACT_SILU: { const float s = sigmoid_(z); return s * (1.f + z * (1.f - s)); }
    case ACT_GELU: return 0.5f * erfcf(-0.70710678f * z) + z * expf(-0.5f * z * z) * 0.39894228f;
    default: return 1.f;
  }
}

enum { OUT_FORWARD = 0, OUT_PLAIN = 1, OUT_PARTIAL = 2 };

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
  const bool sums = OUT == OUT_PARTIAL && G.colpart != nullptr && m0 == 0;
  auto fetch = [&](long long c) __attribute__((always_inline)) {
    TA::load(ra, G.a, G.lda, m0, G.M, c, c1);
    TB::load(rb, G.b, G.ldb, n0, G.N, c, c1);
    if constexpr (MASK == 1) TA::mask(ra, G.mask, G.ldm, m0, G.M, c, c1);
    if constexpr (MASK == 2) TB::mask(rb, G.mask, G.ldm, n0, G.N, c, c1);
  };
  fetch(c0);
  for (long long c = c0; c < c1; c += BK) {
    __syncthreads();
    TA::stage(ra, lds);
    TB::stage(rb, lds + TA::BYTES);
    if constexpr (OUT == OUT_PARTIAL) {
      if (sums) {
#pragma unroll
        for (int i = 0; i < TB::NG; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) cs[j] += gran_get<T>(rb[i], j);
      }
    }
    __syncthreads();
    if (c + BK < c1) fetch(c + BK);
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

  if constexpr (OUT == OUT_PARTIAL) {
    if (G.part != nullptr) {
      float* out = G.part + (size_t)blockIdx.y * G.M * G.N;
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
    if (sums) {      // thread t holds the sums of columns 8 (t & 15) .. over its rows: 16 threads per column group
      float* red = reinterpret_cast<float*>(lds);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) red[(threadIdx.x >> 4) * 128 + 8 * (threadIdx.x & 15) + j] = cs[j];
      __syncthreads();
      if (threadIdx.x < 128 && n0 + threadIdx.x < G.N) {
        float s = 0.f;
        for (int q = 0; q < 16; ++q) s += red[q * 128 + threadIdx.x];
        G.colpart[(size_t)blockIdx.y * G.N + n0 + threadIdx.x] = s;
      }
    }
  } else {
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
#pragma unroll
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
          if (G.act == ACT_RELU) {
            unsigned bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) bits |= (v[j] > 0.f ? 1u : 0u) << j;
            if (G.save != nullptr) static_cast<unsigned char*>(G.save)[m * G.lds + (n >> 3)] = (unsigned char)bits;
          } else if (G.act != ACT_NONE && G.save != nullptr)
            gran_store<T>(static_cast<T*>(G.save) + m * G.lds + n, gran_pack<T>(v), valid);
          if (G.act != ACT_NONE) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = act_value(v[j], G.act);
          }
          if (G.residual != nullptr) {
            const Gran<T> g = gran_load<T>(static_cast<const T*>(G.residual) + m * G.ldr + n, valid);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += gran_get<T>(g, j);
          }
        }
        gran_store<T>(static_cast<T*>(G.y) + m * G.ldy + n, gran_pack<T>(v), valid);
      }
    }
  }
}

// out[i] = sum over the splits, rounded once
template <typename T> __global__ __launch_bounds__(256) void k_sum_splits(const float* __restrict__ part, int splits, long long count, T* __restrict__ out) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= count) return;
  float s = 0.f;
  for (int q = 0; q < splits; ++q) s += part[q * count + i];
  out[i] = from_f32<T>(s);
}

// dz = dy act'(z), once, for the activations whose slope costs more than a bit test (the products below read dz once per tile of their other axis).
// dz is rounded to the tensors' type: the matrix pipe takes it in no other.
template <typename T> __global__ __launch_bounds__(256) void k_dz(const T* __restrict__ dy, long long lddy, const T* __restrict__ z, T* __restrict__ dz, long long m, int n, int act) {
  const int gn = (n + 7) / 8;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < m * gn; i += gridDim.x * 256LL) {
    const long long row = i / gn;
    const int c = (int)(i % gn) * 8;
    const Gran<T> a = gran_load<T>(dy + row * lddy + c, n - c), b = gran_load<T>(z + row * n + c, n - c);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gran_get<T>(a, j) * act_slope(gran_get<T>(b, j), act);
    gran_store<T>(dz + row * n + c, gran_pack<T>(v), n - c);
  }
}

long long up(long long a, long long b) { return (a + b - 1) / b; }
size_t aligned(size_t b) { return (b + 255) & ~(size_t)255; }

struct Splits { int count; long long cps; };
// The weight gradient has few output tiles (4 for 256 x 256) and a long contraction: as many splits as give two workgroups per CU, none shorter than 4 steps
Splits weight_splits(long long m, int k, int n, int bk, int num_cus) {
  const long long tiles = up(k, BM) * up(n, BN), steps = up(m, bk);
  long long want = up(2LL * num_cus, tiles);
  if (want > up(steps, 4)) want = up(steps, 4);
  if (want < 1) want = 1;
  const long long cps = up(steps, want) * bk;
  return {(int)up(m, cps), cps};
}

template <typename T, bool AC, bool BC, int OUT, int MASK> void launch(hipStream_t st, GemmArgs& G) {
  G.tiles_n = (int)up(G.N, BN);
  G.tiles = up(G.M, BM) * G.tiles_n;
  hipLaunchKernelGGL((k_gemm<T, AC, BC, OUT, MASK>), dim3((unsigned)G.tiles, G.splits), dim3(THREADS), 0, st, G);
}

template <typename T> void forward_t(hipStream_t st, const DenseFwd& f) {
  GemmArgs G{};
  G.a = f.x; G.lda = f.ldx; G.b = f.kernel; G.ldb = f.ldk; G.M = f.m; G.N = f.n; G.C = f.k;
  G.bias = f.bias; G.residual = f.residual; G.ldr = f.ldr; G.y = f.y; G.ldy = f.ldy; G.act = f.act;
  G.save = f.save; G.lds = f.act == ACT_RELU ? up(f.n, 8) : f.n;
  G.splits = 1; G.cps = f.k;
  launch<T, true, false, OUT_FORWARD, 0>(st, G);
}

template <typename T> void backward_t(hipStream_t st, const DenseBwd& w, int num_cus) {
  char* ws = static_cast<char*>(w.ws);
  const void* dz = w.dy;
  long long lddz = w.lddy;
  if (w.act != ACT_NONE && w.act != ACT_RELU) {
    const long long grans = w.m * up(w.n, 8), want = up(grans, 256);
    hipLaunchKernelGGL((k_dz<T>), dim3((unsigned)(want < 16LL * num_cus ? want : 16LL * num_cus)), dim3(256), 0, st, static_cast<const T*>(w.dy), w.lddy,
                       static_cast<const T*>(w.save), reinterpret_cast<T*>(ws), w.m, w.n, w.act);
    dz = ws; lddz = w.n;
    ws += aligned((size_t)w.m * w.n * sizeof(T));
  }
  const unsigned char* bits = w.act == ACT_RELU ? static_cast<const unsigned char*>(w.save) : nullptr;
  if (w.dx != nullptr) {
    GemmArgs G{};
    G.a = dz; G.lda = lddz; G.b = w.kernel; G.ldb = w.ldk; G.M = w.m; G.N = w.k; G.C = w.n;
    G.mask = bits; G.ldm = up(w.n, 8); G.y = w.dx; G.ldy = w.lddx; G.splits = 1; G.cps = w.n;
    if (bits) launch<T, true, true, OUT_PLAIN, 1>(st, G); else launch<T, true, true, OUT_PLAIN, 0>(st, G);
  }
  if (w.dkernel != nullptr || w.dbias != nullptr) {
    const Splits s = weight_splits(w.m, w.k, w.n, Shape<T>::BK, num_cus);
    GemmArgs G{};
    G.a = w.x; G.lda = w.ldx; G.b = dz; G.ldb = lddz; G.N = w.n; G.C = w.m;
    G.M = w.dkernel ? w.k : 1;      // (the bias gradient alone: it rides on the first tile of the kernel's rows)
    G.mask = bits; G.ldm = up(w.n, 8); G.splits = s.count; G.cps = s.cps;
    G.part = w.dkernel ? reinterpret_cast<float*>(ws) : nullptr;
    float* col = reinterpret_cast<float*>(ws + aligned((size_t)s.count * w.k * w.n * 4));
    G.colpart = w.dbias ? col : nullptr;
    if (bits) launch<T, false, false, OUT_PARTIAL, 2>(st, G); else launch<T, false, false, OUT_PARTIAL, 0>(st, G);
    if (w.dkernel)
      hipLaunchKernelGGL((k_sum_splits<T>), dim3((unsigned)up((long long)w.k * w.n, 256)), dim3(256), 0, st, G.part, s.count, (long long)w.k * w.n, static_cast<T*>(w.dkernel));
    if (w.dbias)
      hipLaunchKernelGGL((k_sum_splits<T>), dim3((unsigned)up(w.n, 256)), dim3(256), 0, st, col, s.count, (long long)w.n, static_cast<T*>(w.dbias));
  }
}

}  // namespace

size_t dense_save_bytes(int dtype, int act, long long m, int n) {
  return act == ACT_NONE ? 0 : act == ACT_RELU ? (size_t)m * up(n, 8) : (size_t)m * n * dtype_bytes(dtype);
}
size_t dense_bwd_ws(const DenseBwd& a, int num_cus) {
  const Splits s = weight_splits(a.m, a.k, a.n, a.dtype == F32 ? Shape<float>::BK : Shape<f16_t>::BK, num_cus);
  size_t b = a.act != ACT_NONE && a.act != ACT_RELU ? aligned((size_t)a.m * a.n * dtype_bytes(a.dtype)) : 0;
  if (a.dkernel != nullptr || a.dbias != nullptr) b += aligned((size_t)s.count * a.k * a.n * 4) + aligned((size_t)s.count * a.n * 4);
  return b;
}
void dense_forward(hipStream_t st, const DenseFwd& a, int) {
  if (a.dtype == F32) forward_t<float>(st, a);
  else if (a.dtype == F16) forward_t<f16_t>(st, a);
  else forward_t<bf16_t>(st, a);
}
void dense_backward(hipStream_t st, const DenseBwd& a, int num_cus) {
  if (a.m == 0) {      // an empty sum is zero
    const long long kn = (long long)a.k * a.n;
#define CLEAR(T)                                                                                                                                                  \
    do {                                                                                                                                                          \
      if (a.dkernel) hipLaunchKernelGGL((k_sum_splits<T>), dim3((unsigned)up(kn, 256)), dim3(256), 0, st, nullptr, 0, kn, static_cast<T*>(a.dkernel));           \
      if (a.dbias) hipLaunchKernelGGL((k_sum_splits<T>), dim3((unsigned)up(a.n, 256)), dim3(256), 0, st, nullptr, 0, (long long)a.n, static_cast<T*>(a.dbias));  \
    } while (0)
    if (a.dtype == F32) CLEAR(float); else if (a.dtype == F16) CLEAR(f16_t); else CLEAR(bf16_t);
#undef CLEAR
    return;
  }
  if (a.dtype == F32) backward_t<float>(st, a, num_cus);
  else if (a.dtype == F16) backward_t<f16_t>(st, a, num_cus);
  else backward_t<bf16_t>(st, a, num_cus);
}

}  // namespace nerfds_ops
