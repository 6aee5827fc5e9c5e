// The forward and the data gradient of a layer whose whole kernel fits LDS (every layer of the radiance field: 256 x 256 is 128 KiB), for many rows:
// k_resident keeps the kernel in LDS for the life of a persistent workgroup and streams rows past it.  Included by dense_kernel.hip only.
//
// What bounds it: memory (524288 x 256 -> 256 in bf16: 512 bytes in and 512 out per row against 131072 multiply-adds, which the matrix pipe does in a sixth of
// the time).  So everything serves loads in flight: a wave works alone on 16 rows at a time - no barrier after the kernel is in LDS -, its rows come straight
// into registers in the layout the MFMA wants (16 rows x 64 contiguous bytes per load instruction), the next ones while it multiplies, and the residual of
// the rows in hand as well: 64 KiB of x and as much of the residual under way per CU.  LDS gives the kernel's fragments once per 16 rows, a third of its time.
// 524288 x 256 -> 256 in bf16 with bias, relu, its bits and the residual: 211 us (822 MB, 3.9 TB/s; a copy reaches 4.7); the data gradient alone 119 - 128.
// Loads return in order, so nothing small may be asked for behind the next rows and waited for: the bias is one more contraction step of the kernel in LDS,
// against a 1 behind the end of each row.
#pragma once

OPS_DEV f32x4 mma_16(const u32x4& a, const u32x4& b, const f32x4& c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
OPS_DEV f32x4 mma_16(const u32x4& a, const u32x4& b, const f32x4& c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The kernel in LDS: a row is one output line's contraction (padded to 64 steps).
struct Resident {
  static __host__ __device__ int row_bytes(int c) { return (c + 63) / 64 * 128; }
  static __host__ __device__ int bytes(int n, int c) { return (n + 31) / 32 * 32 * row_bytes(c); }
  // (16 lanes read one granule of the lines 0-3, 8-11, 16-19, 24-27 of a pair together: onto the 16 granules that the banks span, in rows of 256 bytes and of 128)
  static OPS_DEV int place(int row_bytes, int row, int g) { return g ^ (row_bytes & 128 ? (row >> 1 & 1) | (row >> 2 & 6) : (row & 3) | (row >> 1 & 12)); }
  // A pair of 16-line tiles covers 32 output lines; line i of tile `half` is output 32 pair + 8 (i >> 2) + 4 half + (i & 3), so that a lane of the accumulators
  // holds 8 consecutive outputs.  Lane l: line l & 15, contraction steps 32 ks + 8 (l >> 4) ..
  static OPS_DEV u32x4 frag(const char* lds, int row_bytes, int pair, int half, int ks) {
    const int lane = threadIdx.x & 63, i = lane & 15, row = 32 * pair + 8 * (i >> 2) + 4 * half + (i & 3);
    return *reinterpret_cast<const u32x4*>(lds + row * row_bytes + (place(row_bytes, row, 4 * ks + (lane >> 4)) << 4));
  }
};

// NP: pairs of output tiles, 32 NP >= N.  MASK: the streamed rows are multiplied by the relu bits.
template <typename T, bool BC, int NP, int OUT, bool MASK, int ACT> __global__ __launch_bounds__(512) void k_resident(const GemmArgs G) {
  constexpr int KS = 8;      // contraction steps of 32 in a chunk of the streamed rows
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
  const bool with_bias = OUT == OUT_FORWARD && G.bias != nullptr;
  const int N = (int)G.N, C = (int)G.C, C1 = C + (with_bias ? 1 : 0), row_bytes = Resident::row_bytes(C1);
  const int grans = row_bytes / 16, lines = (N + 31) / 32 * 32;
  if constexpr (BC) {
    for (int e = threadIdx.x; e < lines * grans; e += 512) {
      const int row = e / grans, g = e - row * grans;
      const Gran<T> w = gran_load<T>(static_cast<const T*>(G.b) + row * G.ldb + 8 * g, row < N ? C - 8 * g : 0);
      *reinterpret_cast<u32x4*>(g_lds + row * row_bytes + (Resident::place(row_bytes, row, g) << 4)) = w.v;
    }
  } else {
    // stored with the contraction down the rows: blocks of 8 x 8 elements are transposed in registers, once
    const int wide = lines / 8;
    for (int e = threadIdx.x; e < wide * grans; e += 512) {
      const int c = e / wide * 8, n = e % wide * 8;
      u32x4 in[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        in[i] = gran_load<T>(c + i < C ? static_cast<const T*>(G.b) + (c + i) * G.ldb + n : static_cast<const T*>(G.bias) + n, c + i < C1 ? N - n : 0).v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __builtin_amdgcn_perm(in[2 * i + 1][j >> 1], in[2 * i][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
        *reinterpret_cast<u32x4*>(g_lds + (n + j) * row_bytes + (Resident::place(row_bytes, n + j, c / 8) << 4)) = out;
      }
    }
  }
  __syncthreads();
  const bool whole = N == 32 * NP;      // (bounds are checked once per 16 rows, not per granule, where nothing is ragged)
  const long long blocks = (G.M + 15) / 16, stride = (long long)gridDim.x * 8;
  long long block = (long long)blockIdx.x * 8 + wave;
  const int chunks = (C1 + 32 * KS - 1) / (32 * KS);
  const unsigned one = with_bias && q == (C & 31) >> 3 ? (unsigned)__builtin_bit_cast(uint16_t, from_f32<T>(1.f)) << (16 * (C & 1)) : 0u;

  struct Chunk { u32x4 v[KS]; u32x4 bits[MASK ? 2 : 1]; };
  auto fetch = [&](Chunk& x, long long b, int ch) __attribute__((always_inline)) {
    const long long m = 16 * b + (lane & 15);
    const bool in = m < G.M;
    const T* p = static_cast<const T*>(G.a) + m * G.lda + 8 * q;
    if (16 * b + 16 <= G.M && 32 * KS * (ch + 1) <= C) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x.v[ks] = *reinterpret_cast<const u32x4_any*>(p + 32 * (KS * ch + ks));
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = 32 * (KS * ch + ks);
        x.v[ks] = u32x4{0, 0, 0, 0};
        if (c < C) x.v[ks] = gran_load<T>(p + c, in ? C - c - 8 * q : 0).v;
      }
    }
    if constexpr (MASK) {      // one byte per granule: 32 bytes a chunk
      const unsigned char* s = G.mask + m * G.ldm + 32 * ch;
      const int left = in ? (int)G.ldm - 32 * ch : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x.bits[h] = u32x4{0, 0, 0, 0};
        typedef u32x4 __attribute__((aligned(1))) u32x4_bytes;
        if (left >= 16 * h + 16) x.bits[h] = *reinterpret_cast<const u32x4_bytes*>(s + 16 * h);
        else
          for (int e = 16 * h; e < left; ++e) x.bits[h][(e & 15) >> 2] |= (unsigned)s[e] << (8 * (e & 3));
      }
    }
  };

  // One unit: a chunk of 16 rows.  The next unit's loads are issued first; two units alternate between two sets of registers (a copy from one to the other
  // would wait for loads that have only just been issued).
  f32x4 acc[NP][2];
  Gran<T> r[OUT == OUT_FORWARD ? NP : 1];
  int ch = 0;
  auto unit = [&](const Chunk& cur, Chunk& next) __attribute__((always_inline)) {
    const long long m = 16 * block + (lane & 15);
    if (ch == 0) {
#pragma unroll
      for (int p = 0; p < NP; ++p) acc[p][0] = acc[p][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (OUT == OUT_FORWARD) {
        if (G.residual != nullptr) {
          const T* p0 = static_cast<const T*>(G.residual) + m * G.ldr + 8 * q;
          if (whole && 16 * block + 16 <= G.M) {
#pragma unroll
            for (int p = 0; p < NP; ++p) r[p].v = *reinterpret_cast<const u32x4_any*>(p0 + 32 * p);
          } else {
#pragma unroll
            for (int p = 0; p < NP; ++p) r[p] = gran_load<T>(p0 + 32 * p, m < G.M ? N - 32 * p - 8 * q : 0);
          }
        }
      }
    }
    const bool wrap = ch + 1 == chunks, all = whole && 16 * block + 16 <= G.M;
    if (!wrap || block + stride < blocks) fetch(next, wrap ? block + stride : block, wrap ? 0 : ch + 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = 32 * (KS * ch + ks);
      if (c < C1) {
        Gran<T> x{cur.v[ks]};
        if constexpr (OUT == OUT_FORWARD) {
          if (c + 32 > C) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x.v[i] |= (C & 7) >> 1 == i ? one : 0u;
          }
        }
        if constexpr (MASK) gran_mask<T>(x, cur.bits[ks >> 2][ks & 3] >> (8 * q));
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[p][h] = mma_16(Resident::frag(g_lds, row_bytes, p, h, KS * ch + ks), x.v, acc[p][h], T{});
      }
    }
    if (!wrap) { ++ch; return; }
    ch = 0;
    block += stride;

    unsigned relu[2] = {};
    const bool in = m < G.M;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int n = 32 * p + 8 * q, valid = in ? N - n : 0;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[p][e >> 2][e & 3];
      if constexpr (OUT == OUT_FORWARD) {
        if (G.save != nullptr) {
          if constexpr (ACT == ACT_RELU) {
            // the 4 bytes of the pair's 32 outputs, put together over the four lanes of a row; lane q keeps the dwords q and q + 4
            unsigned w = relu_bits(v) << (8 * q);      // (columns past N: the kernel's padding is 0, and so are they)
            w |= __shfl_xor(w, 16, 64);
            w |= __shfl_xor(w, 32, 64);
            if ((p & 3) == q) relu[p >> 2] = w;
          } else if constexpr (ACT != ACT_NONE) {
            if (all) *reinterpret_cast<u32x4_any*>(static_cast<T*>(G.save) + m * G.lds + n) = gran_pack<T>(v).v;
            else gran_store<T>(static_cast<T*>(G.save) + m * G.lds + n, gran_pack<T>(v), valid);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = act_value<T, ACT>(v[e]);
        if (G.residual != nullptr) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += gran_get<T>(r[p], e);
        }
      }
      if (all) *reinterpret_cast<u32x4_any*>(static_cast<T*>(G.y) + m * G.ldy + n) = gran_pack<T>(v).v;
      else gran_store<T>(static_cast<T*>(G.y) + m * G.ldy + n, gran_pack<T>(v), valid);
    }
    if constexpr (OUT == OUT_FORWARD && ACT == ACT_RELU) {
      if (G.save != nullptr && in) {
        unsigned char* s = static_cast<unsigned char*>(G.save) + m * G.lds;
        typedef unsigned __attribute__((aligned(1))) u32_any;
#pragma unroll
        for (int p = 0; p < (NP + 3) / 4; ++p) {
          const int at = 16 * p + 4 * q;      // byte
          if (at + 4 <= G.lds) *reinterpret_cast<u32_any*>(s + at) = relu[p];
          else
            for (int e = at; e < G.lds; ++e) s[e] = (unsigned char)(relu[p] >> (8 * (e - at)));
        }
      }
    }
  };
  Chunk x0, x1;
  if (block >= blocks) return;
  fetch(x0, block, 0);
  while (true) {
    unit(x0, x1);
    if (block >= blocks) break;
    unit(x1, x0);
    if (block >= blocks) break;
  }
}
