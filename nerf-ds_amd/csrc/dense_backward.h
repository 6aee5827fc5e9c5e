// Both gradients of a narrow layer (k, n <= 256) from ONE read of x and dy: dx = dz kernel^T and dkernel = x^T dz.  Included by
// dense_kernel.hip only.
//
// What bounds it: memory (524288 x 256 x 256: 822 MB at the least; as two products dy is read twice, 1090 MB).  A persistent workgroup of 8 waves streams 32
// rows of x and dy at a time (16 where k and n are past 128) through LDS by DMA, four such stages deep.  The workgroup's part of dkernel stays in registers
// (up to 128 per lane), written once at the end, and so does the kernel (each wave the 32 rows of it that make its 32 columns of dx); at 256 x 256 only three
// eighths of it find room there, the rest waits in LDS, 80 KB of it (half in registers spilled).  For 16 rows of 256 x 256 a wave does 16 MFMAs of 16 cycles for
// dx and 8 of 32 for dkernel: 0.4 us per CU with two waves on a SIMD, a third of the time that the rows' 25 KB take memory.
// Measured (relu): 197 - 235 us by the card, and 12 to add the 256 parts of dkernel (memory's floor 174; apart 119 - 128 and 130 - 142).
#pragma once

// MODE: what dz is - BOTH_PLAIN: given; BOTH_RELU: dy by the relu bits; BOTH_SLOPE: dy act'(z), made in LDS from both
enum { BOTH_PLAIN = 0, BOTH_RELU = 1, BOTH_SLOPE = 2 };
template <int KP_, int NP_, int MODE> struct Both {
  static constexpr int KP = KP_, NP = NP_;      // k and n, padded to 128 or 256
  // rows per stage: 32, or 16 for the layer of 256 x 256, where KL of its contraction steps of 32 wait in LDS (KR are in registers)
  static constexpr bool FULL = KP == 256 && NP == 256;
  static constexpr int ROWS = FULL ? 16 : 32, XB = ROWS * KP * 2, YB = ROWS * NP * 2, EXTRA = MODE == BOTH_RELU ? ROWS * NP / 8 : MODE == BOTH_SLOPE ? YB : 0,
                       STAGE = XB + YB + EXTRA, RING = MODE == BOTH_SLOPE && NP == 256 ? 3 : 4;      // (z's rows beside dy's leave LDS for three stages)
  static constexpr int KS = NP / 32, KL = FULL ? 5 : 0, KR = KS - KL, LDS = RING * STAGE + 8 * 2 * KL * 1024;
  static constexpr int XI = XB / 8192, YI = YB / 8192;      // DMA instructions of a stage per wave
  // dkernel: GK x GN waves of (32 WK) x (32 WN); dx: RT tiles of 16 rows x 32 columns per wave
  static constexpr int GK = KP == 128 && NP == 256 ? 2 : 4, GN = 8 / GK, WK = KP / 32 / GK, WN = NP / 32 / GN, RT = ROWS * KP / 4096;
  static_assert(WK * GK * 32 == KP && WN * GN * 32 == NP, "waves");
  // Granule g of row r sits at g ^ turn(r): 16 rows of one granule (dx) and 4 rows of 4 granules (dkernel, transposed) both fall on all 16 granules' banks
  static OPS_DEV int turn(int r) { return (r << 2 & 12) | (r >> 2 & 3); }
  template <int P> static OPS_DEV int at(int r, int g) { return r * (P * 2) + ((g ^ turn(r)) << 4); }
  // lines 32 t .. (of P), rows 16 ks ..: transposed reads as in Stage; PERM swaps bits 2 and 3 of the line's number
  template <int P, bool PERM> static OPS_DEV u32x4 across(const char* lds, int t, int ks) {
    const int lane = threadIdx.x & 63, i = lane & 15, piece = PERM ? (i >> 1 & 1) | (i << 1 & 2) : i & 3;
    const int row = 16 * ks + 8 * (lane >> 5) + (i >> 2), g = 4 * t + 2 * ((lane >> 4) & 1) + (piece >> 1);
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + at<P>(row, g) + (piece & 1) * 8)));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + at<P>(row + 4, g) + (piece & 1) * 8)));
    return u32x4{a[0], a[1], b[0], b[1]};
  }
};

struct BothArgs {
  const void* x; long long ldx; const void* dz; long long lddz; const void* kernel; long long ldk;
  const void* save; long long lds; int act;      // relu bits or z
  void* dx; long long lddx;
  float* part; float* colpart;      // [grid][k n rounded up to 4], [grid][n rounded up to 4] (nullptr: no bias gradient)
  long long m; int k, n;
  long long lo;      // elements from dz to its second part (LO)
};

// LO: dz comes in two parts, and every stage twice, with one and the other
template <typename T, int KP, int NP, int MODE, bool LO> __global__ __launch_bounds__(512) void k_both(const BothArgs G) {
  typedef Both<KP, NP, MODE> S;
  constexpr int IPW = S::XI + S::YI + (MODE == BOTH_RELU ? 1 : MODE == BOTH_SLOPE ? S::YI : 0), RT = S::RT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)g_lds);
  const char* const zeros = reinterpret_cast<const char*>(g_zeros);
  const long long stages = (G.m + S::ROWS - 1) / S::ROWS;
  const int cols = KP == 256 ? wave : wave & 3, row_tile = KP == 256 ? 0 : wave >> 2;      // this wave's columns (32 of them) and first 16 rows of dx

  // the kernel's rows 32 cols .. as MFMA operands: line i of tile h is row 32 cols + 8 (i >> 2) + 4 h + (i & 3), so that a lane ends up with 8 consecutive columns of dx
  u32x4 w[2][S::KR];
  u32x4* const mine = reinterpret_cast<u32x4*>(g_lds + S::RING * S::STAGE + wave * (2 * S::KL * 1024)) + lane;      // (read by the wave that wrote them)
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
      const int row = 32 * cols + 8 * (i16 >> 2) + 4 * h + (i16 & 3), c = 32 * ks + 8 * q;
      const u32x4 v = gran_load<T>(static_cast<const T*>(G.kernel) + row * G.ldk + c, row < G.k ? G.n - c : 0).v;
      if (ks < S::KR) w[h][ks] = v; else mine[64 * (2 * (ks - S::KR) + h)] = v;
    }

  long long issued = blockIdx.x;
  int part_issued = 0, part = 0;
  auto issue = [&](int slot) __attribute__((always_inline)) {
    const unsigned base = lds0 + slot * S::STAGE;
    const long long r0 = issued * S::ROWS;
    auto tile = [&](const void* p, long long ld, int width, int instr, int per_row, unsigned to) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (u >= instr) break;
        const int s = (wave + 8 * u) * 64 + lane, row = s / per_row, g = (s % per_row) ^ S::turn(row);
        const bool in = r0 + row < G.m && 8 * g < width;      // (past the last stage: zeros, so that the waits can count)
        dma16(in ? static_cast<const char*>(p) + ((r0 + row) * ld + 8 * g) * 2 : zeros, to + (wave + 8 * u) * 1024);
      }
    };
    tile(G.x, G.ldx, G.k, S::XI, KP / 8, base);
    tile(static_cast<const T*>(G.dz) + (LO && part_issued ? G.lo : 0), G.lddz, G.n, S::YI, NP / 8, base + S::XB);
    if constexpr (MODE == BOTH_SLOPE) tile(G.save, G.lds, G.n, S::YI, NP / 8, base + S::XB + S::YB);
    if constexpr (MODE == BOTH_RELU) {      // NP / 32 dwords a row; the other waves fetch the same again, so that every wave counts alike
      constexpr int D = NP / 32, W = S::EXTRA / 256;
      const int d = 64 * (wave & (W - 1)) + lane, row = d / D, c = d % D;
      const bool in = r0 + row < G.m && 32 * c < G.n;
      dma4(in ? static_cast<const char*>(G.save) + (r0 + row) * G.lds + 4 * c : zeros, base + S::XB + S::YB + (wave & (W - 1)) * 256);
    }
    part_issued ^= 1;
    if (!LO || !part_issued) issued += gridDim.x;
  };

  f32x16 acc[S::WK][S::WN] = {};
  float cs[8] = {};
  const int wk = wave / S::GN, wn = wave % S::GN;
  const bool stores = 32 * cols < G.k;      // (every full stage then stores RT granules per lane)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the kernel's loads: nothing but DMA and this loop's stores on the counter from here
#pragma unroll
  for (int s = 0; s < S::RING - 1; ++s) issue(s);
  int slot = 0, done = 0;
  f32x4 d[RT][2];
  for (long long stage = blockIdx.x; stage < stages;) {
    // this stage's DMA has landed: newer are two stages and, from the fourth stage on, the stores of three (LO: of one at the least; the partial stage, which may
    // store less, is the last)
    if (done >= S::RING - 1 && stores) wait_loads<(S::RING - 2) * IPW + (LO ? 1 : S::RING - 1) * RT>(); else wait_loads<(S::RING - 2) * IPW>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue((slot + S::RING - 1) % S::RING);
    __builtin_amdgcn_sched_barrier(0);
    char* const x = g_lds + slot * S::STAGE;
    char* const y = x + S::XB;
    if (MODE != BOTH_PLAIN || G.colpart != nullptr) {
      // relu bits or slopes multiply dy in place; the column sums are taken of what this thread brought in - the same 8 columns in every stage
      const unsigned char* bits = reinterpret_cast<const unsigned char*>(y + S::YB);
#pragma unroll
      for (int u = 0; u < S::YI; ++u) {
        const int s = (wave + 8 * u) * 64 + lane, row = s / (NP / 8), g = (s % (NP / 8)) ^ S::turn(row);
        Gran<T> v{*reinterpret_cast<const u32x4*>(y + s * 16)};
        if constexpr (MODE == BOTH_RELU) gran_mask<T>(v, bits[row * (NP / 8) + g]);
        if constexpr (MODE == BOTH_SLOPE) {      // (rounded to the tensors' type: the matrix pipe takes it in no other)
          const Gran<T> z{*reinterpret_cast<const u32x4*>(y + S::YB + s * 16)};
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = gran_get<T>(z, e);
          act_slopes<T>(f, G.act);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= gran_get<T>(v, e);
          v = gran_pack<T>(f);
        }
        if constexpr (MODE != BOTH_PLAIN) *reinterpret_cast<u32x4*>(y + s * 16) = v.v;
        if (G.colpart != nullptr) {
#pragma unroll
          for (int e = 0; e < 8; ++e) cs[e] += gran_get<T>(v, e);
        }
      }
      if constexpr (MODE != BOTH_PLAIN) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (!LO || part == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) d[t][0] = d[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const u32x4 z = *reinterpret_cast<const u32x4*>(y + S::template at<NP>(16 * (row_tile + t) + i16, 4 * ks + q));
#pragma unroll
        for (int h = 0; h < 2; ++h) d[t][h] = mma_16(ks < S::KR ? w[h][ks < S::KR ? ks : 0] : mine[64 * (2 * (ks - S::KR) + h)], z, d[t][h], T{});
      }
#pragma unroll
    for (int ks = 0; ks < S::ROWS / 16; ++ks) {
      u32x4 fx[S::WK], fy[S::WN];
#pragma unroll
      for (int i = 0; i < S::WK; ++i) fx[i] = S::template across<KP, false>(x, wk * S::WK + i, ks);
#pragma unroll
      for (int j = 0; j < S::WN; ++j) fy[j] = S::template across<NP, true>(y, wn * S::WN + j, ks);
#pragma unroll
      for (int i = 0; i < S::WK; ++i)
#pragma unroll
        for (int j = 0; j < S::WN; ++j) acc[i][j] = mma(fy[j], fx[i], acc[i][j], T{});
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (LO && part == 0) break;
      const long long m = stage * S::ROWS + 16 * (row_tile + t) + i16;
      const int c = 32 * cols + 8 * q;
      const float v[8] = {d[t][0][0], d[t][0][1], d[t][0][2], d[t][0][3], d[t][1][0], d[t][1][1], d[t][1][2], d[t][1][3]};
      if (m < G.m && c < G.k) *reinterpret_cast<u32x4_any*>(static_cast<T*>(G.dx) + m * G.lddx + c) = gran_pack<T>(v).v;
    }
    slot = slot + 1 == S::RING ? 0 : slot + 1;
    ++done;
    part ^= 1;
    if (!LO || part == 0) stage += gridDim.x;
  }
  wait_loads<0>();      // no DMA may be on its way into LDS that is used otherwise, or no longer this workgroup's

  float* out = G.part + blockIdx.x * (((long long)G.k * G.n + 3) & ~3LL);
#pragma unroll
  for (int i = 0; i < S::WK; ++i)
#pragma unroll
    for (int j = 0; j < S::WN; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = 32 * (wk * S::WK + i) + (lane & 31), n = 32 * (wn * S::WN + j) + 16 * e + 8 * (lane >> 5);
        if (k < G.k && n < G.n) {
          f32x4* o = reinterpret_cast<f32x4*>(out + (long long)k * G.n + n);      // (n, G.n multiples of 8)
          o[0] = f32x4{acc[i][j][8 * e], acc[i][j][8 * e + 1], acc[i][j][8 * e + 2], acc[i][j][8 * e + 3]};
          o[1] = f32x4{acc[i][j][8 * e + 4], acc[i][j][8 * e + 5], acc[i][j][8 * e + 6], acc[i][j][8 * e + 7]};
        }
      }
  if (G.colpart != nullptr) {
    float* red = reinterpret_cast<float*>(g_lds);      // [threads of one column group][NP], added in their order
    const int row = (wave * 64 + lane) / (NP / 8), g = ((wave * 64 + lane) % (NP / 8)) ^ S::turn(row);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) red[row * NP + 8 * g + e] = cs[e];
    __syncthreads();
    if (threadIdx.x < NP && (int)threadIdx.x < G.n) {
      float v = 0.f;
      for (int r = 0; r < 4096 / NP; ++r) v += red[r * NP + threadIdx.x];
      G.colpart[blockIdx.x * ((G.n + 3) & ~3LL) + threadIdx.x] = v;
    }
  }
}
