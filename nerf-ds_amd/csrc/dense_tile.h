// The products of dense_kernel.hip for 16-bit operands whose rows are whole 16-byte granules: operand tiles go from memory to LDS by DMA, RING stages deep, and
// a persistent workgroup streams through its output tiles - the loads of the next tile are under way while the last one's results are written.
// Included by dense_kernel.hip only.
//
// What bounds it and why these shapes: with k = n = 256 (a trunk layer) a byte of x is worth 256 multiply-adds, so the kernel has to stream; with
// k, n in the thousands the matrix pipe is the bound and LDS next to it: a wave of 128 x 64 outputs reads 6 KiB of fragments for 8 MFMAs of 32 cycles, three
// quarters of what LDS can give four SIMDs (64 x 64: all of it).  8 waves share a tile of 256 x 256 (or 256 x 128 where n is no more), one workgroup
// per CU; where those tiles are fewer than the CUs, two workgroups of 4 waves per CU share the card on 128 x 256.  8192 x 2048 -> 4096 in bf16: 139 us for the
// product (989 TFLOP/s), 167 with bias, gelu, its saved input and the residual; dx 133, the weight gradient 151.
#pragma once

extern __shared__ __attribute__((aligned(16))) char g_lds[];
__device__ u32x4 g_zeros[2];      // where the granules outside an operand are read from

// 16 (4) bytes per lane from src to LDS at base + 16 (4) lane; base is uniform.  In assembly, because the compiler puts a wait for ALL loads in front of every
// transposed LDS read once it knows of a DMA; the waits are wait_loads below.  (M0 is nobody else's here: LDS instructions do not use it.)
OPS_DEV void dma16(const void* src, unsigned base) { asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(base) : "memory"); }
OPS_DEV void dma4(const void* src, unsigned base) { asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(base) : "memory"); }
// all but the newest N loads have arrived, and this wave's LDS reads too: past the barrier that follows, the stage they came from may be overwritten
template <int N> OPS_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// One operand's stage: LINES lines of the tile x BK contraction steps.
//   contiguous: LDS row = line, 4 granules of 8 steps; strided: LDS row = step, LINES / 8 granules of 8 lines, read transposed.
//   PERM: fragments take the lines of a 32-line tile with bits 2 and 3 of their number swapped, which leaves each lane of the accumulator 8 consecutive
//   outputs at a time (first operand of the MFMA only).
template <int LINES_, bool CONT_, bool PERM, int WAVES> struct Stage {
  static constexpr int LINES = LINES_, BK = 32, BYTES = LINES * BK * 2, INSTR = BYTES / 1024, IPW = INSTR / WAVES;
  static constexpr bool CONT = CONT_;
  static constexpr int ROWG = CONT ? BK / 8 : LINES / 8;      // granules of an LDS row
  static_assert(INSTR % WAVES == 0, "whole instructions for each wave");
  static OPS_DEV int swz(int row) {
    // (16 lanes read together: 16 lines at one step, 4 to the 256 bytes that the banks span; or 4 steps of 4 granules)
    return CONT ? row >> 2 & 3 : (row & 3) << 2;
  }
  // this lane's granule of DMA instruction u of its wave
  static OPS_DEV void place(int u, int& row, int& g) {
    const int slot = ((threadIdx.x >> 6) + WAVES * u) * 64 + (threadIdx.x & 63);
    row = slot / ROWG;
    g = (slot % ROWG) ^ swz(row);
  }
  static OPS_DEV u32x4 frag(const char* lds, int t, int ks) {
    const int lane = threadIdx.x & 63;
    if constexpr (CONT) {
      const int l = lane & 31, row = 32 * t + (PERM ? (l & 19) | (l >> 1 & 4) | (l << 1 & 8) : l), g = 2 * ks + (lane >> 5);
      return *reinterpret_cast<const u32x4*>(lds + row * (ROWG * 16) + ((g ^ swz(row)) << 4));
    } else {
      // a 16-lane group reads [4 steps][16 lines]: lane i supplies step i / 4 and one of the four 4-line pieces, and receives line i
      const int i = lane & 15, piece = PERM ? (i >> 1 & 1) | (i << 1 & 2) : i & 3;
      const int row = 16 * ks + 8 * (lane >> 5) + (i >> 2), g = 4 * t + 2 * ((lane >> 4) & 1) + (piece >> 1);
      const char* at = lds + row * (ROWG * 16) + ((g ^ swz(row)) << 4) + (piece & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 4 * ROWG * 16)));      // (row + 4 swizzles alike)
      return u32x4{a[0], a[1], b[0], b[1]};
    }
  }
};

// WGM x WGN waves of (32 TM) x (32 TN) outputs
template <int WGM_, int WGN_, int TM_, int TN_, int RING_> struct Grid {
  static constexpr int WGM = WGM_, WGN = WGN_, TM = TM_, TN = TN_, BM = 32 * WGM * TM, BN = 32 * WGN * TN, WAVES = WGM * WGN, RING = RING_;
  static_assert(WAVES == 8 || WAVES == 4, "two waves per SIMD: one workgroup per CU, or two");
};
typedef Grid<2, 4, 4, 2, 4> Grid256;      // 256 x 256
typedef Grid<4, 2, 2, 2, 4> Grid128;      // 256 x 128
typedef Grid<1, 4, 4, 2, 3> GridPair;     // 128 x 256, two workgroups per CU

// Position in the order of work -> output tile: bands of 8 tile rows, down the band first, so that the tiles in flight on one XCD form a block and share
// operand tiles both ways
OPS_DEV void tile_of(long long order, long long tiles_m, long long tiles_n, long long& tm, long long& tn) {
  const long long band = order / (8 * tiles_n), rows = tiles_m - 8 * band < 8 ? tiles_m - 8 * band : 8, r = order - band * 8 * tiles_n;
  tm = 8 * band + r % rows;
  tn = r / rows;
}

// MASK: 0, or the operand (1 = a, 2 = b) that is multiplied by the relu bits, in LDS, after its stage has landed
template <typename T, typename GR, bool AC, bool BC, int OUT, int MASK, int ACT> __global__ __launch_bounds__(64 * GR::WAVES, 2) void k_tile(const GemmArgs G) {
  typedef Stage<GR::BM, AC, false, GR::WAVES> SA;
  typedef Stage<GR::BN, BC, true, GR::WAVES> SB;
  constexpr int BK = 32, RING = GR::RING, WAVES = GR::WAVES, TM = GR::TM, TN = GR::TN;
  constexpr int MW = MASK == 1 ? GR::BM / 64 : GR::BN / 64, MB = MASK ? MW * 256 : 0,      // DMA instructions and bytes of a stage's relu bits
                STAGE = SA::BYTES + SB::BYTES + MB, IPW = SA::IPW + SB::IPW + (MASK ? 1 : 0);
  static_assert(!MASK || ((MASK == 1 ? AC : !BC) && MW <= WAVES), "masked operand");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / GR::WGN, wn = wave % GR::WGN;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)g_lds);
  const char* const zeros = reinterpret_cast<const char*>(g_zeros);

  // this workgroup's items (tile x split): an XCD gets a stretch of the order, its workgroups take turns in it
  const long long items = G.tiles * G.splits, tiles_m = G.tiles / G.tiles_n;
  const int xcds = gridDim.x < 8 ? gridDim.x : 8, xcd = blockIdx.x % xcds, turn = gridDim.x / xcds + (xcd < (int)(gridDim.x % xcds) ? 1 : 0);
  const long long per = items / xcds, rest = items % xcds, first = xcd * per + (xcd < rest ? xcd : rest), last = first + per + (xcd < rest ? 1 : 0);
  long long item = first + blockIdx.x / xcds;
  if (item >= last) return;

  // ---- the issuing side: item `it_i`, step `c_i` ----
  long long it_i = item, c_i, c1_i;
  const char* pa[SA::IPW];
  const char* pb[SB::IPW];
  bool oka[SA::IPW], okb[SB::IPW];
  int ca[SA::IPW], cb[SB::IPW];      // contraction offset of this lane's granule within a stage
  const char* pm = nullptr;
  int cm = 0;
  bool okm = false;
  const long long stepa = (AC ? BK : BK * G.lda) * 2, stepb = (BC ? BK : BK * G.ldb) * 2;
  auto start_item = [&]() __attribute__((always_inline)) {
    const long long split = it_i / G.tiles;
    long long tm, tn;
    tile_of(it_i - split * G.tiles, tiles_m, G.tiles_n, tm, tn);
    const long long m0 = tm * GR::BM, n0 = tn * GR::BN;
    c_i = split * G.cps;
    c1_i = c_i + G.cps < G.C ? c_i + G.cps : G.C;
#pragma unroll
    for (int u = 0; u < SA::IPW; ++u) {
      int row, g;
      SA::place(u, row, g);
      const long long line = m0 + (AC ? row : 8 * g);
      ca[u] = AC ? 8 * g : row;
      oka[u] = line < G.M;
      pa[u] = static_cast<const char*>(G.a) + (AC ? line * G.lda + c_i + ca[u] : (c_i + ca[u]) * G.lda + line) * 2;
    }
#pragma unroll
    for (int u = 0; u < SB::IPW; ++u) {
      int row, g;
      SB::place(u, row, g);
      const long long line = n0 + (BC ? row : 8 * g);
      cb[u] = BC ? 8 * g : row;
      okb[u] = line < G.N;
      pb[u] = static_cast<const char*>(G.b) + (BC ? line * G.ldb + c_i + cb[u] : (c_i + cb[u]) * G.ldb + line) * 2;
    }
    if constexpr (MASK == 1) {      // BM lines x 4 bytes: dword d of the block is line d; waves past the last fetch the same again, so that every wave counts alike
      const long long line = m0 + 64 * (wave & (MW - 1)) + lane;
      okm = line < G.M;
      pm = reinterpret_cast<const char*>(G.mask) + line * G.ldm + (c_i >> 3);
    }
    if constexpr (MASK == 2) {      // 32 steps x BN / 8 bytes
      constexpr int D = GR::BN / 32;
      const int d = 64 * (wave & (MW - 1)) + lane;
      cm = d / D;
      const long long line = n0 + 32 * (d % D);
      okm = line < G.N;
      pm = reinterpret_cast<const char*>(G.mask) + (c_i + cm) * G.ldm + (line >> 3);
    }
  };
  auto issue = [&](int slot) __attribute__((always_inline)) {
    // past the last item: zeros, into a slot nobody reads any more, so that the waits can count instructions
    const bool run = it_i < last;
    const unsigned base = lds0 + slot * STAGE;
#pragma unroll
    for (int u = 0; u < SA::IPW; ++u) {
      dma16(run && oka[u] && c_i + ca[u] < c1_i ? pa[u] : zeros, base + (wave + WAVES * u) * 1024);
      pa[u] += stepa;
    }
#pragma unroll
    for (int u = 0; u < SB::IPW; ++u) {
      dma16(run && okb[u] && c_i + cb[u] < c1_i ? pb[u] : zeros, base + SA::BYTES + (wave + WAVES * u) * 1024);
      pb[u] += stepb;
    }
    if constexpr (MASK != 0) {
      dma4(run && okm && c_i + cm < c1_i ? pm : zeros, base + SA::BYTES + SB::BYTES + (wave & (MW - 1)) * 256);
      pm += MASK == 1 ? BK / 8 : BK * G.ldm;
    }
    c_i += BK;
    if (run && c_i >= c1_i) {
      it_i += turn;
      if (it_i < last) start_item();
    }
  };

  start_item();
#pragma unroll
  for (int s = 0; s < RING - 1; ++s) issue(s);
  int slot = 0;
  for (; item < last; item += turn) {
    const long long split = item / G.tiles;
    long long tm, tn;
    tile_of(item - split * G.tiles, tiles_m, G.tiles_n, tm, tn);
    const long long m0 = tm * GR::BM, n0 = tn * GR::BN, c0 = split * G.cps, c1 = c0 + G.cps < G.C ? c0 + G.cps : G.C;
    const bool sums = OUT == OUT_WEIGHTS && (G.colpart != nullptr || G.dbias != nullptr) && tm == 0 && wm == 0;
    f32x16 acc[TM][TN] = {};
    f32x16 cs[OUT == OUT_WEIGHTS ? TN : 1] = {};
    for (long long c = c0; c < c1; c += BK) {
      wait_loads<(RING - 2) * IPW>();
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      issue((slot + RING - 1) % RING);
      __builtin_amdgcn_sched_barrier(0);
      char* st = g_lds + slot * STAGE;
      if constexpr (MASK != 0) {
        typedef typename std::conditional<MASK == 1, SA, SB>::type SM;
        char* op = st + (MASK == 1 ? 0 : SA::BYTES);
        const unsigned char* bits = reinterpret_cast<const unsigned char*>(st + SA::BYTES + SB::BYTES);
#pragma unroll
        for (int u = 0; u < SM::IPW; ++u) {
          int row, g;
          SM::place(u, row, g);
          u32x4* at = reinterpret_cast<u32x4*>(op + ((wave + WAVES * u) * 64 + lane) * 16);
          Gran<T> v{*at};
          gran_mask<T>(v, bits[row * SM::ROWG + g]);
          *at = v.v;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int ks = 0; ks < BK / 16; ++ks) {
        u32x4 fa[TM], fb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = SB::frag(st + SA::BYTES, wn * TN + j, ks);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = SA::frag(st, wm * TM + i, ks);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j], T{});
        if constexpr (OUT == OUT_WEIGHTS) {      // the column sums of b are its product with ones
          if (sums) {
            const unsigned one2 = __builtin_bit_cast(uint16_t, from_f32<T>(1.f)) * 0x10001u;
#pragma unroll
            for (int j = 0; j < TN; ++j) cs[j] = mma(fb[j], u32x4{one2, one2, one2, one2}, cs[j], T{});
          }
        }
      }
      slot = slot + 1 == RING ? 0 : slot + 1;
    }

    // lane l holds row l & 31 of each 32 x 32 tile; registers 8 d .. 8 d + 7 are columns 16 d + 8 (l >> 5) ..
    const long long mw = m0 + 32 * TM * wm + (lane & 31), nw = n0 + 32 * TN * wn + 8 * (lane >> 5);
    if (OUT == OUT_WEIGHTS && G.part != nullptr) {
      float* out = G.part + split * ((G.M * G.N + 3) & ~3LL);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const long long m = mw + 32 * i, n = nw + 32 * j + 16 * d;
            if (m < G.M && n < G.N) {
              f32x4* o = reinterpret_cast<f32x4*>(out + m * G.N + n);      // (n, G.N multiples of 8)
              o[0] = f32x4{acc[i][j][8 * d], acc[i][j][8 * d + 1], acc[i][j][8 * d + 2], acc[i][j][8 * d + 3]};
              o[1] = f32x4{acc[i][j][8 * d + 4], acc[i][j][8 * d + 5], acc[i][j][8 * d + 6], acc[i][j][8 * d + 7]};
            }
          }
    } else if (OUT != OUT_WEIGHTS || G.y != nullptr) {
      float bias[OUT == OUT_FORWARD ? TN : 1][2][8];
      if constexpr (OUT == OUT_FORWARD) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const long long n = nw + 32 * j + 16 * d;
            const Gran<T> b = gran_load<T>(static_cast<const T*>(G.bias) + n, G.bias != nullptr && n < G.N ? 8 : 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[j][d][e] = gran_get<T>(b, e);
          }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const long long m = mw + 32 * i;
        unsigned relu[2] = {};
        Gran<T> r[TN][2];
        if constexpr (OUT == OUT_FORWARD) {
          if (G.residual != nullptr) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                const long long n = nw + 32 * j + 16 * d;
                r[j][d] = gran_load<T>(static_cast<const T*>(G.residual) + m * G.ldr + n, m < G.M && n < G.N ? 8 : 0);
              }
          }
        }
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const long long n = nw + 32 * j + 16 * d;
            const bool in = m < G.M && n < G.N;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = acc[i][j][8 * d + e];
            if constexpr (OUT == OUT_FORWARD) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] += bias[j][d][e];
              if (G.save != nullptr) {
                if constexpr (ACT == ACT_RELU) {
                  relu[j & 1] |= relu_bits(v) << (16 * d);
                } else if (ACT != ACT_NONE && in) gran_store<T>(static_cast<T*>(G.save) + m * G.lds + n, gran_pack<T>(v), 8);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = act_value<T, ACT>(v[e]);
              if (G.residual != nullptr) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += gran_get<T>(r[j][d], e);
              }
            }
            if (in) gran_store<T>(static_cast<T*>(G.y) + m * G.ldy + n, gran_pack<T>(v), 8);
          }
        if constexpr (OUT == OUT_FORWARD) {
          static_assert(TN == 2, "a wave's 64 columns are 8 bytes of relu bits per row");
          if (ACT == ACT_RELU && G.save != nullptr) {
            // this lane has the bytes 4 j + 2 d + h of its row (h = l >> 5): lane h = 0 puts them together with its partner's
            const unsigned o0 = __shfl_xor(relu[0], 32, 64), o1 = __shfl_xor(relu[1], 32, 64);
            const unsigned w0 = relu[0] | o0 << 8, w1 = relu[1] | o1 << 8;
            const long long n = n0 + 32 * TN * wn;
            if (lane < 32 && m < G.M && n < G.N) {
              unsigned char* p = static_cast<unsigned char*>(G.save) + m * G.lds + (n >> 3);
              if (n + 64 <= G.N) {
                typedef u32x2 __attribute__((aligned(1))) u32x2_any;
                *reinterpret_cast<u32x2_any*>(p) = u32x2{w0, w1};
              } else
                for (int e = 0; n + 8 * e < G.N; ++e) p[e] = (unsigned char)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
            }
          }
        }
      }
    }
    if constexpr (OUT == OUT_WEIGHTS) {
      if (sums && (lane & 31) == 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const long long n = nw + 32 * j + 16 * d;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = cs[j][8 * d + e];
            if (n >= G.N) continue;
            if (G.dbias != nullptr) gran_store<T>(static_cast<T*>(G.dbias) + n, gran_pack<T>(v), 8);
            else gran_store<float>(G.colpart + split * ((G.N + 3) & ~3LL) + n, gran_pack<float>(v), 8);
          }
      }
    }
  }
  wait_loads<0>();      // no DMA may be on its way into LDS that is no longer this workgroup's
}
