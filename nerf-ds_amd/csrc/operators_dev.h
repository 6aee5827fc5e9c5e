// Device helpers shared by the stand-alone operators: 8-element granules of the three element types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nerfds_ops {

#define OPS_DEV __device__ __forceinline__

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
// 16 bytes from / to an address aligned to the element only: global memory takes one unaligned instruction, where the address is aligned it costs nothing
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

struct bf16_t { uint16_t v; };
struct f16_t { _Float16 v; };

template <typename T> OPS_DEV float to_f32(T x);
template <> OPS_DEV float to_f32<float>(float x) { return x; }
template <> OPS_DEV float to_f32<f16_t>(f16_t x) { return (float)x.v; }
template <> OPS_DEV float to_f32<bf16_t>(bf16_t x) { return __builtin_bit_cast(float, (unsigned)x.v << 16); }
template <typename T> OPS_DEV T from_f32(float x);
template <> OPS_DEV float from_f32<float>(float x) { return x; }
template <> OPS_DEV f16_t from_f32<f16_t>(float x) { return f16_t{(_Float16)x}; }
template <> OPS_DEV bf16_t from_f32<bf16_t>(float x) { return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)x)}; }

// 8 consecutive elements as they are stored
template <typename T> struct Gran { u32x4 v; };
template <> struct Gran<float> { f32x4 v[2]; };

template <typename T> OPS_DEV Gran<T> gran_zero() {
  if constexpr (sizeof(T) == 4) return Gran<T>{{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}};
  else return Gran<T>{u32x4{0u, 0u, 0u, 0u}};
}
// the granule at p, of which `valid` elements exist (the others read as 0 and are not touched)
template <typename T> OPS_DEV Gran<T> gran_load(const T* p, long long valid) {
  Gran<T> g = gran_zero<T>();
  if (valid >= 8) {
    if constexpr (sizeof(T) == 4) {
      g.v[0] = *reinterpret_cast<const f32x4_any*>(p);
      g.v[1] = *reinterpret_cast<const f32x4_any*>(p + 4);
    } else g.v = *reinterpret_cast<const u32x4_any*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < valid) {
        if constexpr (sizeof(T) == 4) g.v[i >> 2][i & 3] = p[i];
        else g.v[i >> 1] |= (unsigned)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i & 1));
      }
    }
  }
  return g;
}
template <typename T> OPS_DEV float gran_get(const Gran<T>& g, int i) {
  if constexpr (sizeof(T) == 4) return g.v[i >> 2][i & 3];
  else return to_f32<T>(__builtin_bit_cast(T, (uint16_t)(g.v[i >> 1] >> (16 * (i & 1)))));
}
template <typename T> struct Pair;      // two elements, for the conversions that take two
template <> struct Pair<f16_t> { typedef __attribute__((ext_vector_type(2))) _Float16 type; };
template <> struct Pair<bf16_t> { typedef __attribute__((ext_vector_type(2))) __bf16 type; };
template <typename T> OPS_DEV Gran<T> gran_pack(const float (&f)[8]) {
  Gran<T> g = gran_zero<T>();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) { g.v[i >> 1][2 * (i & 1)] = f[2 * i]; g.v[i >> 1][2 * (i & 1) + 1] = f[2 * i + 1]; }
    else {
      typedef __attribute__((ext_vector_type(2))) float f32x2;
      g.v[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), typename Pair<T>::type));
    }
  }
  return g;
}
template <typename T> OPS_DEV void gran_store(T* p, const Gran<T>& g, long long valid) {
  if (valid >= 8) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_any*>(p) = g.v[0];
      *reinterpret_cast<f32x4_any*>(p + 4) = g.v[1];
    } else *reinterpret_cast<u32x4_any*>(p) = g.v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) {
        if constexpr (sizeof(T) == 4) p[i] = g.v[i >> 2][i & 3];
        else p[i] = __builtin_bit_cast(T, (uint16_t)(g.v[i >> 1] >> (16 * (i & 1))));
      }
  }
}

// Workgroup number -> position in the tile order, so that neighbours in the order (which share operand tiles) run on one XCD and meet in its L2: the
// hardware deals workgroups round-robin over 8 XCDs, so XCD x gets the x-th eighth of the order.
OPS_DEV long long xcd_order(long long wg, long long total) {
  const long long per = total / 8, rest = total % 8, x = wg % 8, i = wg / 8;
  return x * per + (x < rest ? x : rest) + i;
}

// ---- the second stage of a split sum --------------------------------------------------------------------------------------------------------
// out[c] = sum over p of part[p stride + c], rounded once, for two sums (strides are multiples of 4: what lies between count and stride is read, not used)
// in one launch (a weight's gradient and a bias's).  A lane takes 4 columns; DEEP threads share them, each adding every DEEP-th partial, and their sums are
// added in their order: 16 where there are that many partials (one thread per column: 31 us for 128 partials of 256 x 256, so: 7 us), 1 below (2 partials of
// 2048 x 4096: 50 us with 14 of 16 threads idle, 19 us).
struct SplitSum { const float* part; long long stride, count; void* out; };
template <typename T, int DEEP> __global__ __launch_bounds__(256) void k_sum_splits(SplitSum a, SplitSum b, int parts, unsigned blocks_a) {
  constexpr int WIDE = 256 / DEEP;      // lanes along the columns
  __shared__ f32x4 red[DEEP][WIDE];
  const SplitSum S = blockIdx.x < blocks_a ? a : b;
  const int l = threadIdx.x % WIDE, deep = threadIdx.x / WIDE;
  const long long c0 = (long long)(blockIdx.x < blocks_a ? blockIdx.x : blockIdx.x - blocks_a) * (4 * WIDE), c = c0 + 4 * l;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (c < S.count) {
#pragma unroll 8
    for (int p = deep; p < parts; p += DEEP) s += *reinterpret_cast<const f32x4*>(S.part + p * S.stride + c);
  }
  T* out = static_cast<T*>(S.out);
  if constexpr (DEEP == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) if (c + j < S.count) out[c + j] = from_f32<T>(s[j]);
  } else {
    red[deep][l] = s;
    __syncthreads();
    if (threadIdx.x < 4 * WIDE && c0 + threadIdx.x < S.count) {
      float v = 0.f;
      for (int q = 0; q < DEEP; ++q) v += red[q][threadIdx.x >> 2][threadIdx.x & 3];
      out[c0 + threadIdx.x] = from_f32<T>(v);
    }
  }
}
template <typename T, int DEEP> void sum_splits_deep(hipStream_t st, SplitSum a, SplitSum b, int parts) {
  const long long per = 1024 / DEEP;
  const unsigned na = a.out ? (unsigned)((a.count + per - 1) / per) : 0, nb = b.out ? (unsigned)((b.count + per - 1) / per) : 0;
  if (na + nb) hipLaunchKernelGGL((k_sum_splits<T, DEEP>), dim3(na + nb), dim3(256), 0, st, a, b, parts, na);
}
template <typename T> void sum_splits(hipStream_t st, SplitSum a, SplitSum b, int parts) {      // out == nullptr: that sum is not wanted
  if (parts >= 16) sum_splits_deep<T, 16>(st, a, b, parts); else sum_splits_deep<T, 1>(st, a, b, parts);
}

}  // namespace nerfds_ops
