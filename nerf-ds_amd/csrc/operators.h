// Launch-side interface of the stand-alone operators (dense_kernel.hip, norm_kernel.hip, ortho_kernel.hip); the C ABI above it is operators.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nerfds_ops {

enum DType { F32 = 0, F16 = 1, BF16 = 2 };
enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SIGMOID = 2, ACT_SOFTPLUS = 3, ACT_SILU = 4, ACT_GELU = 5, ACT_COUNT = 6 };
inline size_t dtype_bytes(int t) { return t == F32 ? 4 : 2; }

// ---- dense: y = act(x kernel + bias) + residual ------------------------------------------------------------------------------------
struct DenseFwd {
  int dtype, act;
  long long m; int k, n;
  const void* x; long long ldx;             // [m][k]
  const void* kernel; long long ldk;        // [k][n]
  const void* bias;                         // [n] or nullptr
  const void* residual; long long ldr;      // [m][n] or nullptr (ldr 0: one row for all)
  void* y; long long ldy;                   // [m][n]
  void* save;                               // dense_save_bytes() for the backward pass, or nullptr
  void* ws;                                 // dense_fwd_ws() bytes or nullptr
};
struct DenseBwd {
  int dtype, act;
  long long m; int k, n;
  const void* x; long long ldx;
  const void* kernel; long long ldk;
  const void* dy; long long lddy;
  const void* save;
  void* dx; long long lddx;                 // [m][k] or nullptr
  void* dkernel;                            // [k][n] contiguous or nullptr
  void* dbias;                              // [n] or nullptr
  void* ws;                                 // dense_bwd_ws() bytes
};
// What the forward leaves for the backward: relu one bit per element (row-major, rows of whole bytes), the smooth activations the pre-activation in
// the tensors' type, no activation nothing.
size_t dense_save_bytes(int dtype, int act, long long m, int n);
size_t dense_fwd_ws(const DenseFwd& a, int num_cus);
size_t dense_bwd_ws(const DenseBwd& a, int num_cus);
void dense_forward(hipStream_t st, const DenseFwd& a, int num_cus);
void dense_backward(hipStream_t st, const DenseBwd& a, int num_cus);

// ---- layer norm over rows ------------------------------------------------------------------------------------------------------------
struct NormFwd {
  int dtype; long long m; int d; float eps;
  const void* x; long long ldx; const void* scale; const void* bias;      // scale / bias [d] or nullptr
  void* y; long long ldy;
  float* stats;                                                            // [m][2]: mean, 1 / sqrt(var + eps); nullptr = not wanted
};
struct NormBwd {
  int dtype; long long m; int d;
  const void* x; long long ldx; const void* scale; const void* dy; long long lddy; const float* stats;
  void* dx; long long lddx; void* dscale; void* dbias;                     // each may be nullptr
  float* ws;                                                               // norm_bwd_ws() bytes
};
size_t norm_bwd_ws(const NormBwd& a, int num_cus);
void norm_forward(hipStream_t st, const NormFwd& a, int num_cus);
void norm_backward(hipStream_t st, const NormBwd& a, int num_cus);

// ---- orthogonalised update ------------------------------------------------------------------------------------------------------------
struct OrthoMat { const void* u; long long ldu; void* o; long long ldo; int rows, cols; };
size_t ortho_ws(const OrthoMat* mats, int count);
void orthogonalize(hipStream_t st, int dtype, const OrthoMat* mats, int count, int steps, void* ws);


// ---- the trainer's update with orthogonalised kernels (muon_kernel.hip) --------------------------------------------------------------------
// up to 1024 elements of one leaf, from `offset` of the flat vectors; u >= 0: an orthogonalised leaf, its update starts at u of the update buffer
struct UpdateBlock { long long offset, u; int count; float scale; };
void muon_momentum(hipStream_t st, const UpdateBlock* blocks, int count, const float* g, float* m, float* u, float beta, int nesterov, const unsigned* skip);
void muon_update(hipStream_t st, const UpdateBlock* blocks, int count, const float* g, const float* o, float* p, float* m1, float* m2, float lr, float wd, const float* corr,
                 const unsigned* skip);

}  // namespace nerfds_ops
