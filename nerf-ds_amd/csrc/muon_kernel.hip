// The trainer's update with orthogonalised kernels (nerfds_trainer_set_optimizer): element-wise passes either side of ortho_kernel.hip.
//   momentum   m <- beta m + g,  u = g + beta m (Nesterov) or m                        on the orthogonalised leaves
//   update     W <- W (1 - lr wd) - lr 0.2 sqrt(max(rows, cols)) O                     there: an orthogonal O has an RMS of 1 / sqrt(max(rows, cols)), so the factor
//                                                                                      gives every element the RMS of a typical Adam update, 0.2, and both
//                                                                                      kinds of leaves follow one learning-rate schedule
//              flax.optim.Adam's                                                       on all others
// One workgroup per 1024 elements of one leaf (a table made once); both do nothing where the gradient check of the step has raised its flag.  Bound by memory
// and, at the 1.5 million parameters of the field (6 MB a vector), by the launch: 7 and 5 us around the 160 of the 40 orthogonalisations.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "operators.h"

namespace nerfds_ops {

namespace {

__global__ __launch_bounds__(256) void k_momentum(const UpdateBlock* __restrict__ blocks, const float* __restrict__ g, float* __restrict__ m, float* __restrict__ u, float beta, int nesterov,
                                                  const unsigned* __restrict__ skip) {
  const UpdateBlock B = blocks[blockIdx.x];
  if (B.u < 0 || *skip != 0u) return;
  for (int i = threadIdx.x; i < B.count; i += 256) {
    const float gi = g[B.offset + i], mi = fmaf(beta, m[B.offset + i], gi);
    m[B.offset + i] = mi;
    u[B.u + i] = nesterov ? fmaf(beta, mi, gi) : mi;
  }
}

__global__ __launch_bounds__(256) void k_update(const UpdateBlock* __restrict__ blocks, const float* __restrict__ g, const float* __restrict__ o, float* __restrict__ p, float* __restrict__ m1,
                                                float* __restrict__ m2, float lr, float wd, const float* __restrict__ corr, const unsigned* __restrict__ skip) {
  const UpdateBlock B = blocks[blockIdx.x];
  if (*skip != 0u) return;
  if (B.u >= 0) {
    for (int i = threadIdx.x; i < B.count; i += 256) p[B.offset + i] = p[B.offset + i] * (1.f - lr * wd) - lr * B.scale * o[B.u + i];
    return;
  }
  const float b1 = 0.9f, b2 = 0.999f, eps = 1e-8f, c1 = corr[0], c2 = corr[1];
  for (int i = threadIdx.x; i < B.count; i += 256) {
    const long long e = B.offset + i;
    const float gi = g[e], a = (1.0f - b1) * gi + b1 * m1[e], b = (1.0f - b2) * gi * gi + b2 * m2[e];
    m1[e] = a;
    m2[e] = b;
    p[e] -= lr * (a / c1) / (sqrtf(b / c2) + eps);
  }
}

}  // namespace

void muon_momentum(hipStream_t st, const UpdateBlock* blocks, int count, const float* g, float* m, float* u, float beta, int nesterov, const unsigned* skip) {
  hipLaunchKernelGGL(k_momentum, dim3((unsigned)count), dim3(256), 0, st, blocks, g, m, u, beta, nesterov, skip);
}
void muon_update(hipStream_t st, const UpdateBlock* blocks, int count, const float* g, const float* o, float* p, float* m1, float* m2, float lr, float wd, const float* corr,
                 const unsigned* skip) {
  hipLaunchKernelGGL(k_update, dim3((unsigned)count), dim3(256), 0, st, blocks, g, o, p, m1, m2, lr, wd, corr, skip);
}

}  // namespace nerfds_ops
