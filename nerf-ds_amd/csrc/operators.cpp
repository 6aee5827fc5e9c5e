// C ABI of the stand-alone operators (include/nerfds.h): argument checks, the device, the launch.  No C++ exception leaves: messages are formatted
// into a fixed buffer, the batch lists of ortho_kernel.hip live on the stack, and the one temporary of its sort is asked for without throwing.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "nerfds.h"
#include "operators.h"

extern "C" void nerfds_set_last_error(const char* msg);

namespace {

using namespace nerfds_ops;

static_assert(F32 == NERFDS_DTYPE_F32 && F16 == NERFDS_DTYPE_F16 && BF16 == NERFDS_DTYPE_BF16, "element types");
static_assert(ACT_NONE == NERFDS_ACT_NONE && ACT_RELU == NERFDS_ACT_RELU && ACT_SIGMOID == NERFDS_ACT_SIGMOID && ACT_SOFTPLUS == NERFDS_ACT_SOFTPLUS &&
              ACT_SILU == NERFDS_ACT_SILU && ACT_GELU == NERFDS_ACT_GELU, "activations");

int fail(int rc, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int rc, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  try { nerfds_set_last_error(buf); } catch (...) {}
  return rc;
}

// makes `device` current for the call and puts the caller's device back
struct Device {
  int before = -1, device;
  bool ok;
  explicit Device(int d) : device(d) {
    ok = hipGetDevice(&before) == hipSuccess && (before == d || hipSetDevice(d) == hipSuccess);
    if (!ok) (void)hipGetLastError();
  }
  ~Device() { if (ok && before != device) (void)hipSetDevice(before); }
};

constexpr int MAX_DEVICES = 64;
int num_cus(int device) {
  static std::atomic<int> known[MAX_DEVICES];
  if (device < 0 || device >= MAX_DEVICES) return 0;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) { (void)hipGetLastError(); return 0; }
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NERFDS_OK : fail(NERFDS_EDEVICE, "%s: kernel launch failed: %s", who, hipGetErrorString(e));
}

constexpr int64_t MAX_ROWS = 1LL << 40, MAX_LD = 1LL << 40;
constexpr int32_t MAX_WIDTH = 1 << 24;

bool aligned_to(const void* p, size_t b) { return reinterpret_cast<uintptr_t>(p) % b == 0; }
bool element(const void* p, int32_t dtype) { return aligned_to(p, dtype_bytes(dtype)); }
int64_t tiles(int64_t a, int64_t b) { return ((a + 127) / 128) * ((b + 127) / 128); }

int check_dense(const char* who, int32_t dtype, int32_t act, int64_t m, int32_t k, int32_t n) {
  if (dtype < F32 || dtype > BF16) return fail(NERFDS_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (act < 0 || act >= ACT_COUNT) return fail(NERFDS_EINVAL, "%s: unknown activation %d", who, act);
  if (m < 0 || m > MAX_ROWS || k < 1 || n < 1 || k > MAX_WIDTH || n > MAX_WIDTH)
    return fail(NERFDS_EINVAL, "%s: m = %lld, k = %d, n = %d (0 <= m <= 2^40, 1 <= k, n <= 2^24)", who, (long long)m, k, n);
  // (a launch has less than 2^32 threads, a workgroup 256)
  if (tiles(m, n) >= (1LL << 24) || tiles(m, k) >= (1LL << 24) || tiles(k, n) >= (1LL << 24)) return fail(NERFDS_EINVAL, "%s: 2^24 output tiles of 128 x 128 or more", who);
  return NERFDS_OK;
}
int check_array(const char* who, const char* name, const void* p, int32_t dtype, int64_t ld, int64_t least) {
  if (!p || !element(p, dtype)) return fail(NERFDS_EINVAL, "%s: %s is %s", who, name, p ? "not aligned to its element type" : "null");
  if (ld < least || ld > MAX_LD) return fail(NERFDS_EINVAL, "%s: row stride %lld of %s is less than its %lld columns (or beyond 2^40)", who, (long long)ld, name, (long long)least);
  return NERFDS_OK;
}
int check_vector(const char* who, const char* name, const void* p, int32_t dtype) {
  return !p || element(p, dtype) ? NERFDS_OK : fail(NERFDS_EINVAL, "%s: %s is not aligned to its element type", who, name);
}
int check_workspace(const char* who, const void* p, int64_t have, int64_t need) {
  if (need > 0 && (!p || !aligned_to(p, 256) || have < need))
    return fail(NERFDS_EINVAL, "%s: the workspace needs %lld bytes, 256-byte aligned (got %lld at %p)", who, (long long)need, (long long)have, p);
  return NERFDS_OK;
}

DenseFwd dense_fwd_of(const nerfds_dense_forward_args& a) {
  return DenseFwd{a.dtype, a.activation, a.m, a.k, a.n, a.x, a.ldx, a.kernel, a.ldk, a.bias, a.residual, a.ldr, a.y, a.ldy, a.save, a.workspace};
}
DenseBwd dense_bwd_of(const nerfds_dense_backward_args& a) {
  return DenseBwd{a.dtype, a.activation, a.m, a.k, a.n, a.x, a.ldx, a.kernel, a.ldk, a.dy, a.lddy, a.save, a.dx, a.lddx, a.dkernel, a.dbias, a.workspace};
}
NormBwd norm_bwd_of(const nerfds_layer_norm_backward_args& a) {
  return NormBwd{a.dtype, a.m, a.d, a.x, a.ldx, a.scale, a.dy, a.lddy, a.stats, a.dx, a.lddx, a.dscale, a.dbias, static_cast<float*>(a.workspace)};
}
int check_norm(const char* who, int32_t dtype, int64_t m, int32_t d) {
  if (dtype < F32 || dtype > BF16) return fail(NERFDS_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (m < 0 || m > MAX_ROWS || d < 1 || d > MAX_WIDTH) return fail(NERFDS_EINVAL, "%s: m = %lld, d = %d (0 <= m <= 2^40, 1 <= d <= 2^24)", who, (long long)m, d);
  return NERFDS_OK;
}

#define CHECK(call) do { const int rc_ = (call); if (rc_ != NERFDS_OK) return rc_; } while (0)
#define ON_DEVICE(who, device)                                                                                              \
  Device guard(device);                                                                                                     \
  const int cus = guard.ok ? num_cus(device) : 0;                                                                           \
  if (cus == 0) return fail(NERFDS_EDEVICE, "%s: no such HIP device %d (there is no CPU fallback)", who, device)

}  // namespace

extern "C" {

int64_t nerfds_dense_save_bytes(int32_t dtype, int32_t activation, int64_t m, int32_t n) {
  CHECK(check_dense("nerfds_dense_save_bytes", dtype, activation, m, 1, n));
  return (int64_t)dense_save_bytes(dtype, activation, m, n);
}

int64_t nerfds_dense_forward_workspace(int device, const nerfds_dense_forward_args* a) {
  const char* who = "nerfds_dense_forward_workspace";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_dense(who, a->dtype, a->activation, a->m, a->k, a->n));
  const int cus = num_cus(device);
  if (cus == 0) return fail(NERFDS_EDEVICE, "%s: no such HIP device %d", who, device);
  return (int64_t)dense_fwd_ws(dense_fwd_of(*a), cus);
}

int nerfds_dense_forward(int device, const nerfds_dense_forward_args* a, void* hip_stream) {
  const char* who = "nerfds_dense_forward";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_dense(who, a->dtype, a->activation, a->m, a->k, a->n));
  if (a->m == 0) return NERFDS_OK;
  CHECK(check_array(who, "x", a->x, a->dtype, a->ldx, a->k));
  CHECK(check_array(who, "kernel", a->kernel, a->dtype, a->ldk, a->n));
  CHECK(check_array(who, "y", a->y, a->dtype, a->ldy, a->n));
  CHECK(check_vector(who, "bias", a->bias, a->dtype));
  if (a->residual) CHECK(check_array(who, "residual", a->residual, a->dtype, a->ldr == 0 ? a->n : a->ldr, a->n));
  CHECK(check_vector(who, "save", a->save, a->activation == ACT_RELU ? F16 : a->dtype));
  ON_DEVICE(who, device);
  const DenseFwd f = dense_fwd_of(*a);
  if (a->workspace) CHECK(check_workspace(who, a->workspace, a->workspace_bytes, (int64_t)dense_fwd_ws(f, cus)));
  dense_forward(static_cast<hipStream_t>(hip_stream), f, cus);
  return launched(who);
}

int64_t nerfds_dense_backward_workspace(int device, const nerfds_dense_backward_args* a) {
  const char* who = "nerfds_dense_backward_workspace";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_dense(who, a->dtype, a->activation, a->m, a->k, a->n));
  const int cus = num_cus(device);
  if (cus == 0) return fail(NERFDS_EDEVICE, "%s: no such HIP device %d", who, device);
  return a->m == 0 ? 0 : (int64_t)dense_bwd_ws(dense_bwd_of(*a), cus);
}

int nerfds_dense_backward(int device, const nerfds_dense_backward_args* a, void* hip_stream) {
  const char* who = "nerfds_dense_backward";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_dense(who, a->dtype, a->activation, a->m, a->k, a->n));
  CHECK(check_vector(who, "dkernel", a->dkernel, a->dtype));
  CHECK(check_vector(who, "dbias", a->dbias, a->dtype));
  if (a->m > 0) {
    CHECK(check_array(who, "x", a->x, a->dtype, a->ldx, a->k));
    CHECK(check_array(who, "kernel", a->kernel, a->dtype, a->ldk, a->n));
    CHECK(check_array(who, "dy", a->dy, a->dtype, a->lddy, a->n));
    if (a->dx) CHECK(check_array(who, "dx", a->dx, a->dtype, a->lddx, a->k));
    if (a->activation != ACT_NONE && !a->save) return fail(NERFDS_EINVAL, "%s: this activation needs what the forward saved", who);
    CHECK(check_vector(who, "save", a->save, a->activation == ACT_RELU ? F16 : a->dtype));
  }
  ON_DEVICE(who, device);
  const DenseBwd w = dense_bwd_of(*a);
  if (a->m > 0) CHECK(check_workspace(who, a->workspace, a->workspace_bytes, (int64_t)dense_bwd_ws(w, cus)));
  dense_backward(static_cast<hipStream_t>(hip_stream), w, cus);
  return launched(who);
}

int nerfds_layer_norm_forward(int device, const nerfds_layer_norm_forward_args* a, void* hip_stream) {
  const char* who = "nerfds_layer_norm_forward";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_norm(who, a->dtype, a->m, a->d));
  if (!(a->epsilon >= 0.f) || isinf(a->epsilon)) return fail(NERFDS_EINVAL, "%s: epsilon must be finite and >= 0", who);
  if (a->m == 0) return NERFDS_OK;
  CHECK(check_array(who, "x", a->x, a->dtype, a->ldx, a->d));
  CHECK(check_array(who, "y", a->y, a->dtype, a->ldy, a->d));
  CHECK(check_vector(who, "scale", a->scale, a->dtype));
  CHECK(check_vector(who, "bias", a->bias, a->dtype));
  CHECK(check_vector(who, "stats", a->stats, F32));
  ON_DEVICE(who, device);
  norm_forward(static_cast<hipStream_t>(hip_stream), NormFwd{a->dtype, a->m, a->d, a->epsilon, a->x, a->ldx, a->scale, a->bias, a->y, a->ldy, a->stats}, cus);
  return launched(who);
}

int64_t nerfds_layer_norm_backward_workspace(int device, const nerfds_layer_norm_backward_args* a) {
  const char* who = "nerfds_layer_norm_backward_workspace";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_norm(who, a->dtype, a->m, a->d));
  const int cus = num_cus(device);
  if (cus == 0) return fail(NERFDS_EDEVICE, "%s: no such HIP device %d", who, device);
  return a->m == 0 ? 0 : (int64_t)norm_bwd_ws(norm_bwd_of(*a), cus);
}

int nerfds_layer_norm_backward(int device, const nerfds_layer_norm_backward_args* a, void* hip_stream) {
  const char* who = "nerfds_layer_norm_backward";
  if (!a) return fail(NERFDS_EINVAL, "%s: null argument", who);
  CHECK(check_norm(who, a->dtype, a->m, a->d));
  CHECK(check_vector(who, "scale", a->scale, a->dtype));
  CHECK(check_vector(who, "dscale", a->dscale, a->dtype));
  CHECK(check_vector(who, "dbias", a->dbias, a->dtype));
  if (a->m > 0) {
    CHECK(check_array(who, "x", a->x, a->dtype, a->ldx, a->d));
    CHECK(check_array(who, "dy", a->dy, a->dtype, a->lddy, a->d));
    if (a->dx) CHECK(check_array(who, "dx", a->dx, a->dtype, a->lddx, a->d));
    if (!a->stats || !aligned_to(a->stats, 4)) return fail(NERFDS_EINVAL, "%s: stats of the forward are needed", who);
  }
  ON_DEVICE(who, device);
  const NormBwd w = norm_bwd_of(*a);
  if (a->m > 0) CHECK(check_workspace(who, a->workspace, a->workspace_bytes, (int64_t)norm_bwd_ws(w, cus)));
  norm_backward(static_cast<hipStream_t>(hip_stream), w, cus);
  return launched(who);
}

static int check_matrices(const char* who, const nerfds_matrix* mats, int32_t count) {
  if (count < 0 || (count > 0 && !mats)) return fail(NERFDS_EINVAL, "%s: %d matrices at %p", who, count, (const void*)mats);
  for (int32_t i = 0; i < count; ++i)
    if (mats[i].rows < 1 || mats[i].cols < 1 || mats[i].rows > NERFDS_ORTHO_MAX_DIM || mats[i].cols > NERFDS_ORTHO_MAX_DIM)
      return fail(NERFDS_EINVAL, "%s: matrix %d is %d x %d (1 .. %d each)", who, i, mats[i].rows, mats[i].cols, NERFDS_ORTHO_MAX_DIM);
  return NERFDS_OK;
}

// (nerfds_matrix and OrthoMat have one layout: the list is handed down as it is)
static_assert(sizeof(nerfds_matrix) == sizeof(OrthoMat) && offsetof(nerfds_matrix, o) == offsetof(OrthoMat, o) && offsetof(nerfds_matrix, ldo) == offsetof(OrthoMat, ldo) &&
              offsetof(nerfds_matrix, rows) == offsetof(OrthoMat, rows) && offsetof(nerfds_matrix, cols) == offsetof(OrthoMat, cols), "layout");
static const OrthoMat* list_of(const nerfds_matrix* m) { return reinterpret_cast<const OrthoMat*>(m); }

int64_t nerfds_orthogonalize_workspace(const nerfds_matrix* matrices, int32_t count) {
  CHECK(check_matrices("nerfds_orthogonalize_workspace", matrices, count));
  return (int64_t)ortho_ws(list_of(matrices), count);
}

int nerfds_orthogonalize(int device, int32_t dtype, const nerfds_matrix* matrices, int32_t count, int32_t steps, void* workspace, int64_t workspace_bytes,
                         void* hip_stream) {
  const char* who = "nerfds_orthogonalize";
  if (dtype < F32 || dtype > BF16) return fail(NERFDS_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (steps < 1 || steps > 16) return fail(NERFDS_EINVAL, "%s: steps = %d (1 .. 16)", who, steps);
  CHECK(check_matrices(who, matrices, count));
  if (count == 0) return NERFDS_OK;
  for (int32_t i = 0; i < count; ++i) {
    CHECK(check_array(who, "u", matrices[i].u, dtype, matrices[i].ldu, matrices[i].cols));
    CHECK(check_array(who, "o", matrices[i].o, dtype, matrices[i].ldo, matrices[i].cols));
  }
  CHECK(check_workspace(who, workspace, workspace_bytes, (int64_t)ortho_ws(list_of(matrices), count)));
  ON_DEVICE(who, device);
  orthogonalize(static_cast<hipStream_t>(hip_stream), dtype, list_of(matrices), count, steps, workspace);
  return launched(who);
}

}  // extern "C"
