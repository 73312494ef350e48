// What the C-ABI files of the transformer operators share (op_api.cu, attention_api.cu): the plan, checks of arguments, and the order of
// a plan's calls in its workspace.
#pragma once
#include <cstdint>

#include "../../include/euler_b200.h"
#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

int op_fail(int code, const char *fmt, ...);       // keeps the message and logs it

#define OP_TRY(expr)                                                                                                   \
  do {                                                                                                                 \
    cudaError_t e__ = (expr);                                                                                          \
    if (e__ != cudaSuccess) {                                                                                          \
      cudaGetLastError();                                                                                              \
      return op_fail(ELB_GENERAL_ERROR, "CUDA error %s at %s:%d (%s)", cudaGetErrorName(e__), __FILE__, __LINE__,      \
                     cudaGetErrorString(e__));                                                                         \
    }                                                                                                                  \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) { prev = -1; return; }
    if (prev == dev) prev = -1;
    else if (cudaSetDevice(dev) != cudaSuccess) prev = -1;
  }
  ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

enum Kind { LINEAR, NORM, ROUTE, EXPERTS, ROTARY, APPEND, ATTENTION };
constexpr int64_t MAX_ROWS = (1ll << 31) - 4096;
constexpr int MAX_OLD = 40;       // workspaces that a plan has outgrown

inline int et_of(int dt) { return dt == ELB_F32 ? ET_F32 : dt == ELB_BF16 ? ET_BF16 : dt == ELB_F16 ? ET_F16 : -1; }
inline size_t et_bytes(int et) { return et == ET_F32 ? 4 : 2; }
inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int *take_status();
void put_status(int *p);
// A plan of a device (-1: the current one) without its description; and whether `op` is a kind's own plan
int make_op(Kind kind, int device, elb_op **out);
int check_op(const elb_op *op, Kind kind);

}  // namespace elb

struct elb_op {
  elb::Kind kind;
  int device = 0, num_sms = 0, max_pairs = 0;
  bool prepared = false;
  uint64_t launches = 0, bytes = 0;
  int *h_status = nullptr, *d_status = nullptr;
  // Orders the calls of a plan with workspace across streams.
  cudaEvent_t done = nullptr;
  unsigned long long last = 0;      // the last call's stream, by its id
  bool pending = false;
  union {                           // the description; its kind's create sets it
    elb_linear_desc_t lin = {};
    elb_norm_desc_t norm;
    elb_route_desc_t route;
    elb_experts_desc_t exp;
    elb_rotary_desc_t rot;
    elb_append_desc_t app;
    elb_attention_desc_t att;
  };
  void *w[2] = {};            // packed weights: of the product, or into and out of the experts; the angles' steps
  float *f[4] = {};           // bias, or the norms' weights and biases
  void *ws = nullptr;         // the experts' workspace, that of a product for inputs that are not aligned, or attention's partial results
  size_t ws_bytes = 0;
  void *old[elb::MAX_OLD] = {};    // workspaces that have become too small
  int n_old = 0;
  elb::ExpertsParams ep = {};
  bool count_stale = false;   // a call's launches failed half way and the experts' counts could not be cleared behind them
  void *mid = nullptr;
  int64_t pitch_mid = 0;

  explicit elb_op(elb::Kind k) : kind(k) {}
  ~elb_op() {
    elb::DeviceGuard guard(device);
    for (void *q : w) if (q) cudaFree(q);
    for (float *q : f) if (q) cudaFree(q);
    for (int i = 0; i < n_old; ++i) cudaFree(old[i]);
    if (ws) cudaFree(ws);
    if (done) cudaEventDestroy(done);
    elb::put_status(h_status);       // (behind the cudaFree above, which has waited for the plan's kernels)
  }
};

namespace elb {

template <typename T>
int alloc(elb_op &op, T **p, size_t bytes) {
  void *q = nullptr;
  OP_TRY(cudaMalloc(&q, bytes));
  *p = static_cast<T *>(q);
  op.bytes += bytes;
  return ELB_OK;
}

// A tensor of the caller's, in host memory or on any device, as memory of the plan's device (the current one) for the time of a preparation.
struct Staged {
  const void *p = nullptr;
  void *own = nullptr;
  ~Staged() { if (own) cudaFree(own); }
  int take(const elb_op &op, const void *src, size_t bytes) {
    cudaPointerAttributes a = {};
    const bool known = cudaPointerGetAttributes(&a, src) == cudaSuccess;
    if (known && (a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == op.device))) {
      p = src;
      return ELB_OK;
    }
    cudaGetLastError();
    if (known && a.type == cudaMemoryTypeDevice) {     // whatever stream of that device it comes from
      DeviceGuard guard(a.device);
      OP_TRY(cudaDeviceSynchronize());
    }
    OP_TRY(cudaMalloc(&own, bytes));
    OP_TRY(cudaMemcpy(own, src, bytes, cudaMemcpyDefault));
    p = own;
    return ELB_OK;
  }
};

inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int check_call(const elb_op &op, int64_t rows) {
  if (!op.prepared) return op_fail(ELB_GENERAL_ERROR, "the plan is not prepared");
  if (rows < 0 || rows > MAX_ROWS) return op_fail(ELB_GENERAL_ERROR, "%lld rows", (long long)rows);
  return ELB_OK;
}

inline int check_ld(const char *what, int64_t &ld, int64_t dense) {
  if (ld == 0) ld = dense;
  if (ld < dense || ld > (1ll << 40)) return op_fail(ELB_GENERAL_ERROR, "%s rows of %lld elements lie %lld apart", what, (long long)dense, (long long)ld);
  return ELB_OK;
}

inline bool finite(float v) { return v - v == 0.0f; }

// The plan's workspace may still be in use by its last call, on another stream.  Streams are told apart by their ids: cudaStreamPerThread is one
// handle for a stream of each thread, and a destroyed stream's handle may come back while its work still runs.
// A call that fails half way has launched kernels that use it all the same: whatever way the call ends, its last launch is noted.
class WorkspaceCall {
 public:
  bool capturing = false;
  WorkspaceCall(elb_op &op, cudaStream_t s) : op_(op), s_(s) {}
  int enter() {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    OP_TRY(cudaStreamIsCapturing(s_, &st));
    capturing = st != cudaStreamCaptureStatusNone;
    if (capturing) return ELB_OK;
    unsigned long long id = 0;
    OP_TRY(cudaStreamGetId(s_, &id));
    if (op_.pending && op_.last != id) OP_TRY(cudaStreamWaitEvent(s_, op_.done, 0));
    op_.last = id;
    inside_ = true;
    return ELB_OK;
  }
  int leave() {
    if (!inside_) return ELB_OK;
    inside_ = false;
    OP_TRY(cudaEventRecord(op_.done, s_));
    op_.pending = true;
    return ELB_OK;
  }
  ~WorkspaceCall() { if (inside_ && cudaEventRecord(op_.done, s_) == cudaSuccess) op_.pending = true; }

 private:
  elb_op &op_;
  cudaStream_t s_;
  bool inside_ = false;
};

}  // namespace elb
