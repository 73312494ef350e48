// The preparation of the rotary plans (csrc/attention_api.cu) on a CPU, with stand-ins for the CUDA runtime: what a GPU test could only meet by chance
// is that a copy is still on its way when prepare returns, or starts before its source has been written.  Built by tests/test_attention_plan_cpu.py.
//
// A copy from pageable memory may return when its source has been read and end later: it is over when its device has been waited for.  Memory of a device holds
// what its streams have written once that device has been waited for.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

#include "attention.cuh"
#include "op_plan.cuh"

#ifndef __CUDA_ARCH__       // (host code alone)
using namespace elb;

namespace {

int g_bad = 0, g_device = 0;
void need(bool ok, const char *what) {
  if (ok) return;
  ++g_bad;
  std::printf("%s\n", what);
}
std::map<const void *, int> g_on_device;                      // device memory and where it lies
std::map<int, int> g_writing, g_copying;                      // works of a device that are not known to be over: kernels that write frequencies, copies

}  // namespace

// ------------------------------------------------------------------------------------------- the CUDA runtime
extern "C" {
void **__cudaRegisterFatBinary(void *) { static void *p; return &p; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
cudaError_t cudaGetDevice(int *d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { g_device = d; return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { g_writing[g_device] = g_copying[g_device] = 0; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char *cudaGetErrorName(cudaError_t) { return "error"; }
const char *cudaGetErrorString(cudaError_t) { return "stand-in"; }
cudaError_t cudaMalloc(void **p, size_t n) { *p = malloc(n < 64 ? 64 : n); g_on_device[*p] = g_device; return cudaSuccess; }
cudaError_t cudaFree(void *p) { g_on_device.erase(p); free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, cudaMemcpyKind) {
  auto from = g_on_device.find(s);
  if (from != g_on_device.end()) need(g_writing[from->second] == 0, "frequencies are read before their device has been waited for");
  if (g_on_device.count(d)) ++g_copying[g_on_device[d]];
  memcpy(d, s, n);
  return cudaSuccess;
}
cudaError_t cudaMemset(void *p, int v, size_t n) { memset(p, v, n); return cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes *a, const void *p) {
  memset(a, 0, sizeof(*a));
  auto i = g_on_device.find(p);
  a->type = i == g_on_device.end() ? cudaMemoryTypeUnregistered : cudaMemoryTypeDevice;
  a->device = i == g_on_device.end() ? -2 : i->second;
  return cudaSuccess;
}
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamWaitEvent(cudaStream_t, cudaEvent_t, unsigned) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus *st) { *st = cudaStreamCaptureStatusNone; return cudaSuccess; }
cudaError_t cudaStreamGetId(cudaStream_t, unsigned long long *id) { *id = 1; return cudaSuccess; }
}

// ------------------------------------------------------------------------------------------- what attention_api.cu calls
namespace elb {
int op_fail(int code, const char *, ...) { return code; }
int *take_status() { return nullptr; }
void put_status(int *) {}
int make_op(Kind kind, int device, elb_op **out) {
  *out = new elb_op(kind);
  (*out)->device = device;
  (*out)->num_sms = 148;
  return ELB_OK;
}
int check_op(const elb_op *op, Kind kind) { return op && op->kind == kind ? ELB_OK : ELB_GENERAL_ERROR; }
cudaError_t init_attention() { return cudaSuccess; }
cudaError_t init_attention_prompt() { return cudaSuccess; }
bool attention_token_takes(const AttentionParams &) { return false; }
bool attention_prompt_takes(const AttentionParams &) { return false; }
cudaError_t launch_attention_token(const AttentionParams &, const AttentionWorkspace &, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_attention_prompt(const AttentionParams &, const AttentionWorkspace &, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_attention_any(const AttentionParams &, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_rotary(const RotaryParams &, cudaStream_t) { return cudaSuccess; }
}  // namespace elb

namespace {

elb_rotary_desc_t rotary(int device) {
  elb_rotary_desc_t d = {};
  d.heads = d.kv_heads = 2; d.head_dim = d.rotary_dim = 16; d.dt = ELB_BF16; d.base = 10000.0f; d.magnitude = 1.0f; d.device = device;
  return d;
}

// where: the device of the frequencies, -1 the host, -2 none
void prepare(int where, int current) {
  float buf[8];
  for (int i = 0; i < 8; ++i) buf[i] = 1.0f / (i + 1);
  g_on_device.clear();
  if (where >= 0) g_on_device[buf] = where;
  const float *f = where == -2 ? nullptr : buf;
  for (bool append : {false, true}) {
    g_device = current;
    elb_op_t *op = nullptr;
    elb_append_desc_t a = {};
    a.rotary = rotary(0);
    a.page_size = 16;
    need((append ? elb_append_create(&a, &op) : elb_rotary_create(&a.rotary, &op)) == ELB_OK, "create");
    if (where >= 0) g_writing[where] = 1;                      // on a stream that no copy waits for
    need((append ? elb_append_prepare(op, f) : elb_rotary_prepare(op, f)) == ELB_OK, "prepare");
    need(g_copying[0] == 0 && g_copying[1] == 0, "prepare returns while its copies may be on their way");
    need(g_device == current, "the current device has changed");
    delete op;
  }
  g_on_device.erase(buf);
  need(g_on_device.empty(), "memory was not freed");
}

}  // namespace

int main() {
  for (int where : {-2, -1, 0, 1})
    for (int current : {0, 1}) prepare(where, current);
  if (g_bad == 0) std::printf("ok\n");
  return g_bad != 0;
}
#endif
