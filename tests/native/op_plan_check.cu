// The host side of the transformer operators (csrc/op_api.cu) on a CPU: the CUDA runtime and the kernels' launches are stand-ins that keep
// a log, so that what no GPU test may provoke (a launch that fails half way, weights on another GPU) and what it could only meet by
// chance (two calls in one workspace at once) can be looked at.  Built by tests/test_op_plan_cpu.py with op_api.cu itself.
//
// A stand-in stream is an id; the handle a caller passes stands for one, which may change (cudaStreamPerThread in another thread, the
// handle of a destroyed stream).  knows[a][b]: the works of stream b that are over before stream a's next one starts.
#include <cstdio>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "../../include/euler_b200.h"
#include "ops.cuh"

#ifndef __CUDA_ARCH__       // (host code alone)
using namespace elb;

namespace {

int g_bad = 0;
void need(bool ok, const char *what) {
  if (ok) return;
  ++g_bad;
  std::printf("%s\n", what);
}

struct Stream { int works = 0; std::map<unsigned long long, int> knows; };
std::map<unsigned long long, Stream> g_streams;               // by id
std::map<cudaStream_t, unsigned long long> g_ids;             // the id a handle has now
std::map<cudaEvent_t, std::map<unsigned long long, int>> g_events;
std::set<cudaStream_t> g_capturing;
std::map<unsigned long long, int> g_users;                    // the last work of each stream in the plan's workspace
std::string g_fail, g_fail_too;                               // the launches that fail
int g_device = 0;
std::map<const void *, int> g_on_device;                      // device pointers of the caller's, and where they lie
std::map<int, int> g_waits;                                   // cudaDeviceSynchronize per device
bool g_counts_dirty = false;                                  // the experts' counts
const void *g_counts = nullptr;
std::vector<std::string> g_log;
unsigned long long id_of(cudaStream_t s) {
  auto i = g_ids.find(s);
  return i == g_ids.end() ? reinterpret_cast<unsigned long long>(s) : i->second;
}

// a kernel on s that uses the plan's workspace: everything other streams did there has to be over
cudaError_t work(const char *name, cudaStream_t s) {
  g_log.push_back(name);
  if (g_fail == name) return cudaErrorInvalidValue;
  if (g_capturing.count(s)) return cudaSuccess;
  const auto id = id_of(s);
  Stream &st = g_streams[id];
  ++st.works;
  for (auto &u : g_users)
    if (u.first != id && st.knows[u.first] < u.second) {
      std::printf("%s on stream %llu: work %d of stream %llu may still use the workspace\n", name, id, u.second, u.first);
      ++g_bad;
    }
  g_users[id] = st.works;
  return cudaSuccess;
}

}  // namespace

// ------------------------------------------------------------------------------------------- the CUDA runtime
extern "C" {
void **__cudaRegisterFatBinary(void *) { static void *p; return &p; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
cudaError_t cudaGetDeviceCount(int *n) { *n = 2; return cudaSuccess; }
cudaError_t cudaGetDevice(int *d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { g_device = d; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int *v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { ++g_waits[g_device]; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char *cudaGetErrorName(cudaError_t) { return "error"; }
const char *cudaGetErrorString(cudaError_t) { return "stand-in"; }
cudaError_t cudaMalloc(void **p, size_t n) { *p = malloc(n < 64 ? 64 : n); g_on_device[*p] = g_device; return *p ? cudaSuccess : cudaErrorMemoryAllocation; }
cudaError_t cudaFree(void *p) { g_on_device.erase(p); free(p); return cudaSuccess; }
cudaError_t cudaHostAlloc(void **p, size_t n, unsigned) { *p = malloc(n); return cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void **d, void *h, unsigned) { *d = h; return cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, cudaMemcpyKind) { memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemset(void *p, int v, size_t n) { memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void *p, int, size_t, cudaStream_t s) {
  g_log.push_back("memset");
  if (g_fail == "memset" || g_fail_too == "memset") return cudaErrorInvalidValue;
  if (p == g_counts && !g_capturing.count(s)) g_counts_dirty = false;
  return cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes *a, const void *p) {
  memset(a, 0, sizeof(*a));
  auto i = g_on_device.find(p);
  a->type = i == g_on_device.end() ? cudaMemoryTypeUnregistered : cudaMemoryTypeDevice;
  a->device = i == g_on_device.end() ? -2 : i->second;
  return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *e, unsigned) { static size_t n = 0; *e = reinterpret_cast<cudaEvent_t>(++n); return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) {
  const auto id = id_of(s);
  g_events[e] = g_streams[id].knows;
  g_events[e][id] = g_streams[id].works;
  return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) {
  g_log.push_back("wait");
  Stream &st = g_streams[id_of(s)];
  for (auto &k : g_events[e]) if (st.knows[k.first] < k.second) st.knows[k.first] = k.second;
  return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus *st) {
  *st = g_capturing.count(s) ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
cudaError_t cudaStreamGetId(cudaStream_t s, unsigned long long *id) { *id = id_of(s); return cudaSuccess; }
int elb_device_supported(int) { return ELB_OK; }
}

// ------------------------------------------------------------------------------------------- the kernels
namespace elb {
int report_failure(int code, const char *) { return code; }
cudaError_t init_gemm(int, int *pairs) { *pairs = 74; return cudaSuccess; }
bool gemm_wants_gemv(long long rows, int, int) { return rows <= 1; }
bool experts_want_gemv(int slots, int, double) { return slots <= 4; }
bool experts_count_here(int slots) { return slots <= 2048; }
int grouped_tile_tokens(int, int) { return 64; }
// what a preparation's kernel reads has to lie on the plan's device
static cudaError_t reads(const void *src) {
  auto i = g_on_device.find(src);
  need(!src || (i != g_on_device.end() && i->second == g_device), "a preparation's kernel reads memory that is not its device's");
  return cudaSuccess;
}
cudaError_t launch_pack_weights(void *, const void *src, int, int, int, bool, bool, cudaStream_t) { return reads(src); }
cudaError_t launch_pack_bias(float *, const void *src, int, int, int, bool, cudaStream_t) { return reads(src); }
cudaError_t launch_norm_vector(float *, const void *src, int, int, long long, float, cudaStream_t) { return reads(src); }
cudaError_t launch_gemm(const GemmParams &, cudaStream_t s) { return work("gemm", s); }
cudaError_t launch_gemv(const GemmParams &, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_align_rows(void *, long long, const void *, long long, int, int, cudaStream_t s) { return work("align", s); }
cudaError_t launch_gemv_experts(const GemmParams &, const GemmParams &, const int *, const float *, int, int, int, cudaStream_t s) { return work("gemv", s); }
cudaError_t launch_experts_count(const ExpertsParams &p, cudaStream_t s) {
  g_counts = p.count;
  if (!g_capturing.count(s)) {
    need(!g_counts_dirty, "a call counts its slots on top of an earlier call's");
    g_counts_dirty = true;
  }
  return work("count", s);
}
cudaError_t launch_experts_gather(const ExpertsParams &, int, cudaStream_t s) { return work("gather", s); }
cudaError_t launch_experts_combine(const ExpertsParams &p, cudaStream_t s) {
  const cudaError_t e = work("combine", s);
  if (e == cudaSuccess && p.clear && !g_capturing.count(s)) g_counts_dirty = false;
  return e;
}
cudaError_t launch_block_norm(const NormParams &, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_route(const RouteParams &, cudaStream_t) { return cudaSuccess; }
}  // namespace elb

namespace {

char g_tensor[256];                       // never read or written here
cudaStream_t handle(size_t n) { return reinterpret_cast<cudaStream_t>(n); }

// a plan whose calls use its workspace: rows of 333 channels cannot be read by a tiled copy
struct Linear {
  elb_op_t *op = nullptr;
  Linear() {
    elb_linear_desc_t d = {};
    d.ic = 333; d.oc = 64; d.dt_input = d.dt_output = ELB_BF16; d.dt_bias = ELB_F32; d.fmt_weights = ELB_OIHW; d.scale = 1.0f; d.device = 0;
    need(elb_linear_create(&d, &op) == ELB_OK, "create");
    std::vector<char> w(333 * 64 * 2);
    need(elb_linear_prepare(op, w.data(), nullptr) == ELB_OK, "prepare");
  }
  ~Linear() { elb_op_destroy(op); }
  int call(size_t stream) { return elb_linear_enqueue(op, g_tensor, g_tensor, nullptr, 100, handle(stream)); }
};
struct Experts {
  elb_op_t *op = nullptr;
  Experts() {
    elb_experts_desc_t d = {};
    d.experts = 8; d.top_k = 2; d.ic = 64; d.mid = 64; d.dt = ELB_BF16; d.device = 0; d.max_rows = 2000;
    need(elb_experts_create(&d, &op) == ELB_OK, "create");
    std::vector<char> w(8 * 64 * 64 * 2);
    need(elb_experts_prepare(op, w.data(), w.data()) == ELB_OK, "prepare");
  }
  ~Experts() { elb_op_destroy(op); }
  int call(size_t stream, int rows = 1500) {
    return elb_experts_enqueue(op, g_tensor, g_tensor, reinterpret_cast<int *>(g_tensor), reinterpret_cast<float *>(g_tensor), rows, handle(stream));
  }
};

// Calls on streams that have different handles
template <typename Plan>
void streams() {
  Plan p;
  for (size_t s : {5, 5, 6, 7, 5, 0, 6}) need(p.call(s) == ELB_OK, "call");
}
// One handle for two streams: cudaStreamPerThread in two threads, or a new stream that was given a destroyed one's handle
template <typename Plan>
void one_handle() {
  Plan p;
  for (unsigned long long id : {21, 22, 22, 21, 23}) {
    g_ids[handle(2)] = id;
    need(p.call(2) == ELB_OK, "call");
  }
}

// A call whose launch fails half way leaves kernels in flight that use the workspace: a call on another stream comes behind them.
template <typename Plan>
void failed(std::vector<std::string> launches) {
  Plan p;
  need(p.call(5) == ELB_OK, "call");
  for (const std::string &l : launches) {
    g_fail = l;
    need(p.call(6) != ELB_OK, "a call whose launch failed");
    g_fail.clear();
    need(p.call(7) == ELB_OK, "the call behind a failed one");
  }
}

// The experts' counts are zero when a call begins to count, whatever came before: calls that failed behind the counting, captured calls in
// between (which run later, or never), and calls of few slots, which count elsewhere.
void counts() {
  for (const char *launch : {"gather", "gemm", "combine"})
    for (bool memset_fails : {false, true}) {
      Experts p;
      need(p.call(5) == ELB_OK && p.call(5, 10) == ELB_OK && p.call(5) == ELB_OK, "calls");
      g_fail = launch;
      if (!memset_fails) {
        need(p.call(5) != ELB_OK, "a call whose launch failed");
        g_fail.clear();
        need(!g_counts_dirty, "a failed call leaves counts behind that a captured call adds to");
      } else {
        g_fail_too = "memset";
        need(p.call(5) != ELB_OK, "a call whose launch failed, and the clearing behind it");
        g_fail = "memset";
        g_fail_too.clear();
        need(p.call(5) != ELB_OK, "a call that could not clear the counts");
        g_fail.clear();
      }
      g_capturing.insert(handle(6));
      g_log.clear();
      need(p.call(6) == ELB_OK, "a captured call");
      need(!memset_fails || g_log[0] == "memset", "a captured call behind counts that are not zero clears them");
      g_capturing.clear();
      need(p.call(5) == ELB_OK, "the call behind them");
      need(p.call(7) == ELB_OK && !g_counts_dirty, "calls");
      g_users.clear();
    }
  // a capture that breaks off
  Experts p;
  g_capturing.insert(handle(6));
  g_fail = "gemm";
  need(p.call(6) != ELB_OK, "a captured call whose launch failed");
  g_fail.clear();
  need(g_log.back() == "memset", "the graph of a captured call that failed clears the counts");
  g_capturing.clear();
  need(p.call(5) == ELB_OK && p.call(5) == ELB_OK, "calls");
}

// Weights on another device than the plan's: its work is waited for, and the kernels read a copy on the plan's own.
void devices() {
  std::vector<char> buf(4 * 64 * 64 * 2);
  for (int where : {1, 0, -1})                             // the other device, the plan's, the host
    for (int current : {0, 1}) {
      g_on_device.erase(buf.data());
      if (where >= 0) g_on_device[buf.data()] = where;
      g_device = current;
      g_waits.clear();
      elb_op_t *op[4] = {};
      elb_linear_desc_t l = {};
      l.ic = l.oc = 64; l.dt_input = l.dt_output = ELB_BF16; l.dt_bias = ELB_F32; l.fmt_weights = ELB_OIHW; l.with_bias = 1; l.scale = 1.0f;
      elb_norm_desc_t n = {};
      n.channels = 64; n.dt = n.dt_residual = ELB_BF16; n.dt_weights = ELB_F32; n.post = ELB_NORM_RMS; n.pre = ELB_NORM_LAYER; n.scale = 1.0f;
      elb_route_desc_t r = {};
      r.experts = 64; r.top_k = 2; r.dt_logits = ELB_F32; r.with_bias = 1; r.groups = r.top_groups = r.group_best = 1; r.scale = 1.0f;
      elb_experts_desc_t e = {};
      e.experts = 4; e.top_k = 2; e.ic = e.mid = 64; e.dt = ELB_BF16; e.max_rows = 4;
      need(elb_linear_create(&l, &op[0]) == ELB_OK && elb_norm_create(&n, &op[1]) == ELB_OK && elb_route_create(&r, &op[2]) == ELB_OK &&
           elb_experts_create(&e, &op[3]) == ELB_OK, "create");
      g_waits.clear();
      const void *b = buf.data();
      need(elb_linear_prepare(op[0], b, b) == ELB_OK, "linear");
      need(where != 1 || g_waits[1] > 0, "the weights' device was not waited for");
      need(elb_norm_prepare(op[1], b, b, b, b) == ELB_OK, "norm");
      need(elb_route_prepare(op[2], static_cast<const float *>(b)) == ELB_OK, "route");
      need(elb_experts_prepare(op[3], b, b) == ELB_OK, "experts");
      need(g_device == current, "the current device has changed");
      for (elb_op_t *o : op) elb_op_destroy(o);
      g_on_device.erase(buf.data());
      size_t left = 0;
      for (auto &m : g_on_device) left += m.first != nullptr;
      need(left == 0, "memory was not freed");
    }
}

// Every slot belongs to one block of the gather kernel, up to the most that a plan takes (2^31 - 4096).
void shares() {
  for (int warps : {8})
    for (int most : {148 * 8, 16})
      for (int slots : {1, 7, 8, 9, 1000, 9471, 9472, 9473, 12345678, 0x7FFFFFFF - 2000000, 0x7FFFFFFF - 4096, 0x7FFFF000}) {
        const SlotShare s = share_slots(slots, warps, most);
        long long at = 0;
        bool fine = s.per >= 1 && s.blocks >= 1 && s.blocks <= most;
        for (int b = 0; b < s.blocks && fine; ++b) {
          fine = s.first(b) == at && s.end(b, slots) > at;
          at = s.end(b, slots);
        }
        if (!(fine && at == slots)) std::printf("%d slots, %d blocks of %d: ", slots, s.blocks, s.per);
        need(fine && at == slots, "slots without a block of their own");
      }
}

}  // namespace

int main(int argc, char **argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "streams") { streams<Linear>(); g_users.clear(); streams<Experts>(); }
  else if (what == "one_handle") { one_handle<Linear>(); g_users.clear(); one_handle<Experts>(); }
  else if (what == "failed") { failed<Linear>({"gemm"}); g_users.clear(); failed<Experts>({"gather", "gemm", "combine"}); }
  else if (what == "counts") counts();
  else if (what == "devices") devices();
  else if (what == "shares") shares();
  else { std::printf("no such case\n"); return 2; }
  if (g_bad == 0) std::printf("ok\n");
  return g_bad != 0;
}
#endif
