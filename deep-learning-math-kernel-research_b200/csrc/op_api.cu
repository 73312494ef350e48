// C-ABI of the transformer operators (include/euler_b200.h, "Operators of transformer blocks"): descriptions are checked
// when a plan is made, weights are laid out once, and a call checks its arguments and enqueues.
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <new>

#include "op_plan.cuh"

using namespace elb;

namespace elb {

int report_failure(int code, const char *msg);      // elb_api.cu: keeps the message and logs it

int op_fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_failure(code, buf);
}

}  // namespace elb

namespace {

// What every plan of a device needs and is slow to ask for: 10 ms and more of a plan's making went into device properties, kernel
// attributes and a pinned page of its own.
struct DeviceInfo { bool known = false; int num_sms = 0, max_pairs = 0; };
constexpr int MAX_DEVICES = 64;
std::mutex g_mutex;
DeviceInfo g_devices[MAX_DEVICES];

int device_info(int device, DeviceInfo &out) {
  if (device >= MAX_DEVICES) return op_fail(ELB_UNIMPLEMENTED, "device %d", device);
  std::lock_guard<std::mutex> lock(g_mutex);
  DeviceInfo &d = g_devices[device];
  if (!d.known) {
    const int rc = elb_device_supported(device);
    if (rc != ELB_OK) return rc;
    OP_TRY(cudaDeviceGetAttribute(&d.num_sms, cudaDevAttrMultiProcessorCount, device));
    OP_TRY(init_gemm(d.num_sms, &d.max_pairs));
    d.known = true;
  }
  out = d;
  return ELB_OK;
}

// Status words of the plans, in pages of mapped host memory that stay for the next plans.
constexpr int PAGE_WORDS = 1024, MAX_PAGES = 256;
int *g_pages[MAX_PAGES];
bool g_used[MAX_PAGES][PAGE_WORDS];

}  // namespace

namespace elb {

int *take_status() {
  std::lock_guard<std::mutex> lock(g_mutex);
  for (int i = 0; i < MAX_PAGES; ++i) {
    if (!g_pages[i]) {
      void *q = nullptr;
      if (cudaHostAlloc(&q, PAGE_WORDS * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) return nullptr;
      g_pages[i] = static_cast<int *>(q);
    }
    for (int k = 0; k < PAGE_WORDS; ++k)
      if (!g_used[i][k]) {
        g_used[i][k] = true;
        g_pages[i][k] = 0;
        return &g_pages[i][k];
      }
  }
  return nullptr;
}
void put_status(int *p) {
  if (!p) return;
  std::lock_guard<std::mutex> lock(g_mutex);
  for (int i = 0; i < MAX_PAGES && g_pages[i]; ++i)
    if (p >= g_pages[i] && p < g_pages[i] + PAGE_WORDS) g_used[i][p - g_pages[i]] = false;
}

int make_op(Kind kind, int device, elb_op **out) {
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) return elb_device_supported(device);     // (says what is missing)
  if (device < 0) OP_TRY(cudaGetDevice(&device));
  if (device >= count) return elb_device_supported(device);
  DeviceGuard guard(device);
  DeviceInfo info;
  const int rc = device_info(device, info);
  if (rc != ELB_OK) return rc;
  elb_op *op = new (std::nothrow) elb_op(kind);
  if (!op) return op_fail(ELB_GENERAL_ERROR, "out of host memory");
  op->device = device;
  op->num_sms = info.num_sms;
  op->max_pairs = info.max_pairs;
  op->h_status = take_status();
  if (!op->h_status || cudaHostGetDevicePointer(reinterpret_cast<void **>(&op->d_status), op->h_status, 0) != cudaSuccess ||
      cudaEventCreateWithFlags(&op->done, cudaEventDisableTiming) != cudaSuccess) {
    cudaGetLastError();
    delete op;
    return op_fail(ELB_GENERAL_ERROR, "device allocation failed");
  }
  *out = op;
  return ELB_OK;
}

// A kind's own plan, or an error
int check_op(const elb_op *op, Kind kind) {
  if (!op) return op_fail(ELB_GENERAL_ERROR, "null plan");
  if (op->kind != kind) return op_fail(ELB_GENERAL_ERROR, "the plan is of another operator");
  return ELB_OK;
}

}  // namespace elb

namespace {

// The old workspace stays with the plan: calls in flight and captured graphs may still use it.  It at least doubles, so that there
// are few of them.
int grow_workspace(elb_op &op, size_t bytes) {
  if (bytes <= op.ws_bytes) return ELB_OK;
  if (op.ws && op.n_old == MAX_OLD) return op_fail(ELB_GENERAL_ERROR, "the workspace has grown too often");
  const size_t want = bytes > 2 * op.ws_bytes ? bytes : 2 * op.ws_bytes;
  void *q = nullptr;
  OP_TRY(cudaMalloc(&q, want));
  if (op.ws) op.old[op.n_old++] = op.ws;
  op.bytes += want;
  op.ws = q;
  op.ws_bytes = want;
  return ELB_OK;
}

// Weights [experts][rows][ic] -> packed image
int pack(elb_op &op, void **dst, const void *src, int experts, int64_t rows, int ic, bool gated, bool hwio) {
  Staged st;
  int rc = st.take(op, src, (size_t)experts * rows * ic * 2);
  if (rc != ELB_OK) return rc;
  const size_t bytes = (size_t)experts * (up(packed_rows(gated ? rows / 2 : rows, gated), GT_ROWS) / GT_ROWS) * (up(ic, GT_K) / GT_K) * GT_BYTES;
  rc = alloc(op, dst, bytes);
  if (rc != ELB_OK) return rc;
  OP_TRY(launch_pack_weights(*dst, st.p, experts, (int)rows, ic, gated, hwio, nullptr));
  OP_TRY(cudaDeviceSynchronize());
  return ELB_OK;
}

int vector_f32(elb_op &op, float **dst, const void *src, int et, int n, int padded, bool gated) {
  Staged st;
  int rc = st.take(op, src, n * et_bytes(et));
  if (rc != ELB_OK) return rc;
  rc = alloc(op, dst, (size_t)padded * 4);
  if (rc != ELB_OK) return rc;
  OP_TRY(launch_pack_bias(*dst, st.p, et, n, padded, gated, nullptr));
  OP_TRY(cudaDeviceSynchronize());
  return ELB_OK;
}

int64_t norm_pitch(int n) { return up(n + 16, 8); }

// A norm's weights as fp32, offset included; null: ones (offset and all), or no vector for a bias
int norm_vector(elb_op &op, float **dst, const void *src, int et, int n, float offset) {
  Staged st;
  int rc = src ? st.take(op, src, n * et_bytes(et)) : ELB_OK;
  if (rc == ELB_OK) rc = alloc(op, dst, (size_t)norm_pitch(n) * 8 * 4);
  if (rc != ELB_OK) return rc;
  OP_TRY(launch_norm_vector(*dst, st.p, et, n, norm_pitch(n), offset, nullptr));
  OP_TRY(cudaDeviceSynchronize());
  return ELB_OK;
}

// What a failed preparation has allocated goes, so that it can be repeated.
int drop(elb_op &op, int rc) {
  if (rc == ELB_OK) { op.prepared = true; return rc; }
  cudaGetLastError();
  for (void *&q : op.w) if (q) { cudaFree(q); q = nullptr; }
  for (float *&q : op.f) if (q) { cudaFree(q); q = nullptr; }
  op.bytes = op.ws_bytes;       // (a plan that is not prepared has made no call: no older workspaces)
  return rc;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------------------- linear
int elb_linear_create(const elb_linear_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_linear_desc_t d = *desc;
  if (d.ic < 1 || d.oc < 1 || d.ic > (1 << 20) || d.oc > (1 << 20)) return op_fail(ELB_GENERAL_ERROR, "linear of %d to %d channels", d.ic, d.oc);
  if (d.dt_input != ELB_BF16 && d.dt_input != ELB_F16)
    return op_fail(ELB_UNIMPLEMENTED, "linear takes bf16 and f16 operands (fp32 and int8: a 1x1 convolution)");
  if (d.dt_output != d.dt_input && d.dt_output != ELB_F32) return op_fail(ELB_UNIMPLEMENTED, "linear writes its operands' type or fp32");
  if (d.dt_bias != ELB_F32 && d.dt_bias != d.dt_input) return op_fail(ELB_UNIMPLEMENTED, "linear takes a bias in fp32 or its operands' type");
  if (d.fmt_weights != ELB_OIHW && d.fmt_weights != ELB_HWIO) return op_fail(ELB_UNIMPLEMENTED, "linear takes oihw and hwio weights");
  if (d.activation < ELB_ACT_NONE || d.activation > ELB_ACT_SILU) return op_fail(ELB_GENERAL_ERROR, "activation %d", d.activation);
  if (!finite(d.scale)) return op_fail(ELB_GENERAL_ERROR, "scale is not finite");
  int rc = check_ld("input", d.ld_input, d.ic);
  if (rc == ELB_OK) rc = check_ld("output", d.ld_output, d.oc);
  if (rc == ELB_OK) rc = check_ld("residual", d.ld_residual, d.oc);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(LINEAR, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->lin = d;
  *out = op;
  return ELB_OK;
}

int elb_linear_prepare(elb_op_t *op, const void *weights, const void *bias) {
  int rc = check_op(op, LINEAR);
  if (rc != ELB_OK || op->prepared) return rc;
  const elb_linear_desc_t &d = op->lin;
  if (!weights || (d.with_bias && !bias)) return op_fail(ELB_GENERAL_ERROR, "weights or bias are null");
  if (!aligned(weights, 2) || (d.with_bias && !aligned(bias, et_bytes(et_of(d.dt_bias))))) return op_fail(ELB_GENERAL_ERROR, "misaligned weights or bias");
  DeviceGuard guard(op->device);
  const int rows = d.gated ? 2 * d.oc : d.oc;
  OP_TRY(cudaDeviceSynchronize());                // whatever stream the caller's tensors come from
  rc = pack(*op, &op->w[0], weights, 1, rows, d.ic, d.gated, d.fmt_weights == ELB_HWIO);
  if (rc == ELB_OK && d.with_bias) rc = vector_f32(*op, &op->f[0], bias, et_of(d.dt_bias), rows, (int)up(packed_rows(d.oc, d.gated), 2 * GT_ROWS), d.gated);
  return drop(*op, rc);
}

int elb_linear_enqueue(elb_op_t *op, void *output, const void *input, const void *residual, int64_t rows, void *cuda_stream) {
  int rc = check_op(op, LINEAR);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  if (rc != ELB_OK || rows == 0) return rc;
  const elb_linear_desc_t &d = op->lin;
  if (!output || !input || (d.with_residual && !residual)) return op_fail(ELB_GENERAL_ERROR, "null argument");
  const size_t ob = et_bytes(et_of(d.dt_output));
  if (!aligned(input, 2) || !aligned(output, ob) || (d.with_residual && !aligned(residual, ob))) return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  GemmParams p = {};
  p.w = static_cast<const uint8_t *>(op->w[0]);
  p.x = input;
  p.ld_x = d.ld_input;
  p.rows = (int)rows;
  p.ic = d.ic;
  p.kt = (int)(up(d.ic, GT_K) / GT_K);
  p.row_tiles = (int)(up(packed_rows(d.oc, d.gated), GT_ROWS) / GT_ROWS);
  p.w_rows = (long long)p.row_tiles * p.kt * GT_ROWS;
  p.in_et = et_of(d.dt_input);
  p.num_sms = op->num_sms;
  p.max_pairs = op->max_pairs;
  p.status = op->d_status;
  p.epi.out = output;
  p.epi.res = d.with_residual ? residual : nullptr;
  p.epi.bias = op->f[0];
  p.epi.ld_out = d.ld_output;
  p.epi.ld_res = d.ld_residual;
  p.epi.oc = d.oc;
  p.epi.act = d.activation;
  p.epi.gated = d.gated;
  p.epi.out_et = et_of(d.dt_output);
  p.epi.scale = d.scale;
  const int64_t per = 16 / ob;       // elements of 16 bytes
  p.epi.words = aligned(output, 16) && d.ld_output % per == 0 && (!p.epi.res || (aligned(residual, 16) && d.ld_residual % per == 0));
  const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (gemm_wants_gemv(rows, p.row_tiles, p.kt)) {
    OP_TRY(launch_gemv(p, s));
    ++op->launches;
    return ELB_OK;
  }
  if (aligned(input, 16) && d.ld_input % 8 == 0) {
    OP_TRY(launch_gemm(p, s));
    ++op->launches;
    return ELB_OK;
  }
  // rows that a tiled copy cannot read go through the plan's workspace
  const int64_t pitch = up(d.ic, 8);
  WorkspaceCall use(*op, s);
  rc = use.enter();
  if (rc == ELB_OK) rc = grow_workspace(*op, (size_t)rows * pitch * 2);
  if (rc != ELB_OK) return rc;
  OP_TRY(launch_align_rows(op->ws, pitch, input, d.ld_input, (int)rows, d.ic, s));
  p.x = op->ws;
  p.ld_x = pitch;
  OP_TRY(launch_gemm(p, s));
  op->launches += 2;
  return use.leave();
}

// ------------------------------------------------------------------------------------------- norm
int elb_norm_create(const elb_norm_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_norm_desc_t d = *desc;
  if (d.channels < 1) return op_fail(ELB_GENERAL_ERROR, "norm of %d channels", d.channels);
  if (d.channels > 32768) return op_fail(ELB_UNIMPLEMENTED, "norm of %d channels: at most 32768", d.channels);
  if (et_of(d.dt) < 0) return op_fail(ELB_UNIMPLEMENTED, "norm takes fp32, f16 and bf16");
  if (d.dt_residual != d.dt && d.dt_residual != ELB_F32) return op_fail(ELB_UNIMPLEMENTED, "norm takes a residual in its own type or fp32");
  if (d.dt_weights != d.dt && d.dt_weights != ELB_F32) return op_fail(ELB_UNIMPLEMENTED, "norm takes weights in its own type or fp32");
  for (int k : {d.post, d.pre}) if (k < ELB_NORM_NONE || k > ELB_NORM_LAYER) return op_fail(ELB_GENERAL_ERROR, "norm kind %d", k);
  if (!(d.post_eps >= 0.0f) || !(d.pre_eps >= 0.0f) || !finite(d.post_eps) || !finite(d.pre_eps) || !finite(d.scale) || !finite(d.weight_offset))
    return op_fail(ELB_GENERAL_ERROR, "eps, scale or weight offset is negative or not finite");
  if (d.gate_rows < 0) return op_fail(ELB_GENERAL_ERROR, "gate_rows %d", d.gate_rows);
  int rc = ELB_OK;
  int64_t *lds[] = {&d.ld_input, &d.ld_residual, &d.ld_gate, &d.ld_sum, &d.ld_output};
  const char *names[] = {"input", "residual", "gate", "sum", "output"};
  for (int i = 0; i < 5 && rc == ELB_OK; ++i) rc = check_ld(names[i], *lds[i], d.channels);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(NORM, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->norm = d;
  *out = op;
  return ELB_OK;
}

int elb_norm_prepare(elb_op_t *op, const void *post_weight, const void *post_bias, const void *pre_weight, const void *pre_bias) {
  int rc = check_op(op, NORM);
  if (rc != ELB_OK || op->prepared) return rc;
  const elb_norm_desc_t &d = op->norm;
  const void *src[4] = {post_weight, post_bias, pre_weight, pre_bias};
  const int kind[4] = {d.post, d.post, d.pre, d.pre};
  DeviceGuard guard(op->device);
  OP_TRY(cudaDeviceSynchronize());
  for (int i = 0; i < 4 && rc == ELB_OK; ++i) {
    if (kind[i] == ELB_NORM_NONE || (!src[i] && i % 2 == 1)) continue;
    if (src[i] && !aligned(src[i], et_bytes(et_of(d.dt_weights)))) rc = op_fail(ELB_GENERAL_ERROR, "misaligned weights");
    else rc = norm_vector(*op, &op->f[i], src[i], et_of(d.dt_weights), d.channels, i % 2 == 0 ? d.weight_offset : 0.0f);
  }
  return drop(*op, rc);
}

int elb_norm_enqueue(elb_op_t *op, void *output, void *sum, const void *input, const void *residual, const void *gate, int64_t rows,
                     void *cuda_stream) {
  int rc = check_op(op, NORM);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  if (rc != ELB_OK || rows == 0) return rc;
  const elb_norm_desc_t &d = op->norm;
  if (!input || (d.pre != ELB_NORM_NONE && !output) || (d.pre == ELB_NORM_NONE && !sum) || (d.with_residual && !residual) || (d.gate_rows && !gate))
    return op_fail(ELB_GENERAL_ERROR, "null argument");
  const size_t b = et_bytes(et_of(d.dt)), rb = et_bytes(et_of(d.dt_residual));
  if (!aligned(input, b) || !aligned(output, b) || !aligned(gate, b) || !aligned(sum, rb) || !aligned(residual, rb))
    return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  NormParams p = {};
  p.x = input;
  p.res = d.with_residual ? residual : nullptr;
  p.gate = d.gate_rows ? gate : nullptr;
  p.sum = sum;
  p.y = d.pre != ELB_NORM_NONE ? output : nullptr;
  p.post_w = op->f[0]; p.post_b = op->f[1]; p.pre_w = op->f[2]; p.pre_b = op->f[3];
  p.ld_x = d.ld_input; p.ld_res = d.ld_residual; p.ld_gate = d.ld_gate; p.ld_sum = d.ld_sum; p.ld_y = d.ld_output;
  p.rows = rows;
  p.w_pitch = norm_pitch(d.channels);
  p.num_sms = op->num_sms;
  p.channels = d.channels;
  p.gate_rows = d.gate_rows;
  p.post = d.post; p.pre = d.pre;
  p.et = et_of(d.dt); p.et_res = et_of(d.dt_residual);
  p.post_eps = d.post_eps; p.pre_eps = d.pre_eps; p.scale = d.scale;
  OP_TRY(launch_block_norm(p, static_cast<cudaStream_t>(cuda_stream)));
  ++op->launches;
  return ELB_OK;
}

// ------------------------------------------------------------------------------------------- route
int elb_route_create(const elb_route_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_route_desc_t d = *desc;
  if (d.experts < 1 || d.top_k < 1 || d.top_k > d.experts) return op_fail(ELB_GENERAL_ERROR, "%d of %d experts", d.top_k, d.experts);
  if (d.experts > 1024 || d.top_k > 32) return op_fail(ELB_UNIMPLEMENTED, "%d of %d experts: at most 32 of 1024", d.top_k, d.experts);
  if (et_of(d.dt_logits) < 0) return op_fail(ELB_UNIMPLEMENTED, "routing takes fp32, f16 and bf16 logits");
  if (d.score != ELB_SCORE_SOFTMAX && d.score != ELB_SCORE_SIGMOID) return op_fail(ELB_GENERAL_ERROR, "score %d", d.score);
  if (d.groups < 1 || d.experts % d.groups != 0 || d.top_groups < 1 || d.top_groups > d.groups || d.group_best < 1)
    return op_fail(ELB_GENERAL_ERROR, "%d of %d groups of %d experts, by their %d best", d.top_groups, d.groups, d.experts, d.group_best);
  if (d.groups > 32 || d.group_best > 2) return op_fail(ELB_UNIMPLEMENTED, "%d groups by their %d best: at most 32 by 2", d.groups, d.group_best);
  if (d.top_k > d.experts / d.groups * d.top_groups)
    return op_fail(ELB_GENERAL_ERROR, "%d experts of %d groups of %d", d.top_k, d.top_groups, d.experts / d.groups);
  if (!finite(d.scale)) return op_fail(ELB_GENERAL_ERROR, "scale is not finite");
  int rc = check_ld("logits", d.ld_logits, d.experts);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(ROUTE, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->route = d;
  *out = op;
  return ELB_OK;
}

int elb_route_prepare(elb_op_t *op, const float *bias) {
  int rc = check_op(op, ROUTE);
  if (rc != ELB_OK || op->prepared) return rc;
  if (op->route.with_bias && (!bias || !aligned(bias, 4))) return op_fail(ELB_GENERAL_ERROR, "bias is null or misaligned");
  DeviceGuard guard(op->device);
  OP_TRY(cudaDeviceSynchronize());
  if (op->route.with_bias) rc = vector_f32(*op, &op->f[0], bias, ET_F32, op->route.experts, op->route.experts, false);
  return drop(*op, rc);
}

int elb_route_enqueue(elb_op_t *op, int32_t *ids, float *weights, const void *logits, int64_t rows, void *cuda_stream) {
  int rc = check_op(op, ROUTE);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  if (rc != ELB_OK || rows == 0) return rc;
  const elb_route_desc_t &d = op->route;
  if (!ids || !logits) return op_fail(ELB_GENERAL_ERROR, "null argument");
  if (!aligned(ids, 4) || !aligned(weights, 4) || !aligned(logits, et_bytes(et_of(d.dt_logits)))) return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  RouteParams p = {};
  p.logits = logits;
  p.bias = op->f[0];
  p.ids = ids;
  p.weights = weights;
  p.ld = d.ld_logits;
  p.rows = rows;
  p.experts = d.experts; p.top_k = d.top_k; p.et = et_of(d.dt_logits);
  p.sigmoid = d.score == ELB_SCORE_SIGMOID;
  p.groups = d.groups; p.top_groups = d.top_groups; p.group_best = d.group_best;
  p.renormalise = d.renormalise;
  p.scale = d.scale;
  OP_TRY(launch_route(p, static_cast<cudaStream_t>(cuda_stream)));
  ++op->launches;
  return ELB_OK;
}

// ------------------------------------------------------------------------------------------- experts
int elb_experts_create(const elb_experts_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_experts_desc_t d = *desc;
  if (d.experts < 1 || d.top_k < 1 || d.ic < 1 || d.mid < 1 || d.ic > (1 << 20) || d.mid > (1 << 20))
    return op_fail(ELB_GENERAL_ERROR, "%d experts, %d per token, %d and %d channels", d.experts, d.top_k, d.ic, d.mid);
  if (d.experts > 1024 || d.top_k > 32) return op_fail(ELB_UNIMPLEMENTED, "%d of %d experts: at most 32 of 1024", d.top_k, d.experts);
  if (d.dt != ELB_BF16 && d.dt != ELB_F16) return op_fail(ELB_UNIMPLEMENTED, "experts take bf16 and f16");
  if (d.activation < ELB_ACT_NONE || d.activation > ELB_ACT_SILU) return op_fail(ELB_GENERAL_ERROR, "activation %d", d.activation);
  if (d.max_rows < 1 || d.max_rows > MAX_ROWS / d.top_k) return op_fail(ELB_GENERAL_ERROR, "max_rows %lld", (long long)d.max_rows);
  int rc = check_ld("input", d.ld_input, d.ic);
  if (rc == ELB_OK) rc = check_ld("output", d.ld_output, d.ic);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(EXPERTS, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->exp = d;
  DeviceGuard guard(op->device);
  const int64_t slots = d.max_rows * d.top_k, px = up(d.ic, 8), pm = up(d.mid, 8), py = up(d.ic, 4);
  const int64_t tiles = slots / MIN_TILE_TOKENS + d.experts, few = slots < GEMV_SLOTS ? slots : GEMV_SLOTS;    // (those have fp32 middle rows)
  size_t at = 0;
  auto part = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  const size_t o_xs = part(slots * px * 2),
               o_mid = part(slots * pm * 2 > few * pm * 4 ? slots * pm * 2 : few * pm * 4), o_y = part(slots * py * 4), o_pos = part(slots * 4),
               o_place = part(slots * 4), o_tiles = part(tiles * sizeof(GroupTile)), o_n = part(4), o_count = part(d.experts * 4);
  rc = alloc(*op, &op->ws, at);
  if (rc != ELB_OK) { delete op; return rc; }
  op->ws_bytes = at;
  if (cudaMemset(static_cast<uint8_t *>(op->ws) + o_count, 0, d.experts * 4) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
    cudaGetLastError();
    delete op;
    return op_fail(ELB_GENERAL_ERROR, "the workspace could not be cleared");
  }
  uint8_t *b = static_cast<uint8_t *>(op->ws);
  ExpertsParams &e = op->ep;
  e.xs = b + o_xs;
  op->mid = b + o_mid;
  e.y = reinterpret_cast<float *>(b + o_y);
  e.pos = reinterpret_cast<int *>(b + o_pos);
  e.place = reinterpret_cast<int *>(b + o_place);
  e.count = reinterpret_cast<int *>(b + o_count);
  e.tiles = reinterpret_cast<GroupTile *>(b + o_tiles);
  e.n_tiles = reinterpret_cast<int *>(b + o_n);
  e.ld_x = d.ld_input; e.ld_out = d.ld_output; e.pitch_x = px; e.pitch_y = py;
  e.top_k = d.top_k; e.experts = d.experts; e.ic = d.ic; e.et = et_of(d.dt);
  op->pitch_mid = pm;
  *out = op;
  return ELB_OK;
}

int elb_experts_prepare(elb_op_t *op, const void *w_in, const void *w_out) {
  int rc = check_op(op, EXPERTS);
  if (rc != ELB_OK || op->prepared) return rc;
  const elb_experts_desc_t &d = op->exp;
  if (!w_in || !w_out || !aligned(w_in, 2) || !aligned(w_out, 2)) return op_fail(ELB_GENERAL_ERROR, "weights are null or misaligned");
  DeviceGuard guard(op->device);
  OP_TRY(cudaDeviceSynchronize());
  rc = pack(*op, &op->w[0], w_in, d.experts, d.gated ? 2 * d.mid : d.mid, d.ic, d.gated, false);
  if (rc == ELB_OK) rc = pack(*op, &op->w[1], w_out, d.experts, d.ic, d.mid, false, false);
  return drop(*op, rc);
}

int elb_experts_enqueue(elb_op_t *op, void *output, const void *input, const int32_t *ids, const float *weights, int64_t rows,
                        void *cuda_stream) {
  int rc = check_op(op, EXPERTS);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  if (rc != ELB_OK || rows == 0) return rc;
  const elb_experts_desc_t &d = op->exp;
  if (rows > d.max_rows) return op_fail(ELB_GENERAL_ERROR, "%lld rows: the plan was made for %lld", (long long)rows, (long long)d.max_rows);
  if (!output || !input || !ids || !weights) return op_fail(ELB_GENERAL_ERROR, "null argument");
  if (!aligned(output, 2) || !aligned(input, 2) || !aligned(ids, 4) || !aligned(weights, 4)) return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  WorkspaceCall use(*op, s);
  rc = use.enter();
  if (rc != ELB_OK) return rc;
  ExpertsParams e = op->ep;
  e.rows = (int)rows;
  e.x = input;
  e.out = output;
  e.ids = ids;
  e.weights = weights;
  const int slots = (int)(rows * d.top_k), wide = packed_rows(d.mid, d.gated);
  e.tile_tokens = grouped_tile_tokens(slots, d.experts);
  GemmParams p = {};
  p.tiles = e.tiles;
  p.tile_tokens = e.tile_tokens;
  p.n_tiles = e.n_tiles;
  p.max_tiles = slots < d.experts ? slots : slots / e.tile_tokens + d.experts;
  p.in_et = e.et;
  p.num_sms = op->num_sms;
  p.max_pairs = op->max_pairs;
  p.status = op->d_status;
  p.epi.words = 1;
  p.epi.scale = 1.0f;
  GemmParams q = p;
  p.w = static_cast<const uint8_t *>(op->w[0]);
  p.x = e.xs;
  p.ld_x = e.pitch_x;
  p.rows = slots;
  p.ic = d.ic;
  p.kt = (int)(up(d.ic, GT_K) / GT_K);
  p.row_tiles = (int)(up(wide, GT_ROWS) / GT_ROWS);
  p.w_stride = (size_t)p.row_tiles * p.kt * GT_BYTES;
  p.w_rows = (long long)d.experts * p.row_tiles * p.kt * GT_ROWS;
  p.epi.out = op->mid;
  p.epi.ld_out = op->pitch_mid;
  p.epi.oc = (int)op->pitch_mid;          // (channels past the end are products with rows of zeros)
  p.epi.act = d.activation;
  p.epi.gated = d.gated;
  p.epi.out_et = e.et;                    // the middle is a 16-bit operand of the second product: one rounding, as large as the output's
  q.w = static_cast<const uint8_t *>(op->w[1]);
  q.x = op->mid;
  q.ld_x = op->pitch_mid;
  q.rows = slots;
  q.ic = d.mid;
  q.kt = (int)(up(d.mid, GT_K) / GT_K);
  q.row_tiles = (int)(up(d.ic, GT_ROWS) / GT_ROWS);
  q.w_stride = (size_t)q.row_tiles * q.kt * GT_BYTES;
  q.w_rows = (long long)d.experts * q.row_tiles * q.kt * GT_ROWS;
  q.tiles_old = 1;
  q.epi.out = const_cast<float *>(e.y);
  q.epi.ld_out = e.pitch_y;
  q.epi.oc = (int)e.pitch_y;
  q.epi.out_et = ET_F32;
  if (experts_want_gemv(slots, d.experts, (double)p.w_stride + (double)q.w_stride)) {
    p.x = input;
    p.ld_x = d.ld_input;
    p.epi.out_et = ET_F32;
    q.epi.out = output;
    q.epi.ld_out = d.ld_output;
    q.epi.oc = d.ic;
    q.epi.out_et = e.et;
    OP_TRY(launch_gemv_experts(p, q, ids, weights, (int)rows, d.top_k, d.experts, s));
    op->launches += 2;
    return use.leave();
  }
  const bool count = !experts_count_here(slots);
  const size_t count_bytes = d.experts * sizeof(int);
  e.clear = count;
  if (count && op->count_stale) {
    OP_TRY(cudaMemsetAsync(e.count, 0, count_bytes, s));
    if (!use.capturing) op->count_stale = false;       // (what is captured has not run)
  }
  cudaError_t err = count ? launch_experts_count(e, s) : cudaSuccess;
  if (err == cudaSuccess) err = launch_experts_gather(e, op->num_sms, s);
  if (err == cudaSuccess) err = launch_gemm(p, s);
  if (err == cudaSuccess) err = launch_gemm(q, s);
  if (err == cudaSuccess) err = launch_experts_combine(e, s);
  // The sum over a token's experts, which leaves zero counts, has not been launched
  if (err != cudaSuccess && count && cudaMemsetAsync(e.count, 0, count_bytes, s) != cudaSuccess && !use.capturing) op->count_stale = true;
  OP_TRY(err);
  op->launches += count ? 5 : 4;
  return use.leave();
}

// ------------------------------------------------------------------------------------------- all
int elb_op_device_status(elb_op_t *op) {
  if (!op) return -1;
  DeviceGuard guard(op->device);
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  return *reinterpret_cast<volatile int *>(op->h_status);
}
int elb_op_device(const elb_op_t *op) { return op ? op->device : -1; }
uint64_t elb_op_launch_count(const elb_op_t *op) { return op ? op->launches : 0; }
uint64_t elb_op_workspace_bytes(const elb_op_t *op) { return op ? op->bytes : 0; }
void elb_op_destroy(elb_op_t *op) { delete op; }

}  // extern "C"
