// C-ABI of the attention operators (include/euler_b200.h, "Attention"): descriptions are checked when a plan is made, a call checks
// its arguments and enqueues.
#include <cmath>
#include <mutex>

#include "attention.cuh"
#include "op_plan.cuh"

using namespace elb;

namespace {

constexpr int64_t MAX_SEQS = 1 << 24, MAX_LD = 1ll << 40;

int check_rotary(elb_rotary_desc_t &d, bool append) {
  if (d.heads < 0 || d.kv_heads < 0 || d.heads + (int64_t)d.kv_heads < 1 || d.heads > 4096 || d.kv_heads > 4096)
    return op_fail(ELB_GENERAL_ERROR, "rotary of %d and %d heads: at most 4096", d.heads, d.kv_heads);
  if (d.head_dim < 1 || d.head_dim > 1024) return op_fail(ELB_GENERAL_ERROR, "heads of %d channels: 1 to 1024", d.head_dim);
  if (d.rotary_dim < (append ? 0 : 2) || d.rotary_dim > d.head_dim || d.rotary_dim % 2 != 0)
    return op_fail(ELB_GENERAL_ERROR, "%d of %d channels turn", d.rotary_dim, d.head_dim);
  if (et_of(d.dt) < 0) return op_fail(ELB_UNIMPLEMENTED, "rotary takes fp32, f16 and bf16");
  if (d.layout != ELB_ROTARY_HALVES && d.layout != ELB_ROTARY_NEIGHBOURS) return op_fail(ELB_GENERAL_ERROR, "layout %d", d.layout);
  if (d.scaling < ELB_SCALE_NONE || d.scaling > ELB_SCALE_BY_PARTS) return op_fail(ELB_GENERAL_ERROR, "scaling %d", d.scaling);
  if (!finite(d.base) || !(d.base > 0.0f) || !finite(d.magnitude)) return op_fail(ELB_GENERAL_ERROR, "base or magnitude: not finite, or base not above 0");
  if (d.scaling != ELB_SCALE_NONE && (!finite(d.factor) || !(d.factor > 0.0f))) return op_fail(ELB_GENERAL_ERROR, "factor: not finite, or not above 0");
  if (d.scaling == ELB_SCALE_BY_PARTS && (!finite(d.slow) || !finite(d.fast) || !(d.fast > d.slow) || d.original < 1))
    return op_fail(ELB_GENERAL_ERROR, "by parts: slow below fast, original at least 1");
  const int64_t q = (int64_t)d.heads * d.head_dim, k = (int64_t)d.kv_heads * d.head_dim;
  int rc = check_ld("q", d.ld_q, q);
  if (rc == ELB_OK) rc = check_ld("k", d.ld_k, k);
  if (rc == ELB_OK) rc = check_ld("q_out", d.ld_q_out, q);
  if (rc == ELB_OK && !append) rc = check_ld("k_out", d.ld_k_out, k);
  return rc;
}

// Turns per position of each pair, modulo 1, as 64-bit fractions, worked out in the long double's 64 bits: 53 of them would leave the angle of position 2^31 wrong by
// 2^-20 times the frequency in radians.
int make_steps(elb_op &op, const elb_rotary_desc_t &d, const float *frequencies) {
  const int n = d.rotary_dim / 2;
  unsigned long long steps[512];
  float given[512];
  if (frequencies && n > 0) {
    if (!aligned(frequencies, 4)) return op_fail(ELB_GENERAL_ERROR, "misaligned frequencies");
    Staged st;                                                 // (waits for another device's work)
    const int rc = st.take(op, frequencies, n * sizeof(float));
    if (rc != ELB_OK) return rc;
    OP_TRY(cudaMemcpy(given, st.p, n * sizeof(float), cudaMemcpyDefault));
  }
  const long double two_pi = 6.283185307179586476925286766559005768L;
  for (int i = 0; i < n; ++i) {
    long double f = std::pow((long double)d.base, -2.0L * i / d.rotary_dim);
    if (d.scaling == ELB_SCALE_LINEAR) f /= d.factor;
    if (d.scaling == ELB_SCALE_BY_PARTS) {
      long double s = (d.original * f / two_pi - d.slow) / ((long double)d.fast - d.slow);
      s = s < 0.0L ? 0.0L : s > 1.0L ? 1.0L : s;
      f = s * f + (1.0L - s) * f / d.factor;
    }
    if (frequencies) f = given[i];
    if (!std::isfinite(f)) return op_fail(ELB_GENERAL_ERROR, "frequency %d is not finite", i);
    long double turn = f / two_pi;
    turn -= std::floor(turn);
    steps[i] = turn >= 1.0L ? 0ull : (unsigned long long)std::ldexp(turn, 64);
  }
  unsigned long long *dst = nullptr;
  const int rc = alloc(op, &dst, (n > 0 ? n : 1) * sizeof(unsigned long long));
  if (rc != ELB_OK) return rc;
  op.w[0] = dst;
  OP_TRY(cudaMemcpy(dst, steps, n * sizeof(unsigned long long), cudaMemcpyHostToDevice));
  OP_TRY(cudaDeviceSynchronize());                             // (that copy returns when it has read its source; streams that wait for no other come next)
  return ELB_OK;
}

int prepare_rotary(elb_op &op, const elb_rotary_desc_t &d, const float *frequencies) {
  DeviceGuard guard(op.device);
  if (frequencies) OP_TRY(cudaDeviceSynchronize());            // whatever stream the caller's tensor comes from
  const int rc = make_steps(op, d, frequencies);
  if (rc == ELB_OK) { op.prepared = true; return rc; }
  if (op.w[0]) { cudaFree(op.w[0]); op.w[0] = nullptr; }
  op.bytes = 0;
  return rc;
}

RotaryParams rotary_params(const elb_op &op, const elb_rotary_desc_t &d) {
  RotaryParams p = {};
  p.ld_q = d.ld_q; p.ld_k = d.ld_k; p.ld_q_out = d.ld_q_out; p.ld_k_out = d.ld_k_out;
  p.steps = static_cast<const unsigned long long *>(op.w[0]);
  p.heads = d.heads; p.kv_heads = d.kv_heads; p.head_dim = d.head_dim; p.rotary = d.rotary_dim;
  p.neighbours = d.layout == ELB_ROTARY_NEIGHBOURS;
  p.inverse = d.inverse != 0;
  p.et = et_of(d.dt);
  p.magnitude = d.magnitude;
  p.num_sms = op.num_sms;
  p.status = op.d_status;
  return p;
}

// The batch of a call; NULL arguments that may be are the callers' to look at.
int check_sequences(Sequences &b, const int32_t *table, const int32_t *lengths, const int32_t *starts, int64_t rows, int64_t seqs, int64_t pages, int64_t width,
                    int page_size) {
  if (seqs < 0 || seqs > MAX_SEQS || pages < 0 || pages > INT32_MAX || width < 0 || width > INT32_MAX)
    return op_fail(ELB_GENERAL_ERROR, "%lld sequences, %lld pages, width %lld", (long long)seqs, (long long)pages, (long long)width);
  if (!starts && seqs > 0 && rows % seqs != 0) return op_fail(ELB_GENERAL_ERROR, "%lld rows of %lld sequences: starts are wanted", (long long)rows, (long long)seqs);
  if (!aligned(table, 4) || !aligned(lengths, 4) || !aligned(starts, 4)) return op_fail(ELB_GENERAL_ERROR, "misaligned table, lengths or starts");
  b.table = table; b.lengths = lengths; b.starts = starts;
  b.rows = rows; b.seqs = seqs; b.width = width; b.pages = pages;
  b.each = starts || seqs == 0 ? 0 : (int)(rows / seqs);
  const int64_t capacity = page_size ? width * page_size : width;
  b.capacity = (int)(capacity < INT32_MAX - 255 ? capacity : INT32_MAX - 255);     // (a tile's end is a number too)
  return ELB_OK;
}

// Strides of a cache: defaults, and that no two of its elements share a place
int check_cache(int64_t &ld_page, int64_t &ld_head, int64_t &ld_token, int64_t kv_heads, int64_t page_size, int64_t head_dim) {
  if (ld_page < 0 || ld_head < 0 || ld_token < 0 || ld_page > MAX_LD || ld_head > MAX_LD || ld_token > MAX_LD)
    return op_fail(ELB_GENERAL_ERROR, "strides of the cache: %lld, %lld, %lld", (long long)ld_page, (long long)ld_head, (long long)ld_token);
  if (ld_token == 0) ld_token = head_dim;
  if (ld_head == 0) ld_head = page_size * ld_token;
  if (ld_page == 0) ld_page = ld_head > ld_token ? kv_heads * ld_head : page_size * ld_token;
  const int64_t last = (kv_heads - 1) * ld_head + (page_size - 1) * ld_token + head_dim;
  const bool apart = ld_token >= head_dim && (kv_heads == 1 || (ld_head >= head_dim && (ld_head >= (page_size - 1) * ld_token + head_dim || ld_token >= (kv_heads - 1) * ld_head + head_dim)));
  if (!apart || ld_page < last) return op_fail(ELB_GENERAL_ERROR, "pages of %lld heads and %lld tokens overlap", (long long)kv_heads, (long long)page_size);
  return ELB_OK;
}

// Kernel attributes are a device's: once for each of them.
int init_device(int device) {
  static std::mutex mutex;
  static bool known[64];
  std::lock_guard<std::mutex> lock(mutex);
  if (!known[device]) {                                         // (make_op has refused larger ordinals)
    OP_TRY(init_attention());
    OP_TRY(init_attention_prompt());
  }
  known[device] = true;
  return ELB_OK;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------------------- rotary
int elb_rotary_create(const elb_rotary_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_rotary_desc_t d = *desc;
  int rc = check_rotary(d, false);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(ROTARY, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->rot = d;
  *out = op;
  return ELB_OK;
}

int elb_rotary_prepare(elb_op_t *op, const float *frequencies) {
  const int rc = check_op(op, ROTARY);
  return rc != ELB_OK || op->prepared ? rc : prepare_rotary(*op, op->rot, frequencies);
}

int elb_rotary_enqueue(elb_op_t *op, void *q_out, void *k_out, const void *q, const void *k, const int32_t *positions, int64_t rows, void *cuda_stream) {
  int rc = check_op(op, ROTARY);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  if (rc != ELB_OK || rows == 0) return rc;
  const elb_rotary_desc_t &d = op->rot;
  if ((d.heads && (!q_out || !q)) || (d.kv_heads && (!k_out || !k)) || !positions) return op_fail(ELB_GENERAL_ERROR, "null argument");
  const int et = et_of(d.dt);
  const size_t e = et_bytes(et);
  if (!aligned(q, e) || !aligned(k, e) || !aligned(q_out, e) || !aligned(k_out, e) || !aligned(positions, 4)) return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  RotaryParams p = rotary_params(*op, d);
  p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
  p.positions = positions;
  p.rows = rows;
  const int64_t per = 16 / e;
  p.words = aligned(q, 16) && aligned(k, 16) && aligned(q_out, 16) && aligned(k_out, 16) && (d.head_dim | d.ld_q | d.ld_k | d.ld_q_out | d.ld_k_out) % per == 0;
  OP_TRY(launch_rotary(p, static_cast<cudaStream_t>(cuda_stream)));
  ++op->launches;
  return ELB_OK;
}

// ------------------------------------------------------------------------------------------- append
int elb_append_create(const elb_append_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_append_desc_t d = *desc;
  int rc = check_rotary(d.rotary, true);
  if (rc != ELB_OK) return rc;
  if (d.rotary.kv_heads < 1) return op_fail(ELB_GENERAL_ERROR, "a cache of %d heads", d.rotary.kv_heads);
  if (d.page_size < 1 || d.page_size > (1 << 20)) return op_fail(ELB_GENERAL_ERROR, "pages of %d tokens", d.page_size);
  rc = check_ld("v", d.ld_v, (int64_t)d.rotary.kv_heads * d.rotary.head_dim);
  if (rc == ELB_OK) rc = check_cache(d.ld_page, d.ld_head, d.ld_token, d.rotary.kv_heads, d.page_size, d.rotary.head_dim);
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(APPEND, d.rotary.device, &op);
  if (rc != ELB_OK) return rc;
  op->app = d;
  *out = op;
  return ELB_OK;
}

int elb_append_prepare(elb_op_t *op, const float *frequencies) {
  const int rc = check_op(op, APPEND);
  return rc != ELB_OK || op->prepared ? rc : prepare_rotary(*op, op->app.rotary, frequencies);
}

int elb_append_enqueue(elb_op_t *op, void *q_out, void *k_cache, void *v_cache, const void *q, const void *k, const void *v, const int32_t *table,
                       const int32_t *lengths, const int32_t *starts, int64_t rows, int64_t seqs, int64_t pages, int64_t width, void *cuda_stream) {
  int rc = check_op(op, APPEND);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  RotaryParams p = {};
  if (rc == ELB_OK) { p = rotary_params(*op, op->app.rotary); rc = check_sequences(p.seq, table, lengths, starts, rows, seqs, pages, width, op->app.page_size); }
  if (rc != ELB_OK || rows == 0 || seqs == 0) return rc;
  const elb_append_desc_t &d = op->app;
  const elb_rotary_desc_t &r = d.rotary;
  if ((r.heads && (!q_out || !q)) || !k_cache || !v_cache || !k || !v || !table || !lengths) return op_fail(ELB_GENERAL_ERROR, "null argument");
  const size_t e = et_bytes(p.et);
  if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(q_out, e) || !aligned(k_cache, e) || !aligned(v_cache, e))
    return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  p.q = q; p.k = k; p.v = v;
  p.q_out = q_out; p.k_out = k_cache; p.v_out = v_cache;
  p.rows = rows;
  p.page_size = d.page_size;
  p.ld_v = d.ld_v; p.ld_page = d.ld_page; p.ld_head = d.ld_head; p.ld_token = d.ld_token;
  const int64_t per = 16 / e;
  p.words = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
            (r.head_dim | r.ld_q | r.ld_k | r.ld_q_out | d.ld_v | d.ld_page | d.ld_head | d.ld_token) % per == 0;
  OP_TRY(launch_rotary(p, static_cast<cudaStream_t>(cuda_stream)));
  ++op->launches;
  return ELB_OK;
}

// ------------------------------------------------------------------------------------------- attention
int elb_attention_create(const elb_attention_desc_t *desc, elb_op_t **out) {
  if (!desc || !out) return op_fail(ELB_GENERAL_ERROR, "null argument");
  elb_attention_desc_t d = *desc;
  if (d.heads < 1 || d.kv_heads < 1 || d.heads > 4096 || d.heads % d.kv_heads != 0)
    return op_fail(ELB_GENERAL_ERROR, "attention of %d heads over %d: a multiple, at most 4096", d.heads, d.kv_heads);
  if (d.head_dim < 1) return op_fail(ELB_GENERAL_ERROR, "heads of %d channels", d.head_dim);
  if (d.head_dim > 256) return op_fail(ELB_UNIMPLEMENTED, "heads of %d channels: at most 256", d.head_dim);
  if (d.dt != ELB_BF16 && d.dt != ELB_F16) return op_fail(ELB_UNIMPLEMENTED, "attention takes bf16 and f16");
  if (d.page_size < 0 || d.page_size > (1 << 20)) return op_fail(ELB_GENERAL_ERROR, "pages of %d tokens", d.page_size);
  if (!finite(d.scale)) return op_fail(ELB_GENERAL_ERROR, "scale is not finite");
  if (d.scale == 0.0f) d.scale = (float)(1.0 / std::sqrt((double)d.head_dim));
  const int64_t wide = (int64_t)d.heads * d.head_dim;
  int rc = check_ld("input", d.ld_input, wide);
  if (rc == ELB_OK) rc = check_ld("output", d.ld_output, wide);
  if (rc == ELB_OK && d.page_size) rc = check_cache(d.ld_page, d.ld_head, d.ld_token, d.kv_heads, d.page_size, d.head_dim);
  if (rc == ELB_OK && !d.page_size) {
    rc = check_ld("k and v: heads'", d.ld_head, d.head_dim);
    if (rc == ELB_OK) rc = check_ld("k and v: tokens'", d.ld_token, d.ld_token ? d.head_dim : (int64_t)d.kv_heads * d.ld_head);
    if (rc == ELB_OK && (d.ld_page < 0 || d.ld_page > MAX_LD)) rc = op_fail(ELB_GENERAL_ERROR, "sequences of k and v lie %lld apart", (long long)d.ld_page);
  }
  elb_op *op = nullptr;
  if (rc == ELB_OK) rc = make_op(ATTENTION, d.device, &op);
  if (rc != ELB_OK) return rc;
  op->att = d;
  DeviceGuard guard(op->device);
  rc = init_device(op->device);
  op->ws_bytes = attention_workspace_bytes(op->num_sms);
  if (rc == ELB_OK) rc = alloc(*op, &op->ws, op->ws_bytes);
  if (rc == ELB_OK && (cudaMemset(op->ws, 0, op->ws_bytes) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess)) {
    cudaGetLastError();
    rc = op_fail(ELB_GENERAL_ERROR, "the workspace could not be cleared");
  }
  if (rc != ELB_OK) { delete op; return rc; }
  op->prepared = true;
  *out = op;
  return ELB_OK;
}

int elb_attention_enqueue(elb_op_t *op, void *output, const void *input, const void *k, const void *v, const int32_t *table, const int32_t *lengths,
                          const int32_t *starts, int64_t rows, int64_t seqs, int64_t pages, int64_t width, void *cuda_stream) {
  int rc = check_op(op, ATTENTION);
  if (rc == ELB_OK) rc = check_call(*op, rows);
  AttentionParams p = {};
  if (rc == ELB_OK) rc = check_sequences(p.seq, table, lengths, starts, rows, seqs, op->att.page_size ? pages : seqs, width, op->att.page_size);
  if (rc != ELB_OK || rows == 0 || seqs == 0) return rc;
  const elb_attention_desc_t &d = op->att;
  if (!output || !input || (width > 0 && (!k || !v)) || (d.page_size && (!lengths || (width > 0 && !table)))) return op_fail(ELB_GENERAL_ERROR, "null argument");
  if (!d.page_size && table) return op_fail(ELB_GENERAL_ERROR, "a table for dense keys and values");
  if (!aligned(output, 2) || !aligned(input, 2) || !aligned(k, 2) || !aligned(v, 2)) return op_fail(ELB_GENERAL_ERROR, "misaligned tensor");
  DeviceGuard guard(op->device);
  p.out = output; p.q = input; p.k = k; p.v = v;
  p.ld_q = d.ld_input; p.ld_out = d.ld_output;
  p.ld_page = d.ld_page ? d.ld_page : width * d.ld_token;
  p.ld_head = d.ld_head; p.ld_token = d.ld_token;
  p.heads = d.heads; p.kv_heads = d.kv_heads; p.head_dim = d.head_dim;
  p.et = et_of(d.dt);
  p.page_size = d.page_size;
  p.causal = d.causal != 0;
  p.scale = d.scale;
  p.words = aligned(output, 16) && aligned(input, 16) && aligned(k, 16) && aligned(v, 16) &&
            (d.head_dim | d.ld_input | d.ld_output | p.ld_page | p.ld_head | p.ld_token) % 8 == 0 &&
            (d.ld_input | p.ld_page | p.ld_head | p.ld_token) < 1ll << 39;          // (a tiled copy's strides are below 2^40 bytes)
  p.num_sms = op->num_sms;
  p.status = op->d_status;
  const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  const bool token = attention_token_takes(p);
  if (!token && !attention_prompt_takes(p)) {
    OP_TRY(launch_attention_any(p, s));
    ++op->launches;
    return ELB_OK;
  }
  WorkspaceCall use(*op, s);
  rc = use.enter();
  if (rc != ELB_OK) return rc;
  float *partial = static_cast<float *>(op->ws);
  const AttentionWorkspace w = {partial, reinterpret_cast<int *>(partial + attention_partial_floats(op->num_sms))};
  OP_TRY(token ? launch_attention_token(p, w, s) : launch_attention_prompt(p, w, s));
  ++op->launches;
  return use.leave();
}

}  // extern "C"
