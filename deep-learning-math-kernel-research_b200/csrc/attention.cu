// Attention for every shape, on CUDA cores.
//
// A warp takes one head of one new token, its lanes the channels, and goes over the keys that the token sees with the running maximum m and
// sum l of the softmax: with m' = max(m, s), l = l e^(m - m') + e^(s - m') and the same for the weighted sum of values.  Bound by the reductions
// of each score over the lanes, some 40 instructions a key.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"

namespace elb {

namespace {

constexpr int WARPS = 4, MAX_DIM = 256;

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) attention_any_kernel(const AttentionParams p) {
  const int lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  griddep_launch_dependents();
  griddep_wait();
  const long long items = p.seq.rows * p.heads;
  for (long long i = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); i < items; i += (long long)gridDim.x * WARPS) {
    const int row = (int)(i / p.heads), h = (int)(i - (long long)row * p.heads);
    const int s = sequence_of_row(p.seq, row, lane);
    if (s < 0 || s >= p.seq.seqs) continue;                     // behind the last sequence
    const Sequence seq = sequence_of(p.seq, s);
    const int keys = p.causal ? min(seq.length, seq.length - seq.n + (row - seq.first) + 1) : seq.length;
    const T *q = static_cast<const T *>(p.q) + row * p.ld_q + (long long)h * p.head_dim;
    const long long head = (h / group) * p.ld_head;
    float x[MAX_DIM / 32], o[MAX_DIM / 32], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < MAX_DIM / 32; ++c) {
      x[c] = lane + 32 * c < p.head_dim ? to_f32(q[lane + 32 * c]) * p.scale : 0.0f;
      o[c] = 0.0f;
    }
    for (int j = 0; j < keys; ++j) {
      long long at;
      bool there = true;
      if (p.page_size) {
        const int page = p.seq.table[s * p.seq.width + j / p.page_size];
        there = page >= 0 && page < p.seq.pages;
        if (!there && lane == 0) report_status(p.status, ST_BAD_PAGE);
        at = page * p.ld_page + j % p.page_size * p.ld_token + head;
      } else {
        at = s * p.ld_page + j * p.ld_token + head;
      }
      const T *k = static_cast<const T *>(p.k) + at, *v = static_cast<const T *>(p.v) + at;
      float z = 0.0f;
#pragma unroll
      for (int c = 0; c < MAX_DIM / 32; ++c)
        if (lane + 32 * c < p.head_dim && there) z += x[c] * to_f32(k[lane + 32 * c]);
#pragma unroll
      for (int b = 16; b > 0; b >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, b);
      const float top = fmaxf(m, z), base = top == -INFINITY ? 0.0f : top;
      const float keep = expf(m - base), w = expf(z - base);
      m = top;
      l = l * keep + w;
#pragma unroll
      for (int c = 0; c < MAX_DIM / 32; ++c)
        o[c] = o[c] * keep + (lane + 32 * c < p.head_dim && there ? w * to_f32(v[lane + 32 * c]) : 0.0f);
    }
    T *out = static_cast<T *>(p.out) + row * p.ld_out + (long long)h * p.head_dim;
    const float r = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int c = 0; c < MAX_DIM / 32; ++c)
      if (lane + 32 * c < p.head_dim) out[lane + 32 * c] = from_f32<T>(o[c] * r);
  }
}

}  // namespace

cudaError_t launch_attention_any(const AttentionParams &p, cudaStream_t s) {
  const long long blocks = (p.seq.rows * p.heads + WARPS - 1) / WARPS;
  const dim3 grid((unsigned)(blocks < 148ll * 1024 ? blocks : 148ll * 1024));
  if (p.et == ET_BF16) return launch_overlapped(attention_any_kernel<__nv_bfloat16>, grid, dim3(WARPS * 32), 0, s, p);
  return launch_overlapped(attention_any_kernel<__half>, grid, dim3(WARPS * 32), 0, s, p);
}

}  // namespace elb
