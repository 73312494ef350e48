// Attention for every shape, on CUDA cores.
//
// A warp takes one head of one new token (attend_row) and goes over the keys that the token sees.  Bound by the reductions of each score over the
// lanes, some 40 instructions a key: 8192 tokens of 32 heads, causal, take 227 ms, where the tensor cores take 0.5.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"

namespace elb {

namespace {

constexpr int WARPS = 4, MAX_DIM = 256;

// One head of one row by a warp, lanes the channels, in fp32 on CUDA cores: with the running maximum m and sum l of the softmax and
// m' = max(m, s), l = l e^(m - m') + e^(s - m') and the same for the weighted sum of values.
// CHUNKS: of 32 channels
template <typename T, int CHUNKS>
__device__ __forceinline__ void attend_row(const AttentionParams &p, int s, const Sequence &seq, int row, int h, int lane) {
  const int keys = p.causal ? min(seq.length, seq.length - seq.n + (row - seq.first) + 1) : seq.length;
  const T *q = static_cast<const T *>(p.q) + row * p.ld_q + (long long)h * p.head_dim;
  const long long head = h / (p.heads / p.kv_heads) * p.ld_head;
  float x[CHUNKS], o[CHUNKS], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    x[c] = lane + 32 * c < p.head_dim ? to_f32(q[lane + 32 * c]) * p.scale : 0.0f;
    o[c] = 0.0f;
  }
#pragma unroll 1
  for (int j = 0; j < keys; ++j) {
    const long long place = place_of_key(p, s, j), at = place + head;
    const bool there = place >= 0;
    if (!there && lane == 0) report_status(p.status, ST_BAD_PAGE);
    const T *k = static_cast<const T *>(p.k) + at, *v = static_cast<const T *>(p.v) + at;
    float z = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (lane + 32 * c < p.head_dim && there) z += x[c] * to_f32(k[lane + 32 * c]);
#pragma unroll
    for (int b = 16; b > 0; b >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, b);
    const float top = fmaxf(m, z), base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base), w = expf(z - base);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      o[c] = o[c] * keep + (lane + 32 * c < p.head_dim && there ? w * to_f32(v[lane + 32 * c]) : 0.0f);
  }
  T *out = static_cast<T *>(p.out) + row * p.ld_out + (long long)h * p.head_dim;
  const float r = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    if (lane + 32 * c < p.head_dim) out[lane + 32 * c] = from_f32<T>(o[c] * r);
}

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) attention_any_kernel(const AttentionParams p) {
  const int lane = threadIdx.x & 31;
  griddep_launch_dependents();
  griddep_wait();
  const long long items = p.seq.rows * p.heads;
  for (long long i = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); i < items; i += (long long)gridDim.x * WARPS) {
    const int row = (int)(i / p.heads), h = (int)(i - (long long)row * p.heads);
    const int s = sequence_of_row(p.seq, row, lane);
    if (s < 0 || s >= p.seq.seqs) continue;                     // behind the last sequence
    attend_row<T, MAX_DIM / 32>(p, s, sequence_of(p.seq, s), row, h, lane);
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
