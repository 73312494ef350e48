// Attention for every shape, on CUDA cores.
//
// A warp takes one head of one new token (attend_row) and goes over the keys that the token sees.  Bound by the reductions of each score over the
// lanes, some 40 instructions a key: 8192 tokens of 32 heads, causal, take 227 ms, where the tensor cores take 0.44.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"

namespace elb {

namespace {

constexpr int WARPS = 4, MAX_DIM = 256;

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
