// Routing of tokens to experts: scores, a bias for the choice, groups, the top_k choices and their weights.
//
// One warp per row, lane l holding experts l, l + 32, ...  A choice becomes a 32-bit key whose unsigned order is the
// floats' order, so that the best of a row is one redux over the lanes' own best, and among equals the lowest index another.
#include "ops.cuh"

namespace elb {

namespace {

constexpr int WARPS = 4;

__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);                 // -0 counts as 0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;              // larger than 0 for every value, -inf too
}

// ITEMS: experts per lane
template <typename T, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const RouteParams p) {
  __shared__ float group_choice[WARPS][ITEMS * 33];             // [expert + expert / 32]: neighbouring groups fall on other banks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * WARPS + warp;
  if (row >= p.rows) return;
  const T *z = static_cast<const T *>(p.logits) + row * p.ld;
  float score[ITEMS], whole = 1.0f;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int e = lane + 32 * i;
    float v = e < p.experts ? to_f32(z[e]) : -INFINITY;
    if (v != v) v = -INFINITY;
    score[i] = v;
    top = fmaxf(top, v);
  }
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) score[i] = 1.0f / (1.0f + expf(-score[i]));
  } else {
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    whole = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      score[i] = score[i] == -INFINITY ? 0.0f : score[i] == top ? 1.0f : expf(score[i] - top);
      whole += score[i];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) whole += __shfl_xor_sync(0xFFFFFFFFu, whole, d);
  }
  // Without a bias softmax chooses by its numerators, whose order is that of the scores; with one the scores themselves count.
  float choice[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int e = lane + 32 * i;
    choice[i] = score[i];
    if (p.bias && e < p.experts) choice[i] = (p.sigmoid || !(whole > 0.0f) ? score[i] : score[i] / whole) + p.bias[e];
    if (choice[i] != choice[i]) choice[i] = -INFINITY;
  }
  if (p.groups > 1) {
    float *mine = group_choice[warp];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) mine[lane + 33 * i] = choice[i];
    __syncwarp();
    const int size = p.experts / p.groups;
    float a = -INFINITY, b = -INFINITY;                         // the two best of group `lane`
    if (lane < p.groups)
      for (int j = 0; j < size; ++j) {
        const int e = lane * size + j;
        const float v = mine[e + (e >> 5)];
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
      }
    uint32_t key = lane < p.groups ? order_key(p.group_best == 2 && size > 1 ? a + b : a) : 0u;
    uint32_t open = 0;
    for (int j = 0; j < p.top_groups; ++j) {
      const uint32_t best = __reduce_max_sync(0xFFFFFFFFu, key);
      const int who = __ffs(__ballot_sync(0xFFFFFFFFu, key == best)) - 1;
      open |= 1u << who;
      if (lane == who) key = 0u;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts && !((open >> (e / size)) & 1u)) choice[i] = -INFINITY;
    }
  }
  uint32_t key[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) key[i] = lane + 32 * i < p.experts ? order_key(choice[i]) : 0u;
  int my_id = 0;                                                // lane j keeps the j-th choice
  float my_w = 0.0f, sum = 0.0f;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xFFFFFFFFu, best);
    uint32_t e = 0xFFFFFFFFu;
#pragma unroll
    for (int i = ITEMS - 1; i >= 0; --i)
      if (key[i] == best) e = lane + 32 * i;
    e = __reduce_min_sync(0xFFFFFFFFu, e);
    float w = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (lane + 32 * i == (int)e) { w = score[i]; key[i] = 0u; }
    w = __shfl_sync(0xFFFFFFFFu, w, e & 31u);
    sum += w;
    if (lane == j) { my_id = (int)e; my_w = w; }
  }
  if (lane < p.top_k) {
    const float by = p.renormalise ? sum : whole;
    p.ids[row * p.top_k + lane] = my_id;
    if (p.weights) p.weights[row * p.top_k + lane] = by > 0.0f ? my_w / by * p.scale : 0.0f;
  }
}

template <typename T>
cudaError_t launch_as(const RouteParams &p, cudaStream_t s) {
  const unsigned blocks = (unsigned)((p.rows + WARPS - 1) / WARPS);
  const int items = (p.experts + 31) / 32;
  if (items <= 1) route_kernel<T, 1><<<blocks, WARPS * 32, 0, s>>>(p);
  else if (items <= 2) route_kernel<T, 2><<<blocks, WARPS * 32, 0, s>>>(p);
  else if (items <= 4) route_kernel<T, 4><<<blocks, WARPS * 32, 0, s>>>(p);
  else if (items <= 8) route_kernel<T, 8><<<blocks, WARPS * 32, 0, s>>>(p);
  else if (items <= 16) route_kernel<T, 16><<<blocks, WARPS * 32, 0, s>>>(p);
  else route_kernel<T, 32><<<blocks, WARPS * 32, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_route(const RouteParams &p, cudaStream_t s) {
  if (p.et == ET_F32) return launch_as<float>(p, s);
  if (p.et == ET_BF16) return launch_as<__nv_bfloat16>(p, s);
  return launch_as<__half>(p, s);
}

}  // namespace elb
