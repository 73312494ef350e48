// Routing of tokens to experts: scores, a bias for the choice, groups, the top_k choices and their weights.
//
// One warp per row, lane l holding ITEMS neighbouring experts from l * ITEMS on.  A choice becomes a 32-bit key whose unsigned order
// is the floats' order; each lane keeps its best, so that the best of a row is one redux, and the lowest lane among equals has
// the lowest index.  The bound is the warps' instructions, about a thousand a row, not the logits' bytes: 16384 rows of 256
// experts, 4 of 8 groups, top 8, take 18.5 us, the logits' bytes 2.6; with experts dealt to the lanes in turn and a group
// searched by one lane 34.
#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

namespace {

constexpr int WARPS = 4;

__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);                 // -0 counts as 0
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);      // larger than 0 for every value, -inf too
}

// The key of an expert of a closed group: below an open one's whose choice is -inf.  top_k is at most the open experts, so it is never taken.
constexpr uint32_t SHUT_KEY = 1u;

// the two best of (a, b) and (c, d), a >= b and c >= d
__device__ __forceinline__ void merge2(float &a, float &b, float c, float d) {
  b = fmaxf(fminf(a, c), fmaxf(b, d));
  a = fmaxf(a, c);
}

template <typename T, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const RouteParams p) {
  constexpr int PAD = ITEMS < 4 ? ITEMS : ITEMS + 1;            // of a lane in shared memory, against bank conflicts
  __shared__ float all[WARPS][32 * PAD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * ITEMS;
  const long long row = (long long)blockIdx.x * WARPS + warp;
  const bool full = e0 + ITEMS <= p.experts;
  float bias[ITEMS];
  if (p.bias) {
    if (ITEMS >= 4 && full) {                                   // (the plan's own vector, aligned)
#pragma unroll
      for (int i = 0; i < ITEMS / 4; ++i) *reinterpret_cast<float4 *>(bias + 4 * i) = reinterpret_cast<const float4 *>(p.bias + e0)[i];
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) bias[i] = e0 + i < p.experts ? p.bias[e0 + i] : 0.0f;
    }
  }
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows) return;
  const T *z = static_cast<const T *>(p.logits) + row * p.ld;
  float score[ITEMS], whole = 1.0f;
  constexpr int WORDS = ITEMS * (int)sizeof(T) / 16;
  if (WORDS > 0 && p.words && full) {
    uint4 q[WORDS > 0 ? WORDS : 1];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) q[i] = reinterpret_cast<const uint4 *>(z + e0)[i];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) score[i] = to_f32(reinterpret_cast<const T *>(q)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) score[i] = e0 + i < p.experts ? to_f32(z[e0 + i]) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) score[i] = fmaxf(score[i], -INFINITY);        // (a NaN becomes -inf)
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) score[i] = __frcp_rn(1.0f + expf(-score[i]));
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) top = fmaxf(top, score[i]);
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
  for (int i = 0; i < ITEMS; ++i) choice[i] = score[i];
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      choice[i] = fmaxf((p.sigmoid || !(whole > 0.0f) ? score[i] : score[i] / whole) + bias[i], -INFINITY);
    }
  }
  if (!full) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (e0 + i >= p.experts) choice[i] = -INFINITY;
  }
  float *mine = all[warp];                                      // the row's choices, later its scores
  uint32_t shut = 0;                                            // of this lane's experts
  if (p.groups > 1) {
    const int size = p.experts / p.groups;
    float a = -INFINITY, b = -INFINITY;                         // the two best of group `lane`
    if (p.lanes_per_group > 0) {
      // a group is a power of two of whole lanes
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) merge2(a, b, choice[i], -INFINITY);
      for (int d = 1; d < p.lanes_per_group; d <<= 1) {
        const float c = __shfl_xor_sync(0xFFFFFFFFu, a, d), e = __shfl_xor_sync(0xFFFFFFFFu, b, d);
        merge2(a, b, c, e);
      }
      const int from = (lane * p.lanes_per_group) & 31;
      a = __shfl_sync(0xFFFFFFFFu, a, from);
      b = __shfl_sync(0xFFFFFFFFu, b, from);
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) mine[lane * PAD + i] = choice[i];
      __syncwarp();
      if (lane < p.groups)
        for (int e = lane * size; e < (lane + 1) * size; ++e) merge2(a, b, mine[e / ITEMS * PAD + e % ITEMS], -INFINITY);
    }
    uint32_t key = lane < p.groups ? order_key(p.group_best == 2 && size > 1 ? a + b : a) : 0u;
    uint32_t open = 0;
    for (int j = 0; j < p.top_groups; ++j) {
      const uint32_t best = __reduce_max_sync(0xFFFFFFFFu, key);
      const int who = __ffs(__ballot_sync(0xFFFFFFFFu, key == best)) - 1;
      open |= 1u << who;
      if (lane == who) key = 0u;
    }
    if (p.lanes_per_group > 0) {
      if (!((open >> (lane / p.lanes_per_group)) & 1u)) shut = 0xFFFFFFFFu;
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (!((open >> min((e0 + i) / size, 31)) & 1u)) shut |= 1u << i;
    }
  }
  uint32_t key[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) key[i] = order_key(choice[i]);
  if (shut) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if ((shut >> i) & 1u) key[i] = SHUT_KEY;
  }
  if (!full) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (e0 + i >= p.experts) key[i] = 0u;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) mine[lane * PAD + i] = score[i];
  __syncwarp();
  // This lane's best and second best, the lower index first among equals.  A lane seldom gives more than two of the top_k, so
  // that its experts are searched once, and again only after both have gone.
  uint32_t best, second;
  int best_i, second_i;
  auto look = [&] {
    best = key[0];
    best_i = 0;
    second = 0u;
    second_i = 0;
#pragma unroll
    for (int i = 1; i < ITEMS; ++i) {
      if (key[i] > best) { second = best; second_i = best_i; best = key[i]; best_i = i; }
      else if (key[i] > second) { second = key[i]; second_i = i; }
    }
  };
  look();
  bool two = true;                                              // `second` is known
  uint32_t taken = 0;
  int id = 0;                                                   // lane j keeps the j-th choice
  for (int j = 0; j < p.top_k; ++j) {
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    const int who = __ffs(__ballot_sync(0xFFFFFFFFu, best == top)) - 1;
    const int e = __shfl_sync(0xFFFFFFFFu, e0 + best_i, who);
    if (lane == j) id = e;
    if (lane == who) {
      taken |= 1u << best_i;
      if (two) {
        best = second;
        best_i = second_i;
        two = false;
      } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if ((taken >> i) & 1u) key[i] = 0u;
        look();
        two = true;
      }
    }
  }
  float w = lane < p.top_k ? mine[id / ITEMS * PAD + id % ITEMS] : 0.0f, by = whole;
  if (p.renormalise) {
    by = w;
#pragma unroll
    for (int d = 16; d; d >>= 1) by += __shfl_xor_sync(0xFFFFFFFFu, by, d);
  }
  if (lane < p.top_k) {
    p.ids[row * p.top_k + lane] = id;
    if (p.weights) p.weights[row * p.top_k + lane] = by > 0.0f ? w / by * p.scale : 0.0f;
  }
}

template <typename T, int ITEMS>
cudaError_t go(RouteParams p, cudaStream_t s) {
  const int size = p.experts / p.groups, lanes = size / ITEMS;
  p.lanes_per_group = size % ITEMS == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  p.words = (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 && p.ld * sizeof(T) % 16 == 0;
  return launch_overlapped(route_kernel<T, ITEMS>, dim3((unsigned)((p.rows + WARPS - 1) / WARPS)), dim3(WARPS * 32), 0, s, p);
}
template <typename T>
cudaError_t launch_as(const RouteParams &p, cudaStream_t s) {
  const int items = (p.experts + 31) / 32;
  if (items <= 1) return go<T, 1>(p, s);
  if (items <= 2) return go<T, 2>(p, s);
  if (items <= 4) return go<T, 4>(p, s);
  if (items <= 8) return go<T, 8>(p, s);
  if (items <= 16) return go<T, 16>(p, s);
  return go<T, 32>(p, s);
}

}  // namespace

cudaError_t launch_route(const RouteParams &p, cudaStream_t s) {
  if (p.et == ET_F32) return launch_as<float>(p, s);
  if (p.et == ET_BF16) return launch_as<__nv_bfloat16>(p, s);
  return launch_as<__half>(p, s);
}

}  // namespace elb
