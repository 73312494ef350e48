// What lies around the experts' products: slots (a token and one of its experts) are sorted by expert, their tokens'
// rows are brought together, and the products' rows are summed per token with the router's weights.
#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

namespace {

constexpr int MAX_EXPERTS = 1024, COUNT_THREADS = 256, COUNT_SLOTS = 2048;   // slots that a block counts

// Each slot's place among those of its expert, and how many an expert has (p.count, zero before the call).  Places are handed
// out by atomics, in no fixed order: a slot's product does not depend on its place, and the sum over a token's slots goes by the
// slots' own order.
__global__ void __launch_bounds__(COUNT_THREADS) experts_count_kernel(const ExpertsParams p) {
  __shared__ int count[MAX_EXPERTS];
  griddep_launch_dependents();
  const int slots = p.rows * p.top_k, first = blockIdx.x * COUNT_SLOTS;
  for (int i = threadIdx.x; i < p.experts; i += COUNT_THREADS) count[i] = 0;
  __syncthreads();
  griddep_wait();
  constexpr int EACH = COUNT_SLOTS / COUNT_THREADS;
  int e[EACH], at[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = first + j * COUNT_THREADS + threadIdx.x;
    e[j] = i < slots ? p.ids[i] : -1;
    if (e[j] >= p.experts) e[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) at[j] = e[j] >= 0 ? atomicAdd(&count[e[j]], 1) : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.experts; i += COUNT_THREADS)
    if (count[i]) count[i] = atomicAdd(&p.count[i], count[i]);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = first + j * COUNT_THREADS + threadIdx.x;
    if (i < slots) p.pos[i] = e[j] >= 0 ? count[e[j]] + at[j] : -1;
  }
}

// Rows of the experts lie behind one another.  Every block adds up the counts for itself, brings its slots' rows to their
// places and notes these; the first writes the list of token tiles.
// COUNT: few slots, which every block counts for itself, places and all, in the slots' order; there is no kernel before it.
constexpr int GATHER_THREADS = 256, COUNT_HERE = 2048;
template <bool WORDS, bool COUNT>                      // WORDS: rows in 16-byte words
__global__ void __launch_bounds__(GATHER_THREADS) experts_gather_kernel(const ExpertsParams p, const SlotShare share) {
  __shared__ int row0[MAX_EXPERTS];
  __shared__ int2 part[GATHER_THREADS / 32];
  __shared__ short ids[COUNT ? COUNT_HERE : 1];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slots = p.rows * p.top_k;
  if (COUNT) {
    for (int e = tid; e < p.experts; e += GATHER_THREADS) row0[e] = 0;
    __syncthreads();
    for (int i = tid; i < slots; i += GATHER_THREADS) {
      const int e = p.ids[i];
      ids[i] = (short)(e >= 0 && e < p.experts ? e : -1);
      if (e >= 0 && e < p.experts) atomicAdd(&row0[e], 1);
    }
    __syncthreads();
  }
  constexpr int EACH = MAX_EXPERTS / GATHER_THREADS;   // experts of a thread, neighbours
  int c[EACH], rows = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int e = tid * EACH + j;
    c[j] = e >= p.experts ? 0 : COUNT ? row0[e] : p.count[e];
    rows += c[j];
    tiles += (c[j] + p.tile_tokens - 1) / p.tile_tokens;
  }
  int2 sum = make_int2(rows, tiles);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xFFFFFFFFu, sum.x, d), b = __shfl_up_sync(0xFFFFFFFFu, sum.y, d);
    if (lane >= d) { sum.x += a; sum.y += b; }
  }
  if (lane == 31) part[warp] = sum;
  __syncthreads();
  for (int w = 0; w < warp; ++w) { sum.x += part[w].x; sum.y += part[w].y; }
  int r = sum.x - rows, t = sum.y - tiles;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int e = tid * EACH + j;
    row0[e] = r;
    if (blockIdx.x == 0 && c[j] > 0) {
      // tiles of equal size
      const int n = (c[j] + p.tile_tokens - 1) / p.tile_tokens, size = (c[j] + n - 1) / n;
      for (int i = 0; i < n; ++i) p.tiles[t + i] = GroupTile{e, r + i * size, min(size, c[j] - i * size), 0};
      t += n;
    }
    r += c[j];
  }
  if (blockIdx.x == 0 && tid == GATHER_THREADS - 1) *p.n_tiles = t;
  __syncthreads();
  // a warp per slot
  const int end = share.end(blockIdx.x, slots);
  for (int i = share.first(blockIdx.x) + warp; i < end; i += GATHER_THREADS / 32) {
    const int e = COUNT ? ids[i] : p.ids[i];
    if (e < 0 || e >= p.experts) continue;
    int place = 0;
    if (COUNT) {
      for (int k = lane; k < i; k += 32) place += ids[k] == e;
      place = __reduce_add_sync(0xFFFFFFFFu, place);
    } else {
      place = p.pos[i];
    }
    const long long to = row0[e] + place, from = i / p.top_k;
    __syncwarp();
    if (lane == 0) p.place[i] = (int)to;
    if (WORDS) {
      const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.x) + from * p.ld_x);
      uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.xs) + to * p.pitch_x);
      const int n = p.ic / 8;
      int k = lane;
      for (; k + 96 < n; k += 128) {
        const uint4 a = src[k], b = src[k + 32], c4 = src[k + 64], d = src[k + 96];
        dst[k] = a; dst[k + 32] = b; dst[k + 64] = c4; dst[k + 96] = d;
      }
      for (; k < n; k += 32) dst[k] = src[k];
    } else {
      const uint16_t *src = static_cast<const uint16_t *>(p.x) + from * p.ld_x;
      uint16_t *dst = static_cast<uint16_t *>(p.xs) + to * p.pitch_x;
      for (int k = lane; k < p.ic; k += 32) dst[k] = src[k];
    }
  }
}

// A block per token, a thread per four channels (one, where the output's rows are not aligned).
constexpr int COMBINE_THREADS = 256;
template <typename T, bool WORDS>
__global__ void __launch_bounds__(COMBINE_THREADS) experts_combine_kernel(const ExpertsParams p) {
  __shared__ int at[32];
  __shared__ float by[32];
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.x;
  if (threadIdx.x < p.top_k) {
    const int i = t * p.top_k + threadIdx.x, e = p.ids[i];
    at[threadIdx.x] = e >= 0 && e < p.experts ? p.place[i] : -1;
    by[threadIdx.x] = p.weights[i];
  }
  if (blockIdx.x == 0 && p.clear)                      // for the next call
    for (int i = threadIdx.x; i < p.experts; i += COMBINE_THREADS) p.count[i] = 0;
  __syncthreads();
  T *out = static_cast<T *>(p.out) + t * p.ld_out;
  if (WORDS) {
    for (int c = threadIdx.x * 4; c < p.ic; c += COMBINE_THREADS * 4) {
      float s[4] = {};
#pragma unroll 8
      for (int j = 0; j < p.top_k; ++j)
        if (at[j] >= 0) {
          const float4 y = __ldcs(reinterpret_cast<const float4 *>(p.y + at[j] * p.pitch_y + c));
          s[0] = fmaf(by[j], y.x, s[0]); s[1] = fmaf(by[j], y.y, s[1]);
          s[2] = fmaf(by[j], y.z, s[2]); s[3] = fmaf(by[j], y.w, s[3]);
        }
      *reinterpret_cast<uint2 *>(out + c) = make_uint2(pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3]));
    }
  } else {
    for (int c = threadIdx.x; c < p.ic; c += COMBINE_THREADS) {
      float s = 0.0f;
      for (int j = 0; j < p.top_k; ++j)
        if (at[j] >= 0) s = fmaf(by[j], p.y[at[j] * p.pitch_y + c], s);
      out[c] = from_f32<T>(s);
    }
  }
}

}  // namespace

bool experts_count_here(int slots) { return slots <= COUNT_HERE; }
cudaError_t launch_experts_count(const ExpertsParams &p, cudaStream_t s) {
  const int slots = p.rows * p.top_k;
  return launch_overlapped(experts_count_kernel, dim3((slots + COUNT_SLOTS - 1) / COUNT_SLOTS), dim3(COUNT_THREADS), 0, s, p);
}
cudaError_t launch_experts_gather(const ExpertsParams &p, int num_sms, cudaStream_t s) {
  const int slots = p.rows * p.top_k;
  const SlotShare share = share_slots(slots, GATHER_THREADS / 32, num_sms * 8);
  const bool words = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.ld_x % 8 == 0 && p.ic % 8 == 0;
  const bool here = experts_count_here(slots);
  auto k = words ? (here ? experts_gather_kernel<true, true> : experts_gather_kernel<true, false>)
                 : (here ? experts_gather_kernel<false, true> : experts_gather_kernel<false, false>);
  return launch_overlapped(k, dim3(share.blocks), dim3(GATHER_THREADS), 0, s, p, share);
}
cudaError_t launch_experts_combine(const ExpertsParams &p, cudaStream_t s) {
  const bool words = (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && p.ld_out % 4 == 0 && p.ic % 4 == 0;
  auto k = p.et == ET_BF16 ? (words ? experts_combine_kernel<__nv_bfloat16, true> : experts_combine_kernel<__nv_bfloat16, false>)
                           : (words ? experts_combine_kernel<__half, true> : experts_combine_kernel<__half, false>);
  return launch_overlapped(k, dim3(p.rows), dim3(COMBINE_THREADS), 0, s, p);
}

}  // namespace elb
