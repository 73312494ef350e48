// What lies around the experts' products: slots (a token and one of its experts) are sorted by expert, their tokens'
// rows are brought together, and the products' rows are summed per token with the router's weights.
#include "ops.cuh"

namespace elb {

namespace {

constexpr int SORT_THREADS = 1024, MAX_EXPERTS = 1024;

// One block: counts, offsets and token tiles of the experts, and each slot's place.  Places within an expert are handed out
// by atomics, in no fixed order: a slot's product does not depend on its place, and the sum over a token's slots goes by
// the slots' own order.
__global__ void __launch_bounds__(SORT_THREADS) experts_sort_kernel(const ExpertsParams p) {
  __shared__ int count[MAX_EXPERTS], next[MAX_EXPERTS];
  __shared__ int warp_rows[32], warp_tiles[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slots = p.rows * p.top_k;
  count[tid] = 0;
  __syncthreads();
  for (int i = tid; i < slots; i += SORT_THREADS) {
    const int e = p.ids[i];
    if (e >= 0 && e < p.experts) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  const int c = count[tid], t = (c + p.tile_tokens - 1) / p.tile_tokens;
  int rows = c, tiles = t;                             // inclusive sums over the experts
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xFFFFFFFFu, rows, d), b = __shfl_up_sync(0xFFFFFFFFu, tiles, d);
    if (lane >= d) { rows += a; tiles += b; }
  }
  if (lane == 31) { warp_rows[warp] = rows; warp_tiles[warp] = tiles; }
  __syncthreads();
  if (warp == 0) {
    int a = warp_rows[lane], b = warp_tiles[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, a, d), y = __shfl_up_sync(0xFFFFFFFFu, b, d);
      if (lane >= d) { a += x; b += y; }
    }
    warp_rows[lane] = a;
    warp_tiles[lane] = b;
  }
  __syncthreads();
  if (warp > 0) { rows += warp_rows[warp - 1]; tiles += warp_tiles[warp - 1]; }
  const int row0 = rows - c, tile0 = tiles - t;
  next[tid] = row0;
  for (int i = 0; i < t; ++i)
    p.tiles[tile0 + i] = GroupTile{tid, row0 + i * p.tile_tokens, min(p.tile_tokens, c - i * p.tile_tokens), 0};
  if (tid == SORT_THREADS - 1) { *p.n_rows = rows; *p.n_tiles = tiles; }
  __syncthreads();
  for (int i = tid; i < slots; i += SORT_THREADS) {
    const int e = p.ids[i];
    int at = -1;
    if (e >= 0 && e < p.experts) {
      at = atomicAdd(&next[e], 1);
      p.src[at] = i / p.top_k;
    }
    p.pos[i] = at;
  }
}

__global__ void experts_gather_kernel(const ExpertsParams p) {
  const int r = blockIdx.x;
  if (r >= *p.n_rows) return;
  const uint16_t *from = static_cast<const uint16_t *>(p.x) + p.src[r] * p.ld_x;
  uint16_t *to = static_cast<uint16_t *>(p.xs) + r * p.pitch_x;
  for (int i = threadIdx.x; i < p.ic; i += blockDim.x) to[i] = from[i];
}

template <typename T>
__global__ void experts_combine_kernel(const ExpertsParams p) {
  const int t = blockIdx.x;
  T *out = static_cast<T *>(p.out) + t * p.ld_out;
  for (int i = threadIdx.x; i < p.ic; i += blockDim.x) {
    float s = 0.0f;
    for (int j = 0; j < p.top_k; ++j) {
      const int at = p.pos[t * p.top_k + j];
      if (at >= 0) s = fmaf(p.weights[t * p.top_k + j], p.y[at * p.pitch_y + i], s);
    }
    out[i] = from_f32<T>(s);
  }
}

}  // namespace

cudaError_t launch_experts_sort(const ExpertsParams &p, cudaStream_t s) {
  experts_sort_kernel<<<1, SORT_THREADS, 0, s>>>(p);
  return cudaGetLastError();
}
cudaError_t launch_experts_gather(const ExpertsParams &p, cudaStream_t s) {
  experts_gather_kernel<<<p.rows * p.top_k, 128, 0, s>>>(p);
  return cudaGetLastError();
}
cudaError_t launch_experts_combine(const ExpertsParams &p, cudaStream_t s) {
  if (p.et == ET_BF16) experts_combine_kernel<__nv_bfloat16><<<p.rows, 256, 0, s>>>(p);
  else experts_combine_kernel<__half><<<p.rows, 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace elb
