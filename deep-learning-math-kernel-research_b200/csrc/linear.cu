// Matrix products of the transformer operators, dense and grouped by expert, on packed weights (ops.cuh).
#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

namespace {

// One thread per 16-byte chunk of the packed image.
__global__ void pack_weights_kernel(uint4 *dst, const uint16_t *src, int rows, int ic, int kt, int row_tiles, int gated, int hwio,
                                    long long chunks, long long per_expert) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < chunks; i += (long long)gridDim.x * blockDim.x) {
    const long long e = i / per_expert;
    long long r = i - e * per_expert;
    const int slot = (int)(r & 7);
    r >>= 3;
    const int in_tile = (int)(r & (GT_ROWS - 1));
    r >>= 7;
    const int k_tile = (int)(r % kt), row_tile = (int)(r / kt);
    const int p = row_tile * GT_ROWS + in_tile;                          // packed row
    const int row = gated ? (p & 1) * (rows >> 1) + (p >> 1) : p;        // row of the source
    const int k0 = k_tile * GT_K + ((slot ^ (in_tile & 7)) << 3);
    uint16_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = k0 + j;
      v[j] = 0;
      if (p < rows && k < ic)
        v[j] = hwio ? src[(e * ic + k) * rows + row] : src[(e * rows + row) * (long long)ic + k];
    }
    dst[i] = *reinterpret_cast<uint4 *>(v);
  }
}

__global__ void pack_bias_kernel(float *dst, const void *src, int et, int rows, int padded, int gated) {
  const int p = blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= padded) return;
  float v = 0.0f;
  if (p < rows) {
    const int row = gated ? (p & 1) * (rows >> 1) + (p >> 1) : p;
    v = et == ET_F32 ? static_cast<const float *>(src)[row]
      : et == ET_BF16 ? to_f32(static_cast<const __nv_bfloat16 *>(src)[row]) : to_f32(static_cast<const __half *>(src)[row]);
  }
  dst[p] = v;
}

// The plain form on CUDA cores: a block multiplies 128 packed rows (one per thread) by up to 16 tokens, whose channels lie in
// shared memory as fp32, tile by tile of 64.
__global__ void __launch_bounds__(GT_ROWS) gemm_simple_kernel(const GemmParams p) {
  __shared__ float xt[GEMM_TOKENS][GT_K];
  const int row_tile = blockIdx.x % p.row_tiles, tt = blockIdx.x / p.row_tiles;
  int tok0 = tt * GEMM_TOKENS, ntok = min(GEMM_TOKENS, p.rows - tok0);
  const uint8_t *w = p.w;
  if (p.tiles) {
    if (tt >= *p.n_tiles) return;
    const GroupTile g = p.tiles[tt];
    tok0 = g.row0;
    ntok = g.count;
    w += g.expert * p.w_stride;
  }
  w += (size_t)row_tile * p.kt * GT_BYTES;
  const uint16_t *x = static_cast<const uint16_t *>(p.x) + (long long)tok0 * p.ld_x;
  const int r = threadIdx.x;
  float acc[GEMM_TOKENS] = {};
  auto value = [&](uint16_t b) {
    return p.in_et == ET_BF16 ? __uint_as_float((uint32_t)b << 16) : __half2float(__ushort_as_half(b));
  };
  for (int kt = 0; kt < p.kt; ++kt) {
    __syncthreads();
    for (int i = threadIdx.x; i < GEMM_TOKENS * GT_K; i += GT_ROWS) {
      const int t = i / GT_K, k = i % GT_K;
      xt[t][k] = t < ntok && kt * GT_K + k < p.ic ? value(x[t * p.ld_x + kt * GT_K + k]) : 0.0f;
    }
    __syncthreads();
    const uint4 *wr = reinterpret_cast<const uint4 *>(w + (size_t)kt * GT_BYTES + r * 128);
    for (int c = 0; c < 8; ++c) {
      const uint4 q = wr[c ^ (r & 7)];
      const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float wv = value((uint16_t)(words[j >> 1] >> (16 * (j & 1))));
#pragma unroll
        for (int t = 0; t < GEMM_TOKENS; ++t) acc[t] = fmaf(wv, xt[t][c * 8 + j], acc[t]);
      }
    }
  }
  emit<GEMM_TOKENS>(p.epi, acc, row_tile * GT_ROWS + r, tok0, ntok);
}

}  // namespace

cudaError_t launch_pack_weights(void *dst, const void *src, int experts, int rows, int ic, bool gated, bool hwio, cudaStream_t s) {
  const int kt = (ic + GT_K - 1) / GT_K, row_tiles = (rows + GT_ROWS - 1) / GT_ROWS;
  const long long per = (long long)row_tiles * kt * GT_ROWS * 8, chunks = per * experts;
  const int blocks = (int)(chunks / 256 + 1 < 148 * 64 ? chunks / 256 + 1 : 148 * 64);
  pack_weights_kernel<<<blocks, 256, 0, s>>>(static_cast<uint4 *>(dst), static_cast<const uint16_t *>(src), rows, ic, kt, row_tiles,
                                             gated, hwio, chunks, per);
  return cudaGetLastError();
}

cudaError_t launch_pack_bias(float *dst, const void *src, int et, int rows, int padded, bool gated, cudaStream_t s) {
  pack_bias_kernel<<<(padded + 255) / 256, 256, 0, s>>>(dst, src, et, rows, padded, gated);
  return cudaGetLastError();
}

cudaError_t launch_gemm(const GemmParams &p, int num_sms, cudaStream_t s) {
  (void)num_sms;
  const long long tt = p.tiles ? p.max_tiles : (p.rows + GEMM_TOKENS - 1) / GEMM_TOKENS;
  gemm_simple_kernel<<<(unsigned)(tt * p.row_tiles), GT_ROWS, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace elb
