// What lies between two blocks of a transformer: the norm behind a block, its gate and scale, the residual sum and the norm
// in front of the next block, in one pass over the data.
//
//   s = r + scale * gate * post(x);   y = pre(s)
//
// A row's values stay in registers from the load to the last store, so that each tensor is read or written once: the bound
// is HBM for long calls and the chain load -> reductions -> store for short ones.  Layer norm takes its variance around the
// mean, from the registers, not from a difference of sums.  Rows of up to 1024 channels belong to a warp (no block
// barriers), longer ones to a block.
#include "ops.cuh"

namespace elb {

namespace {

// VEC consecutive elements, VEC = 8: 16-byte aligned
template <typename T, int VEC>
struct Raw {
  static constexpr int WORDS = VEC == 1 ? 1 : VEC * (int)sizeof(T) / 16;
  uint4 q[WORDS];
  T one;
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VEC == 1) one = *p;
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) q[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (VEC == 1) v[0] = to_f32(one);
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) v[i * 4 + j] = __uint_as_float(w[j]);
          else {
            const float2 f = unpack2<T>(w[j]);
            v[i * 8 + 2 * j] = f.x;
            v[i * 8 + 2 * j + 1] = f.y;
          }
        }
      }
    }
  }
  __device__ __forceinline__ static void store(T *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = from_f32<T>(v[0]);
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[i * 4 + j]);
          else w[j] = pack2<T>(v[i * 8 + 2 * j], v[i * 8 + 2 * j + 1]);
        }
        reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

template <int VEC>
__device__ __forceinline__ void load_w(float (&w)[VEC], const float *p) {
  if constexpr (VEC == 1) w[0] = *p;
  else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 f = reinterpret_cast<const float4 *>(p)[i];
      w[4 * i] = f.x; w[4 * i + 1] = f.y; w[4 * i + 2] = f.z; w[4 * i + 3] = f.w;
    }
  }
}

// Sum over the threads of a row.  `slot`: another one for each call of a kernel, so that one barrier is enough.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float (&part)[4][32], int slot) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[slot][warp] = v;
    __syncthreads();
    v = lane < warps ? part[slot][lane] : 0.0f;
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  }
  return v;
}

constexpr int WARP_ROWS = 4;    // rows of a block whose rows belong to warps

template <typename T, typename TR, int VEC, int ITEMS, bool WARP>
__global__ void __launch_bounds__(WARP ? WARP_ROWS * 32 : 1024) block_norm_kernel(const NormParams p) {
  __shared__ float part[4][32];
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x, step = (WARP ? 32 : blockDim.x) * VEC;
  const long long row = WARP ? (long long)blockIdx.x * WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const T *x = static_cast<const T *>(p.x) + row * p.ld_x;
  float v[ITEMS][VEC];
  Raw<TR, VEC> res[ITEMS];
  Raw<T, VEC> gate[ITEMS];
  {
    Raw<T, VEC> raw[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = lane * VEC + i * step;
      if (c < p.channels) {
        raw[i].load(x + c);
        if (p.res) res[i].load(static_cast<const TR *>(p.res) + row * p.ld_res + c);
        if (p.gate) gate[i].load(static_cast<const T *>(p.gate) + row / p.gate_rows * p.ld_gate + c);
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (lane * VEC + i * step < p.channels) raw[i].get(v[i]);
      else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
      }
    }
  }
  // v <- norm(v); values past the row are 0 and stay out of the sums
  auto norm = [&](int kind, float eps, const float *w, const float *b, int slot) {
    float mean = 0.0f, sq = 0.0f;
    if (kind == 2) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[i][j];
      mean = row_sum<WARP>(s, part, slot) / p.channels;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (lane * VEC + i * step < p.channels) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { v[i][j] -= mean; sq = fmaf(v[i][j], v[i][j], sq); }
      }
    const float by = 1.0f / sqrtf(row_sum<WARP>(sq, part, slot + 1) / p.channels + eps);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = lane * VEC + i * step;
      if (c < p.channels) {
        float wv[VEC];
        load_w<VEC>(wv, w + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = v[i][j] * by * wv[j];
        if (b) {
          load_w<VEC>(wv, b + c);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += wv[j];
        }
      }
    }
  };
  if (p.post != 0) norm(p.post, p.post_eps, p.post_w, p.post_b, 0);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = lane * VEC + i * step;
    if (c < p.channels) {
      float o[VEC];
      if (p.gate) {
        gate[i].get(o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= o[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= p.scale;
      if (p.res) {
        res[i].get(o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += o[j];
      }
      if (p.sum) Raw<TR, VEC>::store(static_cast<TR *>(p.sum) + row * p.ld_sum + c, v[i]);
    }
  }
  if (p.pre == 0 || !p.y) return;
  norm(p.pre, p.pre_eps, p.pre_w, p.pre_b, 2);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = lane * VEC + i * step;
    if (c < p.channels) Raw<T, VEC>::store(static_cast<T *>(p.y) + row * p.ld_y + c, v[i]);
  }
}

template <typename T, typename TR, int VEC, int ITEMS>
cudaError_t go(const NormParams &p, int threads, cudaStream_t s) {
  if (threads == 32) {
    if constexpr (VEC * ITEMS <= 32)
      block_norm_kernel<T, TR, VEC, ITEMS, true><<<(unsigned)((p.rows + WARP_ROWS - 1) / WARP_ROWS), WARP_ROWS * 32, 0, s>>>(p);
  } else {
    block_norm_kernel<T, TR, VEC, ITEMS, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename T, typename TR>
cudaError_t launch_as(const NormParams &p, cudaStream_t s) {
  auto whole = [](const void *q, long long ld) { return !q || ((reinterpret_cast<uintptr_t>(q) & 15) == 0 && ld % 8 == 0); };
  const bool vec = p.channels % 8 == 0 && whole(p.x, p.ld_x) && whole(p.res, p.ld_res) && whole(p.gate, p.ld_gate) &&
                   whole(p.sum, p.ld_sum) && whole(p.y, p.ld_y);
  const int n = vec ? p.channels / 8 : p.channels;              // loads of a row
  auto threads = [&](int items) { return ((n + items - 1) / items + 31) / 32 * 32; };
  if (vec) {
    if (n <= 32) return go<T, TR, 8, 1>(p, 32, s);
    if (n <= 64) return go<T, TR, 8, 2>(p, 32, s);
    if (n <= 128) return go<T, TR, 8, 4>(p, 32, s);
    if (n <= 2048) return go<T, TR, 8, 2>(p, threads(2), s);
    return go<T, TR, 8, 4>(p, threads(4), s);
  }
  if (n <= 32) return go<T, TR, 1, 1>(p, 32, s);
  if (n <= 128) return go<T, TR, 1, 4>(p, 32, s);
  if (n <= 512) return go<T, TR, 1, 16>(p, 32, s);
  if (n <= 1024) return go<T, TR, 1, 32>(p, 32, s);
  if (n <= 4096) return go<T, TR, 1, 4>(p, threads(4), s);
  if (n <= 16384) return go<T, TR, 1, 16>(p, threads(16), s);
  return go<T, TR, 1, 32>(p, threads(32), s);
}

__global__ void norm_vector_kernel(float *dst, const void *src, int et, int n, float offset) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  dst[i] = !src ? 1.0f
         : offset + (et == ET_F32 ? static_cast<const float *>(src)[i]
                     : et == ET_BF16 ? to_f32(static_cast<const __nv_bfloat16 *>(src)[i]) : to_f32(static_cast<const __half *>(src)[i]));
}

}  // namespace

cudaError_t launch_norm_vector(float *dst, const void *src, int et, int n, float offset, cudaStream_t s) {
  norm_vector_kernel<<<(n + 255) / 256, 256, 0, s>>>(dst, src, et, n, offset);
  return cudaGetLastError();
}

cudaError_t launch_block_norm(const NormParams &p, cudaStream_t s) {
  if (p.et == ET_F32) return launch_as<float, float>(p, s);
  if (p.et == ET_BF16) return p.et_res == ET_F32 ? launch_as<__nv_bfloat16, float>(p, s) : launch_as<__nv_bfloat16, __nv_bfloat16>(p, s);
  return p.et_res == ET_F32 ? launch_as<__half, float>(p, s) : launch_as<__half, __half>(p, s);
}

}  // namespace elb
