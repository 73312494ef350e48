// The products for a handful of tokens: matrix times vector on CUDA cores, over the same packed weights (ops.cuh) as linear.cu.
//
// A call reads its weights once and that is its time, so what counts is to have all of them on their way at once and few steps
// behind them: a block owns four or eight packed rows, its warps share the channels, every thread has eight 16-byte loads in
// flight before it needs the first, and the loads of a dense call are issued before the kernel in front of it has ended.  No
// tensor memory, clusters or barriers in memory: 1 x 4096 -> 4096 takes the tensor-core kernel 10.7 us a call in a stream of
// calls, most of it set-up and hand-overs.
#include <type_traits>

#include "elb_common.cuh"
#include "gemm_epilogue.cuh"
#include "ops.cuh"

namespace elb {

namespace {

constexpr int MAX_WARPS = 8;
constexpr int LOADS = 8;          // of a thread at a time: packed rows of a block x steps (a warp's 256 channels) that are issued together

struct GemvParams {
  const uint8_t *w;
  size_t w_stride;
  const void *x;                // operands' type; fp32 in the experts' second product
  long long ld_x;
  int rows, ic, kt, words;      // words: rows of x are 16-byte aligned
  const int *ids;               // experts: of each slot; null: dense
  const float *share;           // experts, second product: the router's weights; its blocks sum over the slots of a token
  int top_k, experts;
  Epilogue epi;
};

// Two fp32 values in a 64-bit register, and a multiply-add on both: each half rounds as fmaf does
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum2(uint64_t a) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a));
  return lo + hi;
}
template <typename E>
__device__ __forceinline__ void unpack8(const uint4 &q, uint64_t (&f)[4]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<E>(w[i]);
    f[i] = both(v.x, v.y);
  }
}

// packed row i of a block's, which are as many channels or, gated, the gates and then the ups of half as many
template <bool GATED, int ROWS>
__device__ __forceinline__ int row_of(int block, int i) {
  constexpr int H = ROWS / 2;
  return GATED ? block * H / 8 * 16 + block * H % 8 + i % H + i / H * 8 : block * ROWS + i;
}

// eight values of a row of x from channel k; past the end zeros
template <typename X>
__device__ __forceinline__ void load_x(uint64_t (&f)[4], const X *x, int k, int ic, bool words) {
  if (words && k + 8 <= ic) {
    if constexpr (sizeof(X) == 2) {
      unpack8<X>(*reinterpret_cast<const uint4 *>(x + k), f);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 q = reinterpret_cast<const float4 *>(x + k)[i];
        f[2 * i] = both(q.x, q.y);
        f[2 * i + 1] = both(q.z, q.w);
      }
    }
    return;
  }
  auto one = [&](int i) { return k + i < ic ? to_f32(x[k + i]) : 0.0f; };
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = both(one(2 * i), one(2 * i + 1));
}

// E: element type of the operands; T: tokens of a block (1 for experts); MODE 0 dense (a block per T tokens), 1 an expert's first product (a block per
// slot), 2 the second (a block per token)
template <typename E, typename OT, int T, bool GATED, int MODE, int ROWS>
__global__ void __launch_bounds__(MAX_WARPS * 32, T == 1 ? 3 : 2) gemv_kernel(const __grid_constant__ GemvParams p) {
  constexpr int UNROLL = LOADS / ROWS;
  __shared__ float part[MAX_WARPS][ROWS * T];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int groups = (p.kt + 3) / 4, chunk = lane & 7;
  // (a block's rows lie in one tile: its numbers of rows and channels divide a tile's)
  const int row0 = row_of<GATED, ROWS>(blockIdx.x, 0);
  const uint8_t *wr = p.w + (size_t)(row0 >> 7) * p.kt * GT_BYTES;
  auto in_tile = [&](int i) {
    const int r = row_of<GATED, ROWS>(blockIdx.x, i) & 127;
    return r * 128 + ((chunk ^ (r & 7)) << 4);
  };
  using X = std::conditional_t<MODE == 2, float, E>;
  uint64_t acc[T][ROWS] = {};
  griddep_launch_dependents();
  if (MODE != 0) griddep_wait();                                // (the experts come from the router)
  const int first = MODE == 2 ? blockIdx.y * p.top_k : blockIdx.y, slots = MODE == 2 ? p.top_k : 1;
  const int steps = groups * slots;
  bool waited = MODE != 0;
  for (int s0 = warp; s0 < steps; s0 += warps * UNROLL) {
    uint4 w[UNROLL][ROWS];
    bool live[UNROLL];
    int kt[UNROLL], slot[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int s = s0 + u * warps;
      slot[u] = MODE == 2 ? s / groups : 0;
      kt[u] = (MODE == 2 ? s - slot[u] * groups : s) * 4 + (lane >> 3);
      live[u] = s < steps && kt[u] < p.kt;
      size_t at = (size_t)kt[u] * GT_BYTES;
      if (MODE != 0 && live[u]) {
        const int e = p.ids[first + slot[u]];
        if (e < 0 || e >= p.experts) live[u] = false;
        else at += e * p.w_stride;
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        w[u][i] = make_uint4(0, 0, 0, 0);
        if (live[u]) w[u][i] = __ldcs(reinterpret_cast<const uint4 *>(wr + at + in_tile(i)));
      }
    }
    if (!waited) { griddep_wait(); waited = true; }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (!live[u]) continue;
      float by = 1.0f;
      if (MODE == 2) by = p.share[first + slot[u]];
      uint64_t x[T][4];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int r = MODE == 0 ? min((int)blockIdx.y * T + t, p.rows - 1) : MODE == 1 ? blockIdx.y / p.top_k : first + slot[u];
        load_x<X>(x[t], static_cast<const X *>(p.x) + r * p.ld_x, kt[u] * GT_K + chunk * 8, p.ic, p.words);
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        uint64_t f[4];
        unpack8<E>(w[u][i], f);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          if (MODE == 2) {
            uint64_t d = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) d = fma2(f[j], x[t][j], d);
            acc[t][i] = fma2(d, both(by, by), acc[t][i]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][i] = fma2(f[j], x[t][j], acc[t][i]);
          }
        }
      }
    }
  }
  if (!waited) griddep_wait();
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      float a = sum2(acc[t][i]);
#pragma unroll
      for (int d = 16; d; d >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
      if (lane == 0) part[warp][t * ROWS + i] = a;
    }
  __syncthreads();
  // one thread per result
  constexpr int OUTS = GATED ? ROWS / 2 : ROWS;
  if (threadIdx.x >= T * OUTS) return;
  const int t = threadIdx.x / OUTS, i = threadIdx.x % OUTS;
  if (MODE == 0 && blockIdx.y * T + t >= p.rows) return;
  if (MODE == 1) {
    const int e = p.ids[first];
    if (e < 0 || e >= p.experts) return;
  }
  const int ch = blockIdx.x * OUTS + i;
  if (ch >= p.epi.oc) return;
  float z = 0.0f, u = 0.0f;
  for (int k = 0; k < warps; ++k) {
    z += part[k][t * ROWS + i];
    if (GATED) u += part[k][t * ROWS + i + OUTS];
  }
  if (p.epi.bias) {
    const int pr = row_of<GATED, ROWS>(blockIdx.x, i);
    z += p.epi.bias[pr];
    if (GATED) u += p.epi.bias[pr + 8];
  }
  float v[8] = {z};                                             // (the activations take values by eights)
  activate(v, p.epi.act);
  float y = v[0];
  if (GATED) y *= u;
  y *= p.epi.scale;
  const long long r = MODE == 0 ? blockIdx.y * T + t : blockIdx.y;
  if (p.epi.res) y += to_f32(static_cast<const OT *>(p.epi.res)[r * p.epi.ld_res + ch]);
  static_cast<OT *>(p.epi.out)[r * p.epi.ld_out + ch] = from_f32<OT>(y);
}

template <typename E, typename OT, int T, bool GATED, int MODE>
cudaError_t go(const GemvParams &p, int along, cudaStream_t s) {
  const int steps = (p.kt + 3) / 4 * (MODE == 2 ? p.top_k : 1);
  const int warps = steps < MAX_WARPS ? steps : MAX_WARPS;
  const int channels = GATED ? 2 : 4;
  // eight rows where a warp has one step, so that there are eight loads in flight all the same, and for two tokens, so that
  // their values are fetched for more weights
  if (T == 2 || steps <= MAX_WARPS)
    return launch_overlapped(gemv_kernel<E, OT, T, GATED, MODE, 8>, dim3((p.epi.oc + 2 * channels - 1) / (2 * channels), along), dim3(warps * 32), 0, s, p);
  return launch_overlapped(gemv_kernel<E, OT, T, GATED, MODE, 4>, dim3((p.epi.oc + channels - 1) / channels, along), dim3(warps * 32), 0, s, p);
}

template <typename E, typename OT>
cudaError_t dense(const GemvParams &p, cudaStream_t s) {
  if (p.rows == 1) return p.epi.gated ? go<E, OT, 1, true, 0>(p, 1, s) : go<E, OT, 1, false, 0>(p, 1, s);
  const int along = (p.rows + 1) / 2;
  return p.epi.gated ? go<E, OT, 2, true, 0>(p, along, s) : go<E, OT, 2, false, 0>(p, along, s);
}

GemvParams from(const GemmParams &g) {
  GemvParams p = {};
  p.w = g.w;
  p.w_stride = g.w_stride;
  p.x = g.x;
  p.ld_x = g.ld_x;
  p.rows = g.rows;
  p.ic = g.ic;
  p.kt = g.kt;
  p.words = (reinterpret_cast<uintptr_t>(g.x) & 15) == 0 && g.ld_x % 8 == 0;
  p.epi = g.epi;
  return p;
}

template <typename E>
cudaError_t experts_as(const GemvParams &p, const GemvParams &q, int rows, cudaStream_t s) {
  const cudaError_t e = p.epi.gated ? go<E, float, 1, true, 1>(p, rows * p.top_k, s) : go<E, float, 1, false, 1>(p, rows * p.top_k, s);
  return e != cudaSuccess ? e : go<E, E, 1, false, 2>(q, rows, s);
}

}  // namespace

cudaError_t launch_gemv(const GemmParams &g, cudaStream_t s) {
  const GemvParams p = from(g);
  if (g.in_et == ET_BF16) return g.epi.out_et == ET_F32 ? dense<__nv_bfloat16, float>(p, s) : dense<__nv_bfloat16, __nv_bfloat16>(p, s);
  return g.epi.out_et == ET_F32 ? dense<__half, float>(p, s) : dense<__half, __half>(p, s);
}

cudaError_t launch_gemv_experts(const GemmParams &in, const GemmParams &out, const int *ids, const float *share, int rows, int top_k, int experts,
                                cudaStream_t s) {
  GemvParams p = from(in), q = from(out);
  p.ids = q.ids = ids;
  q.share = share;
  p.top_k = q.top_k = top_k;
  p.experts = q.experts = experts;
  return in.in_et == ET_BF16 ? experts_as<__nv_bfloat16>(p, q, rows, s) : experts_as<__half>(p, q, rows, s);
}

}  // namespace elb
