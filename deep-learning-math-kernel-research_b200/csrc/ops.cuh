// Shared declarations of the transformer operators (elb_linear_*, elb_norm_*, elb_route_*, elb_experts_*): element types,
// the epilogue of the matrix products, parameter blocks and launcher prototypes.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace elb {

enum : int { ET_F32 = 0, ET_BF16 = 1, ET_F16 = 2 };

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two values as one 32-bit word, `lo` at the lower address.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// ---------------------------------------------------------------------------------------------
// Epilogue of the matrix products.  The products are computed with the weights as the left operand, so
// that a lane of a warp holds one weight row for several tokens: 32 lanes are 32 consecutive packed rows,
// which are channels, or gate and up rows in turn (row 2q the gate of channel q, row 2q + 1 its up).
// ---------------------------------------------------------------------------------------------
struct Epilogue {
  void *out;
  const void *res;          // null: no residual
  const float *bias;        // in packed row order, padded with zeros to whole tiles; null: none
  long long ld_out, ld_res;
  int oc;                   // output channels (packed rows are 2 * oc where gated)
  int act, gated, out_et;
  int pairs;                // 16-bit results: out and res allow 4-byte accesses at even channels
  float scale;
};

template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  switch (act) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];       // (a NaN stays one)
      break;
    case 2:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678118654752f));
      break;
    case 3:   // 0.5 z (1 + tanh u) = z / (1 + exp(-2 u))
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u2 = 1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]);
        v[i] = __fdividef(v[i], 1.0f + __expf(-u2));
      }
      break;
    case 4:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __fdividef(v[i], 1.0f + __expf(-v[i]));
      break;
    default: break;
  }
}

// v[j]: packed row `prow` (this lane's) of token tok0 + j, of which ntok are real.  A converged warp, prow - lane a
// multiple of 32.
template <typename OT, int NT>
__device__ __forceinline__ void emit_as(const Epilogue &e, float (&v)[NT], int prow, long long tok0, int ntok) {
  const int odd = prow & 1;
  OT *out = static_cast<OT *>(e.out);
  const OT *res = static_cast<const OT *>(e.res);
  if (e.bias) {
    const float b = e.bias[prow];
#pragma unroll
    for (int j = 0; j < NT; ++j) v[j] += b;
  }
  if (e.gated) {
    // The even lane holds the gate and the odd one the up row of a channel: they trade half of their tokens, after
    // which the even lane has both for the even tokens and the odd lane for the odd ones.
    float g[NT / 2], u[NT / 2];
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * j] : v[2 * j + 1], 1);
      g[j] = odd ? got : v[2 * j];
      u[j] = odd ? v[2 * j + 1] : got;
    }
    activate(g, e.act);
    const int ch = prow >> 1;
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      const int t = 2 * j + odd;
      if (t < ntok && ch < e.oc) {
        float y = g[j] * u[j] * e.scale;
        if (res) y += to_f32(res[(tok0 + t) * e.ld_res + ch]);
        out[(tok0 + t) * e.ld_out + ch] = from_f32<OT>(y);
      }
    }
    return;
  }
  activate(v, e.act);
  if constexpr (sizeof(OT) == 2) {
    if (e.pairs) {
      // neighbouring lanes trade half of their tokens, so that each holds two channels of every second token
      const int ch = prow & ~1;
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * j] : v[2 * j + 1], 1);
        float lo = (odd ? got : v[2 * j]) * e.scale, hi = (odd ? v[2 * j + 1] : got) * e.scale;
        const int t = 2 * j + odd;
        if (t < ntok && ch + 1 < e.oc) {
          if (res) {
            const float2 r = unpack2<OT>(*reinterpret_cast<const uint32_t *>(res + (tok0 + t) * e.ld_res + ch));
            lo += r.x;
            hi += r.y;
          }
          *reinterpret_cast<uint32_t *>(out + (tok0 + t) * e.ld_out + ch) = pack2<OT>(lo, hi);
        } else if (t < ntok && ch < e.oc) {
          if (res) lo += to_f32(res[(tok0 + t) * e.ld_res + ch]);
          out[(tok0 + t) * e.ld_out + ch] = from_f32<OT>(lo);
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (j < ntok && prow < e.oc) {
      float y = v[j] * e.scale;
      if (res) y += to_f32(res[(tok0 + j) * e.ld_res + prow]);
      out[(tok0 + j) * e.ld_out + prow] = from_f32<OT>(y);
    }
  }
}
template <int NT>
__device__ __forceinline__ void emit(const Epilogue &e, float (&v)[NT], int prow, long long tok0, int ntok) {
  if (e.out_et == ET_BF16) emit_as<__nv_bfloat16, NT>(e, v, prow, tok0, ntok);
  else if (e.out_et == ET_F16) emit_as<__half, NT>(e, v, prow, tok0, ntok);
  else emit_as<float, NT>(e, v, prow, tok0, ntok);
}

// The same for 16 real tokens and a warp whose channels all exist, 16-bit results and residuals at even channels in 4-byte
// words: `out` and `res` are this lane's first element, from first_element().  Without the tests of the general form a
// token costs a warp about 5 instructions instead of 38, which is what a long call's epilogue is bound by.
template <typename OT, bool GATED>
__device__ __forceinline__ long long first_token(int prow) {     // of the 16, the first that this lane stores
  if (!GATED) return sizeof(OT) == 2 ? prow & 1 : 0;
  return sizeof(OT) == 2 ? (prow & 2) + (prow & 1) : prow & 1;
}
template <typename OT, bool GATED>
__device__ __forceinline__ int first_channel(int prow) {
  if (!GATED) return sizeof(OT) == 2 ? prow & ~1 : prow;
  return sizeof(OT) == 2 ? (prow >> 1) & ~1 : prow >> 1;
}
template <typename OT, bool GATED>
__device__ __forceinline__ void emit_full(const Epilogue &e, float (&v)[16], int prow, float bias, OT *out, const OT *res) {
  const int odd = prow & 1;
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += bias;
  constexpr int EACH = sizeof(OT) == 2 ? (GATED ? 4 : 2) : (GATED ? 2 : 1);     // tokens from one of this lane's stores to the next
  constexpr int N = 16 / EACH;
  const long long so = e.ld_out * EACH, sr = e.ld_res * EACH;
  if constexpr (GATED) {
    float y[8], u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * j] : v[2 * j + 1], 1);
      y[j] = odd ? got : v[2 * j];
      u[j] = odd ? v[2 * j + 1] : got;
    }
    activate(y, e.act);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = y[j] * u[j] * e.scale;
    if constexpr (sizeof(OT) == 4) {
      float r[8] = {};
      if (res) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = res[j * sr];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j * so] = y[j] + r[j];
    } else {
      // a second trade, between lanes of neighbouring channels: two channels of every fourth token
      const int high = prow & 2;
      uint32_t r[4] = {};
      if (res) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const uint32_t *>(res + j * sr);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float got = __shfl_xor_sync(0xFFFFFFFFu, high ? y[2 * j] : y[2 * j + 1], 2);
        const float2 add = unpack2<OT>(r[j]);
        *reinterpret_cast<uint32_t *>(out + j * so) = pack2<OT>((high ? got : y[2 * j]) + add.x, (high ? y[2 * j + 1] : got) + add.y);
      }
    }
  } else {
    activate(v, e.act);
    if constexpr (sizeof(OT) == 4) {
      float r[16] = {};
      if (res) {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = res[j * sr];
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) out[j * so] = fmaf(v[j], e.scale, r[j]);
    } else {
      uint32_t r[N] = {};
      if (res) {
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = *reinterpret_cast<const uint32_t *>(res + j * sr);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2 * j] : v[2 * j + 1], 1);
        const float2 add = unpack2<OT>(r[j]);
        *reinterpret_cast<uint32_t *>(out + j * so) =
            pack2<OT>(fmaf(odd ? got : v[2 * j], e.scale, add.x), fmaf(odd ? v[2 * j + 1] : got, e.scale, add.y));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Matrix products on packed weights.  The packed image is the shared-memory operand image itself: tiles of 128 rows x
// 64 channels, [row tile][channel tile][128 rows][128 bytes], the 16-byte chunks of a row permuted as the 128-byte
// swizzle has them; rows and channels past the end are zero.
// ---------------------------------------------------------------------------------------------
constexpr int GT_ROWS = 128, GT_K = 64, GT_BYTES = GT_ROWS * GT_K * 2;

// Rows of one expert: input rows [row0, row0 + count) of the sorted rows.
struct GroupTile { int expert, row0, count, pad; };

struct GemmParams {
  const uint8_t *w;                 // packed weights; expert e at w + e * w_stride
  size_t w_stride;
  const void *x;                    // tokens, [rows][ld_x] 16-bit
  long long ld_x;
  int rows, ic, kt, row_tiles;      // kt: channel tiles of 64; row_tiles: tiles of 128 packed rows
  int in_et;                        // ET_BF16 or ET_F16
  const GroupTile *tiles;           // grouped: the token tiles, *n_tiles of them; null: dense
  const int *n_tiles;
  int max_tiles, tile_tokens;       // grouped: the most that *n_tiles can be; tokens of a tile (grouped_tile_tokens)
  long long w_rows;                 // rows of 128 bytes of the whole packed image
  int num_sms, max_pairs;
  int *status;
  Epilogue epi;
};

// rows: rows of a source matrix per expert (2 * oc where gated), experts matrices behind one another
cudaError_t launch_pack_weights(void *dst, const void *src, int experts, int rows, int ic, bool gated, bool hwio, cudaStream_t s);
cudaError_t launch_pack_bias(float *dst, const void *src, int et, int rows, int padded, bool gated, cudaStream_t s);
cudaError_t launch_gemm(const GemmParams &p, cudaStream_t s);
cudaError_t init_gemm(int num_sms, int *max_pairs);
// x and ld_x of GemmParams are multiples of 16 bytes; other rows are copied first
cudaError_t launch_align_rows(void *dst, long long pitch, const void *src, long long ld, int rows, int n, cudaStream_t s);
int grouped_tile_tokens(int slots, int experts);
constexpr int MIN_TILE_TOKENS = 16;

struct ExpertsParams {
  const int *ids;
  const float *weights;
  const void *x;
  void *xs;                         // sorted rows [slots][pitch_x]
  const float *y;                   // products of the sorted rows [slots][pitch_y]
  void *out;
  int *count;                       // slots of each expert; zero between calls
  int *pos, *place;                 // of each slot: among those of its expert; its sorted row
  GroupTile *tiles;
  int *n_tiles;
  long long ld_x, ld_out, pitch_x, pitch_y;
  int rows, top_k, experts, ic, et, tile_tokens;    // tile_tokens: the most that a token tile holds
};
cudaError_t launch_experts_count(const ExpertsParams &p, cudaStream_t s);
cudaError_t launch_experts_gather(const ExpertsParams &p, int num_sms, cudaStream_t s);
cudaError_t launch_experts_combine(const ExpertsParams &p, cudaStream_t s);

struct NormParams {
  const void *x, *res, *gate;
  void *sum, *y;
  const float *post_w, *post_b, *pre_w, *pre_b;     // never null where their norm is not NONE
  long long ld_x, ld_res, ld_gate, ld_sum, ld_y;
  long long rows;
  int channels, gate_rows, post, pre, et, et_res;
  float post_eps, pre_eps, scale;
};
// dst = offset + src, or ones where src is null
cudaError_t launch_norm_vector(float *dst, const void *src, int et, int n, float offset, cudaStream_t s);
cudaError_t launch_block_norm(const NormParams &p, cudaStream_t s);

struct RouteParams {
  const void *logits;
  const float *bias;
  int *ids;
  float *weights;
  long long ld, rows;
  int experts, top_k, et, sigmoid, groups, top_groups, group_best, renormalise;
  float scale;
};
cudaError_t launch_route(const RouteParams &p, cudaStream_t s);

}  // namespace elb
