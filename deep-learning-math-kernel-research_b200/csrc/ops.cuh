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

// What becomes of the products (gemm_epilogue.cuh).  Packed rows are output channels in order, or, gated, groups of 16: the
// gates of eight channels, then their ups.
struct Epilogue {
  void *out;
  const void *res;          // null: no residual
  const float *bias;        // in packed row order, padded with zeros to whole pairs of tiles; null: none
  long long ld_out, ld_res;
  int oc;                   // output channels (packed rows are 2 * oc where gated)
  int act, gated, out_et;
  int words;                // rows of out and res start at 16-byte boundaries
  float scale;
};
// the source's row of packed row p, of `rows` (2 * oc where gated); rows or more: none, a row of zeros
__host__ __device__ inline int packed_source(int p, int rows, bool gated) {
  if (!gated) return p;
  const int ch = (p >> 4) * 8 + (p & 7), oc = rows >> 1;
  return ch < oc ? ch + ((p >> 3) & 1) * oc : rows;
}

// ---------------------------------------------------------------------------------------------
// Matrix products on packed weights.  The packed image is the shared-memory operand image itself: tiles of 128 rows x
// 64 channels, [row tile][channel tile][128 rows][128 bytes], the 16-byte chunks of a row permuted as the 128-byte
// swizzle has them; rows and channels past the end are zero.  (packed_rows: 16 for every 8 channels where gated.)
// ---------------------------------------------------------------------------------------------
inline int packed_rows(int oc, bool gated) { return gated ? (oc + 7) / 8 * 16 : oc; }
constexpr int GT_ROWS = 128, GT_K = 64, GT_BYTES = GT_ROWS * GT_K * 2;

// Rows of one expert: input rows [row0, row0 + count) of the sorted rows.
struct alignas(16) GroupTile { int expert, row0, count, pad; };

struct GemmParams {
  const uint8_t *w;                 // packed weights; expert e at w + e * w_stride
  size_t w_stride;
  const void *x;                    // tokens, [rows][ld_x] 16-bit
  long long ld_x;
  int rows, ic, kt, row_tiles;      // kt: channel tiles of 64; row_tiles: tiles of 128 packed rows
  int in_et;                        // ET_BF16 or ET_F16
  const GroupTile *tiles;           // grouped: the token tiles, *n_tiles of them; null: dense
  const int *n_tiles;
  int tiles_old;                    // they were written before the kernel in front of this one started
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
// A handful of rows, any alignment of x
bool gemm_wants_gemv(long long rows, int row_tiles, int kt);
bool experts_want_gemv(int slots, int experts, double expert_bytes);
cudaError_t launch_gemv(const GemmParams &p, cudaStream_t s);
// Both products and the sum over a token's experts, slot by slot, GEMV_SLOTS at most: in.x the tokens, in.epi.out and out.x the middle
// rows of the slots, in fp32 (few slots cost little more so, and the middle needs no rounding)
constexpr int GEMV_SLOTS = 256;
cudaError_t launch_gemv_experts(const GemmParams &in, const GemmParams &out, const int *ids, const float *share, int rows, int top_k, int experts,
                                cudaStream_t s);
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
  int clear;                        // the combine kernel leaves zero counts
  int rows, top_k, experts, ic, et, tile_tokens;    // tile_tokens: the most that a token tile holds
};
// Slots of the gather kernel's blocks, `per` each (the last one fewer).  In 64 bits: the last block's end may pass 2^31 before it is cut.
struct SlotShare {
  int per, blocks;
  __host__ __device__ int first(int block) const { return block * per; }
  __host__ __device__ int end(int block, int slots) const {
    const long long e = (block + 1ll) * per;
    return e < slots ? (int)e : slots;
  }
};
inline SlotShare share_slots(int slots, int warps, int most) {
  const int blocks = (slots + warps - 1) / warps < most ? (slots + warps - 1) / warps : most, per = (slots + blocks - 1) / blocks;
  return {per, (int)(((long long)slots + per - 1) / per)};
}
bool experts_count_here(int slots);      // the gather kernel counts few slots itself
cudaError_t launch_experts_count(const ExpertsParams &p, cudaStream_t s);
cudaError_t launch_experts_gather(const ExpertsParams &p, int num_sms, cudaStream_t s);
cudaError_t launch_experts_combine(const ExpertsParams &p, cudaStream_t s);

struct NormParams {
  const void *x, *res, *gate;
  void *sum, *y;
  const float *post_w, *post_b, *pre_w, *pre_b;     // never null where their norm is not NONE
  long long ld_x, ld_res, ld_gate, ld_sum, ld_y;
  long long rows, w_pitch;                          // elements from one of the eight copies of a weight vector to the next
  int channels, gate_rows, post, pre, et, et_res, num_sms;
  float post_eps, pre_eps, scale;
};
// eight copies of offset + src (of ones where src is null), copy a from index a on, zeros around
cudaError_t launch_norm_vector(float *dst, const void *src, int et, int n, long long pitch, float offset, cudaStream_t s);
cudaError_t launch_block_norm(const NormParams &p, cudaStream_t s);

struct RouteParams {
  const void *logits;
  const float *bias;
  int *ids;
  float *weights;
  long long ld, rows;
  int experts, top_k, et, sigmoid, groups, top_groups, group_best, renormalise;
  int lanes_per_group, words;       // set by the launch: whole lanes of a group (0: groups and lanes do not fit), 16-byte rows
  float scale;
};
cudaError_t launch_route(const RouteParams &p, cudaStream_t s);

}  // namespace elb
