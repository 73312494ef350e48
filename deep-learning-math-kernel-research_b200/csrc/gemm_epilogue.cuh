// Epilogue of the matrix products: bias, activation, gate, scale and residual on accumulators in tensor memory, whose lanes are
// packed weight rows (channels) and whose columns are tokens.
//
// A warp owns 32 lanes and takes 16 tokens at a time.  tcgen05.ld.16x256b hands them out as the fragments of an 8 x 8 matrix
// instruction: thread T has of 8 lanes by 8 columns the lane T / 4 and the columns 2 (T % 4) and + 1.  The gate and the up row
// of a channel lie 8 lanes apart and so meet in one thread; two tokens of a channel become one word of 16-bit values, and
// stmatrix.trans turns 8 channels by 8 tokens of those round, so that shared memory holds each token's channels in
// order and global memory is written (and the residual read) 16 bytes per thread.  Measured for a tile of 128 channels
// by 256 tokens, bf16, 12 warps, one CTA on every SM: 2700 cycles (gated silu 3700, silu with a bias 6000, gelu with one 7600, fp32 results 4900), bound by the
// warps' instructions; with one lane of tensor memory per thread, neighbouring lanes trading values and 4-byte stores 6700.
#pragma once
#include "ops.cuh"
#include "umma.cuh"

namespace elb {

// The hardware's 2^x and 1 / x, relative errors of about 2^-22 and 2^-23
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + 2^t) for two values with one reciprocal: 2^-t / (1 + 2^-t) where t > 0, so that the exponentials are at most 1 and the product of
// the denominators at most 4, whatever t is (a sum of -1e20 gives a factor of 0; below 2^-126 it is flushed there).  min drops a NaN, which stays out of
// the other value's factor: the caller multiplies it back in.  (silu with a bias 6000 cycles a tile; 2^t cut at 63 and 2^-t selected beyond it 6600.)
__device__ __forceinline__ void logistic2(float t0, float t1, float &s0, float &s1) {
  const float e0 = ex2(fminf(-fabsf(t0), 0.0f)), e1 = ex2(fminf(-fabsf(t1), 0.0f)), d0 = 1.0f + e0, d1 = 1.0f + e1;
  const float r = rcp(d0 * d1);
  s0 = r * (t0 > 0.0f ? e0 * d1 : d1);
  s1 = r * (t1 > 0.0f ? e1 * d0 : d0);
}

// v / (1 + 2^t(v)).  Values i and i + 4 are two channels of one token: what a value comes to depends on no other token.
template <int N, typename F>
__device__ __forceinline__ void logistic_times(float (&v)[N], F t) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i & 4) continue;
    float s0, s1;
    logistic2(t(v[i]), t(v[i + 4]), s0, s1);
    v[i] *= s0;
    v[i + 4] *= s1;
  }
}

template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  switch (act) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];       // (a NaN stays one)
      break;
    case 2:
      // z Phi(z), Phi(-a) = erfc(a / sqrt 2) / 2 = (c1 t + ... + c8 t^8) exp(-a^2 / 2), t = 1 / (1 + 0.43 a / sqrt 2): the form of Abramowitz and
      // Stegun 7.1.26, with coefficients fitted to the least relative error (least squares over Chebyshev polynomials, reweighted until
      // the errors were level; 8.4e-8, in 32 bits 3.7e-7), so that values far below zero keep their digits too.  Their five coefficients hold the
      // absolute error to 1.5e-7 and were 5e-4 off, relatively, at z = -4.
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = rcp(fmaf(0.30405593f, fabsf(v[i]), 1.0f));
        float q = fmaf(0.03685394f, t, -0.1551866f);
        q = fmaf(q, t, 0.19185269f);
        q = fmaf(q, t, -0.042862747f);
        q = fmaf(q, t, 0.12342216f);
        q = fmaf(q, t, 0.10247557f);
        q = fmaf(q, t, 0.12218772f);
        q = fmaf(q, t, 0.121257305f);
        const float phi = q * t * ex2(v[i] * v[i] * -0.72134752f);
        v[i] *= v[i] < 0.0f ? phi : 1.0f - phi;
      }
      break;
    case 3:   // 0.5 z (1 + tanh u) = z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3)
      logistic_times(v, [](float z) { return -2.3022081983586606f * fmaf(0.044715f * z * z, z, z); });
      break;
    case 4:
      logistic_times(v, [](float z) { return z * -1.4426950408889634f; });
      break;
    default: break;
  }
}

// 16 lanes by 16 columns: registers 4g and 4g + 1 are lane T / 4, columns 8g + 2 (T % 4) and + 1; 4g + 2 and 4g + 3 are lane 8 + T / 4.
__device__ __forceinline__ void tmem_ld_fragments(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
// A warp's 32 lanes by 16 columns: r[8 h + ..] for the lanes 16 h ..
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld_fragments(taddr, r);
  tmem_ld_fragments(taddr + (16u << 16), r + 8);
}
__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

constexpr int EPI_STAGE = 1024;     // bytes of shared memory of a warp, 16-byte aligned

// One warp's part of a tile: CH channels (32, or 16 where gated) of up to 16 tokens at a time.  fp32 results go to memory as
// they are: a store then has eight channels, a whole sector, of four tokens.
template <typename OT, bool GATED>
struct EpilogueWarp {
  static constexpr int CH = GATED ? 16 : 32, CHUNKS = CH / 8;                // channels; 16-byte chunks of a token's row in shared memory
  static constexpr int STEP = 32 / CHUNKS, N = 16 / STEP;                    // tokens of one access of the warp; accesses of a block
  static constexpr int G = GATED ? 2 : 4, VALUES = 4 * G;                    // groups of eight channels; values of a thread
  static constexpr bool HALF = sizeof(OT) == 2;

  const Epilogue &e;
  uint8_t *stage;
  int lane, ch0, sub_t, sub_c;      // first channel of the warp; this thread's token and chunk of an access
  uint32_t matrix;                  // this thread's row of the first four matrices in shared memory, the others 512 bytes behind
  float bias[4];
  bool whole;                       // all of the warp's channels exist and rows are aligned
  uint4 ahead[N];                   // the next block's residual: 16-byte chunks, or, where not whole, one value per pass

  __device__ __forceinline__ EpilogueWarp(const Epilogue &e_, uint8_t *stage_, int lane_, int prow0) : e(e_), stage(stage_), lane(lane_) {
    ch0 = GATED ? prow0 >> 1 : prow0;
    sub_t = lane / CHUNKS;
    sub_c = lane % CHUNKS;
    whole = HALF && e.words && ch0 + CH <= e.oc;
    matrix = smem_u32(GATED ? at((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1) : at(lane & 7, lane >> 3));
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = e.bias ? e.bias[prow0 + (lane >> 2) + 8 * i] : 0.0f;
  }
  // the 16-byte chunk c of token t in shared memory, chunks permuted so that neither side meets bank conflicts
  __device__ __forceinline__ uint8_t *at(int t, int c) const { return stage + (t * CHUNKS + (c ^ (GATED ? (t >> 2) & 1 : (t >> 1) & 3))) * 16; }
  // the first of the two values of matrix q of the m-th four (of 8 channels by 8 tokens: all channels of 8 tokens, or, gated, of 16)
  static __device__ __forceinline__ constexpr int index(int m, int q) { return GATED ? 4 * (q & 1) + 2 * (q >> 1) : 4 * q + 2 * m; }
  __device__ __forceinline__ void fetch(long long tok0, int ntok) {
    if (!HALF || !e.res || ntok <= 0) return;
    if (whole) {
      const OT *res = static_cast<const OT *>(e.res) + (tok0 + sub_t) * e.ld_res + ch0 + sub_c * 8;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n * STEP + sub_t < ntok) ahead[n] = *reinterpret_cast<const uint4 *>(res + n * STEP * e.ld_res);
    } else {
      const uint16_t *res = static_cast<const uint16_t *>(e.res) + (tok0 + lane / CH) * e.ld_res + ch0 + lane % CH;
      const bool has = ch0 + lane % CH < e.oc;
      uint32_t one[PASSES];
#pragma unroll
      for (int n = 0; n < PASSES; ++n) one[n] = has && n * TP + lane / CH < ntok ? res[n * TP * e.ld_res] : 0u;
#pragma unroll
      for (int n = 0; n < N; ++n)
        ahead[n] = make_uint4(one[8 * n] | one[8 * n + 1] << 16, one[8 * n + 2] | one[8 * n + 3] << 16, one[8 * n + 4] | one[8 * n + 5] << 16,
                              one[8 * n + 6] | one[8 * n + 7] << 16);
    }
  }
  // One by one, where the rows are not aligned or channels are missing: neighbouring lanes, neighbouring channels
  static constexpr int TP = 32 / CH, PASSES = 16 / TP;
  __device__ __forceinline__ OT &single(int n) const { return reinterpret_cast<OT *>(at(n * TP + lane / CH, lane % CH >> 3))[lane & 7]; }
  __device__ __forceinline__ void singles_in() {
#pragma unroll
    for (int n = 0; n < PASSES; ++n) {
      const uint32_t w[4] = {ahead[n / 8].x, ahead[n / 8].y, ahead[n / 8].z, ahead[n / 8].w};
      reinterpret_cast<uint16_t &>(single(n)) = (uint16_t)(w[n / 2 % 4] >> (16 * (n & 1)));
    }
  }
  __device__ __forceinline__ void singles_out(long long tok0, int ntok) {
    OT *out = static_cast<OT *>(e.out) + (tok0 + lane / CH) * e.ld_out + ch0 + lane % CH;
    const bool has = ch0 + lane % CH < e.oc;
#pragma unroll
    for (int n = 0; n < PASSES; ++n)
      if (has && n * TP + lane / CH < ntok) out[n * TP * e.ld_out] = single(n);
  }
  // acc: the block's accumulators as tmem_ld_block has them, ntok real tokens from tok0; the residual of the block behind (`next`
  // tokens from next0) is fetched here.
  __device__ __forceinline__ void block(const uint32_t (&acc)[16], long long tok0, int ntok, long long next0, int next) {
    // y[4 i + 2 g + j]: channel 8 i + T / 4 of the warp's, token 8 g + 2 (T % 4) + j
    float y[VALUES], u[GATED ? VALUES : 1];
#pragma unroll
    for (int v = 0; v < VALUES; ++v) {
      const int i = v / 4, g = v / 2 % 2, j = v % 2;
      if constexpr (GATED) {
        y[v] = __uint_as_float(acc[8 * i + 4 * g + j]);
        u[v] = __uint_as_float(acc[8 * i + 4 * g + 2 + j]);
      } else {
        y[v] = __uint_as_float(acc[8 * (i >> 1) + 4 * g + 2 * (i & 1) + j]);
      }
    }
    if (e.bias) {
#pragma unroll
      for (int v = 0; v < VALUES; ++v) {
        if constexpr (GATED) { y[v] += bias[v / 4 * 2]; u[v] += bias[v / 4 * 2 + 1]; }
        else y[v] += bias[v / 4];
      }
    }
    activate(y, e.act);
    if constexpr (GATED) {
#pragma unroll
      for (int v = 0; v < VALUES; ++v) y[v] *= u[v];
    }
    if (e.scale != 1.0f) {
#pragma unroll
      for (int v = 0; v < VALUES; ++v) y[v] *= e.scale;
    }
    if constexpr (!HALF) {
      const long long t0 = tok0 + 2 * (lane & 3);
      const int ch = ch0 + (lane >> 2);
      float *out = static_cast<float *>(e.out) + t0 * e.ld_out + ch;
      if (e.res) {
        const float *res = static_cast<const float *>(e.res) + t0 * e.ld_res + ch;
#pragma unroll
        for (int v = 0; v < VALUES; ++v) {
          const int i = v / 4, t = v / 2 % 2 * 8 + v % 2;
          if (ch + 8 * i < e.oc && t + 2 * (lane & 3) < ntok) y[v] += res[t * e.ld_res + 8 * i];
        }
      }
#pragma unroll
      for (int v = 0; v < VALUES; ++v) {
        const int i = v / 4, t = v / 2 % 2 * 8 + v % 2;
        if (ch + 8 * i < e.oc && t + 2 * (lane & 3) < ntok) out[t * e.ld_out + 8 * i] = y[v];
      }
    } else {
      if (e.res) {
        if (whole) {
#pragma unroll
          for (int n = 0; n < N; ++n) *reinterpret_cast<uint4 *>(at(n * STEP + sub_t, sub_c)) = ahead[n];
        } else {
          singles_in();
        }
        fetch(next0, next);
        __syncwarp();
#pragma unroll
        for (int m = 0; m < G / 2; ++m) {
          uint32_t r[4];
          ldmatrix4_trans(matrix + m * 512, r);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 add = unpack2<OT>(r[q]);
            y[index(m, q)] += add.x;
            y[index(m, q) + 1] += add.y;
          }
        }
      }
#pragma unroll
      for (int m = 0; m < G / 2; ++m) {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = pack2<OT>(y[index(m, q)], y[index(m, q) + 1]);
        stmatrix4_trans(matrix + m * 512, w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
      if (whole) {
        OT *out = static_cast<OT *>(e.out) + (tok0 + sub_t) * e.ld_out + ch0 + sub_c * 8;
        uint4 q[N];
#pragma unroll
        for (int n = 0; n < N; ++n) q[n] = *reinterpret_cast<const uint4 *>(at(n * STEP + sub_t, sub_c));
        if (ntok >= 16) {
#pragma unroll
          for (int n = 0; n < N; ++n) *reinterpret_cast<uint4 *>(out + n * STEP * e.ld_out) = q[n];
        } else {
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n * STEP + sub_t < ntok) *reinterpret_cast<uint4 *>(out + n * STEP * e.ld_out) = q[n];
        }
      } else {
        singles_out(tok0, ntok);
      }
      __syncwarp();
    }
  }
};

// All tokens of a tile, in blocks of 16 that go round the `parts` warps of a quarter of the lanes.  wait() returns when the
// accumulator is complete (false: never); the bias and the first residual are on their way before.  release() runs when the last
// of this warp's accumulators has been read.  A block's last columns may lie past the tile's: the accumulator has them.
template <typename OT, bool GATED, typename W, typename F>
__device__ __forceinline__ bool epilogue_tile_as(const Epilogue &e, uint8_t *stage, uint32_t taddr, int part, int parts, int lane, int prow0,
                                                 long long tok0, int ntok, W wait, F release) {
  EpilogueWarp<OT, GATED> w(e, stage, lane, prow0);
  const int step = parts * 16;
  w.fetch(tok0 + part * 16, ntok - part * 16);
  if (!wait()) return false;
#pragma unroll 1
  for (int t = part * 16; t < ntok; t += step) {
    uint32_t a[16];             // (asking for the next block's meanwhile costs more in moved registers than it hides)
    tmem_ld_block(taddr + t, a);
    tmem_ld_wait16(a);
    if (t + step >= ntok) release();
    w.block(a, tok0 + t, ntok - t, tok0 + t + step, ntok - t - step);
  }
  if (part * 16 >= ntok) release();
  return true;
}
// f: a call with the result's type and the gate as template arguments
template <typename F>
__device__ __forceinline__ bool by_kind(const Epilogue &e, F f) {
  if (e.gated) {
    if (e.out_et == ET_BF16) return f.template operator()<__nv_bfloat16, true>();
    if (e.out_et == ET_F16) return f.template operator()<__half, true>();
    return f.template operator()<float, true>();
  }
  if (e.out_et == ET_BF16) return f.template operator()<__nv_bfloat16, false>();
  if (e.out_et == ET_F16) return f.template operator()<__half, false>();
  return f.template operator()<float, false>();
}

}  // namespace elb
