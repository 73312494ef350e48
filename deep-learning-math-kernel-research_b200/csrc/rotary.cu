// Rotary positions, of queries and keys or on the way into a cache of pages.
//
// (a, b) -> magnitude * (a cos x - b sin x, b cos x + a sin x), x = position * f.  An angle of 10^5 radians has no fraction left in 32 bits, so a plan holds
// f / (2 pi) modulo 1 as a 64-bit fraction: its product with the position, modulo 2^64, is the turn without a rounding, and its upper 32
// bits are the argument of sincospi.
//
// A block takes up to eight tokens, a warp one each for its place and its table of cosines and sines, which all heads share; then the block's threads go
// over the heads' channels in words of 16 bytes.  The bound is the bytes of rows in and out.
#include "attention.cuh"
#include "elb_common.cuh"

namespace elb {

namespace {

constexpr int WARPS = 8;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Word { T v[VEC]; };

template <typename T, int VEC>
__global__ void __launch_bounds__(WARPS * 32) rotary_kernel(const RotaryParams p, int tokens) {
  extern __shared__ float2 turns[];                             // [tokens][rotary / 2] cosines and sines
  __shared__ long long place[WARPS];                            // of each token in the cache; -1: the row is left out
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = p.rotary / 2;
  const long long row0 = (long long)blockIdx.x * tokens;
  griddep_launch_dependents();
  griddep_wait();
  if (warp < tokens) {
    const long long row = row0 + warp;
    long long at = -1;
    int position = 0;
    if (row < p.rows) {
      if (p.positions) {
        at = 0;
        position = p.positions[row];
      } else {
        const int s = sequence_of_row(p.seq, (int)row, lane);
        if (s >= 0 && s < p.seq.seqs) {
          const Sequence q = sequence_of(p.seq, s);
          position = q.length - q.n + ((int)row - q.first);
          int page = -1;
          if (position >= 0 && (int)row < q.first + q.n) page = p.seq.table[s * p.seq.width + position / p.page_size];
          if (page >= 0 && page < p.seq.pages) at = page * p.ld_page + position % p.page_size * p.ld_token;
          else if (lane == 0) report_status(p.status, ST_BAD_PAGE);
        }
      }
    }
    if (lane == 0) place[warp] = at;
    if (at >= 0) {
      for (int i = lane; i < pairs; i += 32) {
        const int turn = (int)(((unsigned long long)(long long)position * p.steps[i]) >> 32);     // in 2^-32 of a whole one
        float s, c;
        sincospif((float)turn * 0x1p-31f, &s, &c);
        turns[warp * pairs + i] = make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
      }
    }
  }
  __syncthreads();
  using W = Word<T, VEC>;
  // words of a head: first those of whole pairs, two words each, then those that are copied
  const int turned = pairs / VEC, units = turned + (p.head_dim - p.rotary) / VEC, copied = p.head_dim / VEC;
  const int nq = p.heads * units, nk = p.kv_heads * units, all = nq + nk + (p.v ? p.kv_heads * copied : 0);
  for (int u = threadIdx.x; u < all * tokens; u += WARPS * 32) {
    const int t = u / all;
    int i = u - t * all;
    const long long row = row0 + t, at = place[t];
    if (at < 0) continue;
    const T *src;
    T *dst;
    int h, n = units;
    if (i < nq) {
      h = i / units;
      src = static_cast<const T *>(p.q) + row * p.ld_q;
      dst = static_cast<T *>(p.q_out) + row * p.ld_q_out + (long long)h * p.head_dim;
    } else if ((i -= nq) < nk) {
      h = i / units;
      src = static_cast<const T *>(p.k) + row * p.ld_k;
      dst = static_cast<T *>(p.k_out) + (p.positions ? row * p.ld_k_out + (long long)h * p.head_dim : at + h * p.ld_head);
    } else {
      i -= nk;
      n = copied;
      h = i / n;
      src = static_cast<const T *>(p.v) + row * p.ld_v;
      dst = static_cast<T *>(p.v_out) + at + h * p.ld_head;
    }
    src += (long long)h * p.head_dim;
    i -= h * n;
    if (n == units && i < turned) {
      const int a = p.neighbours ? 2 * i * VEC : i * VEC, b = p.neighbours ? a + VEC : pairs + a;
      const W wa = *reinterpret_cast<const W *>(src + a), wb = *reinterpret_cast<const W *>(src + b);
      const float2 *cs = turns + t * pairs + i * VEC;
      T in[2 * VEC], out[2 * VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) { in[e] = wa.v[e]; in[VEC + e] = wb.v[e]; }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float x = to_f32(p.neighbours ? in[2 * e] : in[e]), y = to_f32(p.neighbours ? in[2 * e + 1] : in[VEC + e]);
        const float2 w = cs[e];
        const T lo = from_f32<T>(x * w.x - y * w.y), hi = from_f32<T>(y * w.x + x * w.y);
        if (p.neighbours) { out[2 * e] = lo; out[2 * e + 1] = hi; }
        else { out[e] = lo; out[VEC + e] = hi; }
      }
      W ra, rb;
#pragma unroll
      for (int e = 0; e < VEC; ++e) { ra.v[e] = out[e]; rb.v[e] = out[VEC + e]; }
      *reinterpret_cast<W *>(dst + a) = ra;
      *reinterpret_cast<W *>(dst + b) = rb;
    } else {
      const int a = n == units ? p.rotary + (i - turned) * VEC : i * VEC;
      *reinterpret_cast<W *>(dst + a) = *reinterpret_cast<const W *>(src + a);
    }
  }
}

template <typename T>
cudaError_t go(const RotaryParams &p, cudaStream_t s) {
  const int tokens = p.rows >= 148 * WARPS ? WARPS : 1;
  const dim3 grid((unsigned)((p.rows + tokens - 1) / tokens));
  const size_t smem = (size_t)tokens * (p.rotary / 2) * sizeof(float2);
  constexpr int VEC = 16 / sizeof(T);
  if (p.words && p.rotary % (2 * VEC) == 0) return launch_overlapped(rotary_kernel<T, VEC>, grid, dim3(WARPS * 32), smem, s, p, tokens);
  return launch_overlapped(rotary_kernel<T, 1>, grid, dim3(WARPS * 32), smem, s, p, tokens);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams &p, cudaStream_t s) {
  switch (p.et) {
    case ET_F32: return go<float>(p, s);
    case ET_BF16: return go<__nv_bfloat16>(p, s);
    default: return go<__half>(p, s);
  }
}

}  // namespace elb
