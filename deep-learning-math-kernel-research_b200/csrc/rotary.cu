// Rotary positions, of queries and keys or on the way into a cache of pages.
//
// (a, b) -> magnitude * (a cos x - b sin x, b cos x + a sin x), x = position * f.  An angle of 10^5 radians has no fraction left in 32 bits, so a plan holds
// f / (2 pi) modulo 1 as a 64-bit fraction: its product with the position, modulo 2^64, is taken without a rounding, and its upper 32
// bits are the argument of sincospi.
//
// A warp takes a token where there are many, the warps of a block its heads where there are few.  A lane has one 16-byte word of a head, or two words that turn
// together, and goes over the heads with it: its cosines and sines stay in registers, and there is nothing to work out from one head to the next.  The bound is
// the bytes of rows in and out, and how many of them are on their way: 32 warps an SM with one pair of words each bring 15 k tokens of 32 heads, 8 + 8 of them cached,
// past in 74 us (5.2 TB/s); with two pairs each in 24 warps 83, with words dealt out over the lanes and a division each 78, with seven pairs 205.
#include "attention.cuh"
#include "elb_common.cuh"

namespace elb {

namespace {

constexpr int WARPS = 8;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Word { T v[VEC]; };

template <typename T, int VEC, bool NEAR, bool TEAM>             // TEAM: a token per block
__global__ void __launch_bounds__(WARPS * 32, 4) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 turns[];                             // [tokens][rotary / 2] cosines and sines
  __shared__ long long shared_place;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = p.rotary / 2;
  const long long row = TEAM ? (long long)blockIdx.x : (long long)blockIdx.x * WARPS + warp;
  float2 *cs = turns + (TEAM ? 0 : warp * pairs);
  long long at = -1;                                            // the token's place in the cache; -1: the row is left out
  griddep_launch_dependents();
  griddep_wait();
  if ((!TEAM || warp == 0) && row < p.rows) {
    int position = 0;
    if (p.positions) {
      at = 0;
      position = p.positions[row];
    } else {
      const int s = sequence_of_row(p.seq, (int)row, lane);
      const int length = s >= 0 && s < p.seq.seqs ? p.seq.lengths[s] : 0;
      if (length > 0) {                                         // (an empty sequence's rows fill a batch up)
        const Sequence q = sequence_of(p.seq, s);
        position = length - q.n + ((int)row - q.first);         // (a length past the table is none that it can hold: no place)
        int page = -1, offset = 0;
        if (position >= 0 && (int)row < q.first + q.n) {
          const int i = position / p.page_size;
          offset = position - i * p.page_size;
          if (i < p.seq.width) page = p.seq.table[s * p.seq.width + i];
        }
        if (page >= 0 && page < p.seq.pages) at = page * p.ld_page + offset * p.ld_token;
        else if (lane == 0) report_status(p.status, ST_BAD_PAGE);
      }
    }
    if (at >= 0) {
      for (int i = lane; i < pairs; i += 32) {
        const int turn = (int)(((unsigned long long)(long long)position * p.steps[i]) >> 32);     // in 2^-32 of a whole one
        float s, c;
        sincospif((float)turn * 0x1p-31f, &s, &c);
        cs[i] = make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
      }
    }
  }
  if (TEAM) {
    if (threadIdx.x == 0) shared_place = at;
    __syncthreads();
    at = shared_place;
  } else {
    __syncwarp();
  }
  if (at < 0) return;
  using W = Word<T, VEC>;
  // Words of a head side by side in the lanes, as many heads as fit; a head of more words than lanes in several goes
  auto over_heads = [&](int units, auto each_word) {
    const int side = units < 32 ? 32 / units : 1, across = units < 32 ? lane / units : 0, step = TEAM ? side * WARPS : side;
    for (int from = 0; from < units; from += 32) {
      const int unit = from + (units < 32 ? lane - across * units : lane);
      if (unit < units && across < side) each_word(unit, across + (TEAM ? warp * side : 0), step);
    }
  };
  const int turned = pairs / VEC;
  // rows of heads from src to dst: their turned words in pairs, then those that are copied
  auto rows_of = [&](const T *src, T *dst, long long dst_head, int heads) {
    over_heads(turned + (p.head_dim - p.rotary) / VEC, [&](int unit, int h0, int step) {
      if (unit >= turned) {
        const int a = p.rotary + (unit - turned) * VEC;
        for (int h = h0; h < heads; h += step) *reinterpret_cast<W *>(dst + h * dst_head + a) = *reinterpret_cast<const W *>(src + h * p.head_dim + a);
        return;
      }
      const int a = (NEAR ? 2 : 1) * unit * VEC, b = NEAR ? a + VEC : a + pairs;
      float2 w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = cs[unit * VEC + e];
      auto turn = [&](W &x, W &y) {
        T in[2 * VEC], out[2 * VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) { in[e] = x.v[e]; in[VEC + e] = y.v[e]; }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int i = NEAR ? 2 * e : e, j = NEAR ? 2 * e + 1 : VEC + e;
          const float c = to_f32(in[i]), d = to_f32(in[j]);
          out[i] = from_f32<T>(c * w[e].x - d * w[e].y);
          out[j] = from_f32<T>(d * w[e].x + c * w[e].y);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) { x.v[e] = out[e]; y.v[e] = out[VEC + e]; }
      };
      for (int h = h0; h < heads; h += step) {
        W x = *reinterpret_cast<const W *>(src + h * p.head_dim + a), y = *reinterpret_cast<const W *>(src + h * p.head_dim + b);
        turn(x, y);
        *reinterpret_cast<W *>(dst + h * dst_head + a) = x;
        *reinterpret_cast<W *>(dst + h * dst_head + b) = y;
      }
    });
  };
  rows_of(static_cast<const T *>(p.q) + row * p.ld_q, static_cast<T *>(p.q_out) + row * p.ld_q_out, p.head_dim, p.heads);
  if (p.positions) rows_of(static_cast<const T *>(p.k) + row * p.ld_k, static_cast<T *>(p.k_out) + row * p.ld_k_out, p.head_dim, p.kv_heads);
  else rows_of(static_cast<const T *>(p.k) + row * p.ld_k, static_cast<T *>(p.k_out) + at, p.ld_head, p.kv_heads);
  if (p.v) {
    const T *src = static_cast<const T *>(p.v) + row * p.ld_v;
    T *dst = static_cast<T *>(p.v_out) + at;
    over_heads(p.head_dim / VEC, [&](int unit, int h0, int step) {
      for (int h = h0; h < p.kv_heads; h += step)
        *reinterpret_cast<W *>(dst + h * p.ld_head + unit * VEC) = *reinterpret_cast<const W *>(src + h * p.head_dim + unit * VEC);
    });
  }
}

template <typename T, int VEC, bool NEAR>
cudaError_t go(const RotaryParams &p, cudaStream_t s) {
  // A token per block is done sooner, a token per warp needs no barrier and no second wave: blocks' while warps' would not fill the SMs with a block each.  (us, block / warp, in a
  // graph: 32 + 8 heads of 128: 64 rows 3.3/5.7, 592 4.2/6.0, 1036 6.9/10.0, 1600 9.6/10.4, 2400 13.3/11.0; 16 + 16 of 80: 1036 5.7/7.9, 2400 11.3/8.3; 1 + 1 of 128: 296 2.5/2.6,
  // 1036 4.6/3.9.  Warps' grids of half of the SMs or just all of them are quicker than their neighbours: 1184 rows of 32 + 8 heads 7.4/5.9.  By rows alone the limit is a
  // compromise: the two cross near 500 rows of 2 heads, 1700 of 40.)
  const bool team = p.rows < (long long)p.num_sms * WARPS;
  const dim3 grid((unsigned)(team ? p.rows : (p.rows + WARPS - 1) / WARPS));
  const size_t smem = (size_t)(team ? 1 : WARPS) * (p.rotary / 2) * sizeof(float2);
  return team ? launch_overlapped(rotary_kernel<T, VEC, NEAR, true>, grid, dim3(WARPS * 32), smem, s, p)
              : launch_overlapped(rotary_kernel<T, VEC, NEAR, false>, grid, dim3(WARPS * 32), smem, s, p);
}
template <typename T>
cudaError_t go(const RotaryParams &p, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (p.words && p.rotary % (2 * VEC) == 0) return p.neighbours ? go<T, VEC, true>(p, s) : go<T, VEC, false>(p, s);
  return p.neighbours ? go<T, 1, true>(p, s) : go<T, 1, false>(p, s);
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
