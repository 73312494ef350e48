// Attention of few new tokens over long keys: a step of answers.
//
// What it is made of is reading K and V once.  All rows of a key head (its g heads times the sequence's new tokens) share a tile of
// 64 keys; the call's tiles, of all sequences and key heads in order, are dealt out evenly to one CTA per SM, whatever their lengths, so a
// sequence's length is split wherever that falls.  A CTA's producer keeps up to 192 KB of tiled copies in flight; four warps take 16 of a tile's
// 64 keys each, with a running maximum, sum and result of their own, so that they meet only at the end of a piece.  Then their results are joined,
// written out if the piece is all of its key head's keys, and left in the workspace otherwise, where the last CTA of those that share it joins
// them in the order of the keys: no result depends on timing.
//
// Products are mma.sync m16n8k16: 16 rows are the least a matrix instruction takes, and at HBM's rate (23 bytes per SM and cycle) one of them is wanted
// every 22 cycles, far below what it can do; tcgen05 would pad 128 rows and bring each score through tensor memory.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"
#include "umma.cuh"

namespace elb {

namespace {

constexpr int TILE = 64, WARPS = 4, THREADS = WARPS * 32 + 32;
constexpr int BOX_BYTES = TILE * 128;                           // 64 keys of 64 channels

// CB: boxes of 64 channels; MB: blocks of 16 rows
template <int CB, int MB>
struct Smem {
  static constexpr int STAGE = 2 * CB * BOX_BYTES;
  static constexpr int MERGE = WARPS * MB * CB * 8 * 32 * 16;   // every warp's results
  static constexpr int STAGES = (224 * 1024 - MERGE) / STAGE;
  static constexpr int MERGE_OFF = STAGES * STAGE;
  static constexpr int ML_OFF = MERGE_OFF + MERGE;              // maxima and sums, [WARPS][MB * 16]
  static constexpr int BAR_OFF = ML_OFF + WARPS * MB * 16 * 8;
  static constexpr int MISC_OFF = BAR_OFF + 2 * STAGES * 8;
  static constexpr int TOTAL = MISC_OFF + 256 + 1024;
};

struct alignas(64) TokenLaunch {
  CUtensorMap kmap, vmap;
  AttentionParams p;
  AttentionWorkspace w;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The call's tiles in order: sequences, their key heads, their tiles (one at least, so that every row is written).  CTA c of `ctas` takes those
// from c * total / ctas on.
struct Deal {
  long long total;
  int ctas;
  __device__ __forceinline__ long long begin(int c) const { return c * total / ctas; }
  __device__ __forceinline__ int owner(long long tile) const { return (int)(((tile + 1) * ctas - 1) / total); }
};
// Where a CTA is: tile `at` of the call lies in key head `head` of sequence s, whose `tiles` tiles of head 0 begin at `base`
struct Walk {
  const AttentionParams &p;
  const KeyTiles<TILE> kt;
  Sequence q;
  long long at, base;
  int s, head, tiles;
  __device__ __forceinline__ Walk(const AttentionParams &p, long long at, int s, long long base) : p(p), kt(p.page_size), at(at), base(base), s(s) {
    read();
    head = (int)((at - base) / tiles);
  }
  __device__ __forceinline__ void read() {
    q = sequence_of(p.seq, s);
    tiles = max(1, kt.count(q.length));
  }
  __device__ __forceinline__ long long item() const { return base + (long long)head * tiles; }
  __device__ __forceinline__ int tile() const { return (int)(at - item()); }
  // to `next`, which is not behind the end of the item
  __device__ __forceinline__ void go(long long next, long long end) {
    at = next;
    if (at < item() + tiles || at >= end) return;
    if (++head == p.kv_heads) {
      base += (long long)p.kv_heads * tiles;
      head = 0;
      ++s;
      read();
    }
  }
};

// The deal of a call and this CTA's first sequence, from the sequences' lengths, by all threads of the block.
__device__ __forceinline__ void find_start(const AttentionParams &p, long long *shared, Deal &deal, int &s, long long &base) {
  // shared: [0, 8) the warps' sums, 8: sequence, 9: base
  const KeyTiles<TILE> kt(p.page_size);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (int)((p.seq.seqs + THREADS - 1) / THREADS), s0 = threadIdx.x * per, s1 = (int)min((long long)s0 + per, p.seq.seqs);
  auto tiles = [&](int i) { return (long long)max(1, kt.count(sequence_of(p.seq, i).length)) * p.kv_heads; };
  long long sum = 0;
  for (int i = s0; i < s1; ++i) sum += tiles(i);
  long long scan = sum;
#pragma unroll
  for (int b = 1; b < 32; b <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, scan, b);
    if (lane >= b) scan += v;
  }
  if (lane == 31) shared[warp] = scan;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += shared[w];
    total += shared[w];
  }
  deal.total = total;
  deal.ctas = (int)min((long long)gridDim.x, total);
  const long long at = (int)blockIdx.x < deal.ctas ? deal.begin(blockIdx.x) : -1;
  long long here = before + scan - sum;
  if (at >= here && at < here + sum) {
    int i = s0;
    for (long long t = tiles(i); at >= here + t; t = tiles(i)) { here += t; ++i; }
    shared[8] = i;
    shared[9] = here;
  }
  __syncthreads();
  s = (int)shared[8];
  base = shared[9];
}

template <typename T, int CB, int MB>
__global__ void __launch_bounds__(THREADS, 1) attention_token_kernel(const __grid_constant__ TokenLaunch g) {
  using L = Smem<CB, MB>;
  constexpr int STAGES = L::STAGES, NB = CB * 8;                // NB: blocks of 8 channels
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF);
  int *verdict = reinterpret_cast<int *>(smem + L::MISC_OFF + 4);
  long long *found = reinterpret_cast<long long *>(smem + L::MISC_OFF + 8);
  const AttentionParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], WARPS); }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  griddep_launch_dependents();
  griddep_wait();
  Deal deal;
  int s0;
  long long base0;
  find_start(p, found, deal, s0, base0);                        // (its barriers order the initialisation above)
  if ((int)blockIdx.x >= deal.ctas) return;
  const long long first = deal.begin(blockIdx.x), end = deal.begin(blockIdx.x + 1);
  Walk walk(p, first, s0, base0);
  const KeyTiles<TILE> &kt = walk.kt;
  int fail_code = 0;

  if (warp == WARPS) {
    // ---- the producer: a lane per copy, [K or V][64 channels][page of the tile]
    const int boxes = kt.pages ? kt.pages : 1, bytes = 2 * CB * boxes * kt.box() * 128;
    const int which = lane / boxes, page_in_tile = lane - which * boxes, cb = which % CB;
    const bool mine = lane < 2 * CB * boxes, values = which >= CB;
    const CUtensorMap *map = values ? &g.vmap : &g.kmap;
    // the page and the first token in it of this lane's copy; a page that is not there: one outside the map
    auto place = [&](int &page, int &token) {
      page = (int)p.seq.pages;
      token = 0;
      if (!mine) return;
      const int t = walk.tile();
      if (!kt.page) {
        page = walk.s;
        token = t * TILE;
        return;
      }
      const int i = kt.pages ? t * kt.pages + page_in_tile : t / kt.parts;
      if (!kt.pages) token = t % kt.parts * TILE;
      if ((long long)i * kt.page >= walk.q.length) return;      // behind the sequence's end
      const int named = p.seq.table[walk.s * p.seq.width + i];
      if (named >= 0 && named < p.seq.pages) page = named;
      else if (which == 0) report_status(p.status, ST_BAD_PAGE);
    };
    int stage = 0, page, token;
    uint32_t phase = 1;
    place(page, token);
    for (long long i = first; i < end; ++i) {
      const int head = walk.head, now = page, at = token;
      if (i + 1 < end) {                                        // the next tile's page is on its way while this one's slot is waited for
        walk.go(i + 1, end);
        place(page, token);
      }
      if (!mbar_wait_warp(&empty[stage], phase, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_PRODUCER; break; }
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
      __syncwarp();
      if (mine)
        tma_tile_4d(smem + stage * L::STAGE + which * BOX_BYTES + page_in_tile * kt.page * 128, map, cb * 64, at, head, now, &full[stage]);
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
  } else {
    // ---- the consumers.  Accumulators of a lane: rows lane / 4 and lane / 4 + 8 of a block, channels 2 * (lane % 4) and the next of eight
    const int group = p.heads / p.kv_heads, quad = lane & 3, ksteps = (p.head_dim + 15) / 16;
    const float c = p.scale * 1.4426950408889634f;
    float4 *merge = reinterpret_cast<float4 *>(smem + L::MERGE_OFF);
    float2 *ml = reinterpret_cast<float2 *>(smem + L::ML_OFF);
    const int kid = lane >> 3, krow = lane & 7;
    const uint32_t k_off = (warp * 16 + (kid >> 1) * 8 + krow) * 128, v_off = (warp * 16 + (kid & 1) * 8 + krow) * 128;
    int stage = 0;
    uint32_t phase = 0;
    while (walk.at < end) {
      const long long item = walk.item(), item_end = item + walk.tiles, stop = min(end, item_end);
      const int t0 = walk.tile(), t1 = (int)(stop - item), rows = walk.q.n * group, length = walk.q.length;
      // Q of this key head's rows, in the products' own order
      uint32_t q[MB][CB * 4][4];
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = b * 16 + half * 8 + (lane >> 2);
          const T *src = static_cast<const T *>(p.q) + (long long)(walk.q.first + r / group) * p.ld_q + (long long)(walk.head * group + r % group) * p.head_dim;
#pragma unroll
          for (int k = 0; k < CB * 4; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int ch = k * 16 + j * 8 + quad * 2;
              q[b][k][half + 2 * j] = r < rows && ch < p.head_dim ? *reinterpret_cast<const uint32_t *>(src + ch) : 0u;
            }
        }
      float o[MB][NB][4], m[MB][2], l[MB][2];
      int seen[MB][2];                                          // the first key that a row does not see
#pragma unroll
      for (int b = 0; b < MB; ++b) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[b][n][i] = 0.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          m[b][half] = -INFINITY;
          l[b][half] = 0.0f;
          const int r = b * 16 + half * 8 + (lane >> 2);
          seen[b][half] = p.causal ? length - walk.q.n + r / group + 1 : length;
        }
      }
      const int seen_by_all = p.causal ? length - walk.q.n + 1 : length;
      for (int t = t0; t < t1; ++t) {
        if (!mbar_wait_warp(&full[stage], phase, abort_flag)) fail_code = ST_WAIT_TIMEOUT_MMA;
        const int key0 = kt.first(t) + warp * 16, here = kt.held(t, length) - warp * 16;     // of this warp's 16 keys: how many there are
        if (here > 0) {
          const uint32_t kb = smem_u32(smem + stage * L::STAGE), vb = kb + CB * BOX_BYTES;
          const bool whole = here >= 16 && key0 + 16 <= seen_by_all;
          float sc[MB][2][4];
#pragma unroll
          for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[b][i >> 2][i & 3] = 0.0f;
#pragma unroll
          for (int k = 0; k < CB * 4; ++k) {
            if (k < ksteps) {
              uint32_t kf[4];
              ldmatrix4(kf, kb + (k >> 2) * BOX_BYTES + k_off + ((((k & 3) * 2 + (kid & 1)) ^ krow) << 4));
#pragma unroll
              for (int b = 0; b < MB; ++b) {
                mma16816<T>(sc[b][0], q[b][k], kf[0], kf[1]);
                mma16816<T>(sc[b][1], q[b][k], kf[2], kf[3]);
              }
            }
          }
          uint32_t pf[MB][4];
          bool moved = false;
          float keep[MB][2];
#pragma unroll
          for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float z[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                z[i] = sc[b][i >> 1][half * 2 + (i & 1)] * c;
                if (!whole) {
                  const int key = (i >> 1) * 8 + quad * 2 + (i & 1);
                  if (key >= here || key0 + key >= seen[b][half]) z[i] = -INFINITY;
                }
              }
              float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
              top = fmaxf(top, m[b][half]);
              const float from = top == -INFINITY ? 0.0f : top;
              keep[b][half] = exp2_approx(m[b][half] - from);
              moved |= top > m[b][half];
              m[b][half] = top;
              float w[4], sum = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; ++i) { w[i] = exp2_approx(z[i] - from); sum += w[i]; }
              l[b][half] = l[b][half] * keep[b][half] + sum;     // (of this lane's keys: the four lanes of a row meet at the end)
              pf[b][half] = pack2<T>(w[0], w[1]);
              pf[b][half + 2] = pack2<T>(w[2], w[3]);
            }
          if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
              for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b][n][i] *= keep[b][i >> 1];
          }
          // values of places that hold no keys may be anything, and 0 times anything is not always 0
          uint32_t mask[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
          if (here < 16) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int key = j * 8 + quad * 2;
              mask[j] = (key < here ? 0xFFFFu : 0u) | (key + 1 < here ? 0xFFFF0000u : 0u);
            }
          }
#pragma unroll
          for (int n = 0; n < NB; n += 2) {
            uint32_t vf[4];
            ldmatrix4_trans(vf, vb + (n >> 3) * BOX_BYTES + v_off + ((((n & 7) + (kid >> 1)) ^ krow) << 4));
            if (here < 16) {
#pragma unroll
              for (int i = 0; i < 4; ++i) vf[i] &= mask[i & 1];
            }
#pragma unroll
            for (int b = 0; b < MB; ++b) {
              mma16816<T>(o[b][n], pf[b], vf[0], vf[1]);
              mma16816<T>(o[b][n + 1], pf[b], vf[2], vf[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      // ---- the warps' results together
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float sum = l[b][half];
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
          if (quad == 0) ml[warp * MB * 16 + b * 16 + half * 8 + (lane >> 2)] = make_float2(m[b][half], sum);
        }
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int n = 0; n < NB; ++n)
          merge[((warp * MB + b) * NB + n) * 32 + lane] = make_float4(o[b][n][0], o[b][n][1], o[b][n][2], o[b][n][3]);
      named_bar_sync(1, WARPS * 32);
      // A warp takes every fourth block of channels.  Piece of a whole item: out; otherwise to the workspace, and the last one there joins all of them.
      const int c0 = deal.owner(item), c1 = deal.owner(item_end - 1);
      const bool alone = c0 == c1;
      float *mine = g.w.partial + ((size_t)blockIdx.x * 2 + (item >= first ? 1 : 0)) * PARTIAL_FLOATS;
      constexpr int PER = NB / WARPS;
      float4 sum[MB][PER];
      float lsum[MB][2];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        float weight[WARPS][2], top[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = b * 16 + half * 8 + (lane >> 2);
          float2 x[WARPS];
          top[half] = -INFINITY;
          lsum[b][half] = 0.0f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) { x[w] = ml[w * MB * 16 + r]; top[half] = fmaxf(top[half], x[w].x); }
          const float from = top[half] == -INFINITY ? 0.0f : top[half];
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            weight[w][half] = exp2_approx(x[w].x - from);
            lsum[b][half] += x[w].y * weight[w][half];
          }
          if (!alone && warp == 0 && quad == 0) *reinterpret_cast<float2 *>(mine + PARTIAL_ROWS * 128 + r * 2) = make_float2(top[half], lsum[b][half]);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int n = i * WARPS + warp;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            const float4 x = merge[((w * MB + b) * NB + n) * 32 + lane];
            v.x += x.x * weight[w][0]; v.y += x.y * weight[w][0];
            v.z += x.z * weight[w][1]; v.w += x.w * weight[w][1];
          }
          sum[b][i] = v;
          if (!alone) reinterpret_cast<float4 *>(mine)[(b * NB + n) * 32 + lane] = v;
        }
      }
      bool write = alone;
      if (!alone) {
        __threadfence();
        named_bar_sync(1, WARPS * 32);
        if (threadIdx.x == 0) {
          const int last = atomicAdd(&g.w.arrived[c0], 1) == c1 - c0;
          if (last) g.w.arrived[c0] = 0;
          *verdict = last;
          __threadfence();
        }
        named_bar_sync(1, WARPS * 32);
        write = *verdict != 0;
        if (write) {
          auto part = [&](int cta) { return g.w.partial + ((size_t)cta * 2 + (cta == c0 ? 1 : 0)) * PARTIAL_FLOATS; };
#pragma unroll
          for (int b = 0; b < MB; ++b) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 4
            for (int cta = c0; cta <= c1; ++cta)
#pragma unroll
              for (int half = 0; half < 2; ++half)
                top[half] = fmaxf(top[half], __ldcg(part(cta) + PARTIAL_ROWS * 128 + (b * 16 + half * 8 + (lane >> 2)) * 2));
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[b][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            lsum[b][0] = lsum[b][1] = 0.0f;
#pragma unroll 4
            for (int cta = c0; cta <= c1; ++cta) {
              const float *from = part(cta);
              float weight[2];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float2 x = __ldcg(reinterpret_cast<const float2 *>(from + PARTIAL_ROWS * 128 + (b * 16 + half * 8 + (lane >> 2)) * 2));
                weight[half] = exp2_approx(x.x - (top[half] == -INFINITY ? 0.0f : top[half]));
                lsum[b][half] += x.y * weight[half];
              }
#pragma unroll
              for (int i = 0; i < PER; ++i) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(from) + (b * NB + i * WARPS + warp) * 32 + lane);
                sum[b][i].x += x.x * weight[0]; sum[b][i].y += x.y * weight[0];
                sum[b][i].z += x.z * weight[1]; sum[b][i].w += x.w * weight[1];
              }
            }
          }
        }
      }
      if (write) {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = b * 16 + half * 8 + (lane >> 2);
            if (r >= rows) continue;
            const float total = lsum[b][half], inv = total == 0.0f ? 0.0f : 1.0f / total;
            T *out = static_cast<T *>(p.out) + (long long)(walk.q.first + r / group) * p.ld_out + (long long)(walk.head * group + r % group) * p.head_dim;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int ch = (i * WARPS + warp) * 8 + quad * 2;
              const float4 v = sum[b][i];
              if (ch < p.head_dim) *reinterpret_cast<uint32_t *>(out + ch) = half ? pack2<T>(v.z * inv, v.w * inv) : pack2<T>(v.x * inv, v.y * inv);
            }
          }
      }
      walk.go(stop, end);
      named_bar_sync(1, WARPS * 32);                            // the merge area may be written again
    }
  }
  if (fail_code != 0 && lane == 0) report_status(p.status, fail_code);
}

template <typename T, int CB, int MB>
cudaError_t go(TokenLaunch &g, cudaStream_t s) {
  using L = Smem<CB, MB>;
  return launch_overlapped(attention_token_kernel<T, CB, MB>, dim3(g.p.num_sms), dim3(THREADS), L::TOTAL, s, g);
}
template <typename T>
cudaError_t go(TokenLaunch &g, int rows, cudaStream_t s) {
  if (g.p.head_dim <= 64) return rows <= 16 ? go<T, 1, 1>(g, s) : go<T, 1, 2>(g, s);
  return rows <= 16 ? go<T, 2, 1>(g, s) : go<T, 2, 2>(g, s);
}
template <typename K>
cudaError_t allow(K kern, int smem) { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }
template <typename T>
cudaError_t allow_all() {
  cudaError_t e = allow(attention_token_kernel<T, 1, 1>, Smem<1, 1>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_token_kernel<T, 1, 2>, Smem<1, 2>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_token_kernel<T, 2, 1>, Smem<2, 1>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_token_kernel<T, 2, 2>, Smem<2, 2>::TOTAL);
  return e;
}

// the most rows that a key head of one sequence has
long long most_rows(const AttentionParams &p) { return (p.seq.starts ? p.seq.rows : p.seq.each) * (p.heads / p.kv_heads); }

}  // namespace

bool encode_keys(CUtensorMap *m, const AttentionParams &p, const void *base, int rows) {
  PFN_encodeTiled fn = get_encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)(p.page_size ? p.page_size : p.seq.width), (cuuint64_t)p.kv_heads, (cuuint64_t)p.seq.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)p.ld_token * 2, (cuuint64_t)p.ld_head * 2, (cuuint64_t)p.ld_page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, one[4] = {1, 1, 1, 1};
  return fn(m, p.et == ET_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t init_attention() {
  const cudaError_t e = allow_all<__nv_bfloat16>();
  return e == cudaSuccess ? allow_all<__half>() : e;
}

bool attention_token_takes(const AttentionParams &p) {
  return p.words && p.head_dim <= 128 && p.page_size % 8 == 0 && p.seq.width > 0 && p.seq.pages > 0 && most_rows(p) <= 32;
}

cudaError_t launch_attention_token(const AttentionParams &p, const AttentionWorkspace &w, cudaStream_t s) {
  TokenLaunch g;
  g.p = p;
  g.w = w;
  const int rows = KeyTiles<TILE>(p.page_size).box();
  if (!encode_keys(&g.kmap, p, p.k, rows) || !encode_keys(&g.vmap, p, p.v, rows)) return cudaErrorInvalidValue;
  return p.et == ET_BF16 ? go<__nv_bfloat16>(g, (int)most_rows(p), s) : go<__half>(g, (int)most_rows(p), s);
}

}  // namespace elb
