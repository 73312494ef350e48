// Attention of few new tokens over long keys: a step of answers.
//
// What it is made of is reading K and V once.  All rows of a key head (its g heads times the sequence's new tokens) share a tile of
// 32 keys; the call's tiles, of all sequences and key heads in order, are dealt out evenly to two or three CTAs per SM, whatever their lengths, so a
// sequence's length is split wherever that falls.  A CTA's producer keeps 32 to 64 KB of tiled copies in flight, and four warps take a tile each, in
// turns, with a running maximum, sum and result of their own, so that they meet only at the end of a piece.  Then their results are joined,
// written out if the piece is all of its key head's keys, and left in the workspace otherwise, where the last CTA of those that share it joins
// them in the order of the keys: no result depends on timing.  While one CTA of an SM does that, the others read.
//
// Products are mma.sync m16n8k16: 16 rows are the least a matrix instruction takes, and at HBM's rate (23 bytes per SM and cycle) one of them is wanted
// every 22 cycles, far below what it can do; tcgen05 would pad 128 rows and bring each score through tensor memory.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"
#include "umma.cuh"

namespace elb {

namespace {

constexpr int TILE = 32, WARPS = 4, THREADS = WARPS * 32 + 32;
constexpr int BOX_BYTES = TILE * 128;                           // the keys of a tile, 64 channels each

// CB: boxes of 64 channels; MB: blocks of 16 rows, each a warp's.  The warps of a block take turns in TURNS.
template <int CB, int MB>
struct Smem {
  static constexpr int CTAS = CB == 1 ? 3 : 2;                  // per SM
  static constexpr int TURNS = WARPS / MB, NB = CB * 8;
  static constexpr int STAGE = 2 * CB * BOX_BYTES;
  // A multiple of the turns: the same warps then come back to a stage, and see each of its phases.  (One bit of parity does not tell a stage that has
  // not been filled from one that has been twice.)
  static constexpr int STAGES = (CB == 1 && MB == 2 ? 6 : 4) / TURNS * TURNS;
  static constexpr int Q_BYTES = CB * MB * 16 * 128, Q_OFF = STAGES * STAGE;       // two slots
  static constexpr int MERGE_OFF = Q_OFF + 2 * Q_BYTES;
  static constexpr int MERGE = WARPS / 2 * NB * 32 * 16;        // the results of half of the warps
  static constexpr int ML_OFF = MERGE_OFF + MERGE;              // maxima and sums, [WARPS][16]
  static constexpr int BAR_OFF = ML_OFF + WARPS * 16 * 8;       // full[S], empty[S], qfull[2], qempty[2]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 4) * 8;
  static constexpr int TOTAL = MISC_OFF + 128 + 1024;
  static constexpr int PARTIAL = MB * 16 * (CB * 64 + 2);       // floats of a partial result: rows, then their maxima and sums
};

struct alignas(64) TokenLaunch {
  CUtensorMap kmap, vmap, qmap;
  AttentionParams p;
  AttentionWorkspace w;
  int box;                          // new tokens of a copy of queries
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

__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// The call's tiles in order: sequences, their key heads, their tiles (one at least, so that every row is written).  The first `more` CTAs take
// each + 1 of them, the others `each`.
struct Deal {
  long long each, more;
  int ctas;
  __device__ __forceinline__ Deal(long long total) {
    ctas = (int)min((long long)gridDim.x, total);
    each = quotient(total, ctas);
    more = total - each * ctas;
  }
  __device__ __forceinline__ long long begin(int c) const { return c * each + min((long long)c, more); }
  __device__ __forceinline__ int owner(long long tile) const {
    const long long of_more = more * (each + 1);
    return (int)(tile < of_more ? quotient(tile, each + 1) : more + quotient(tile - of_more, each));
  }
};
// Where a CTA is: tile t of `tiles` of key head `head` of sequence s
struct Walk {
  const AttentionParams &p;
  const KeyTiles<TILE> kt;
  Sequence q;
  int s, head, tiles, t;
  __device__ __forceinline__ Walk(const AttentionParams &p, long long at, int s, long long base) : p(p), kt(p.page_size), s(s) {
    read();
    head = (int)quotient(at - base, tiles);
    t = (int)(at - base - (long long)head * tiles);
  }
  __device__ __forceinline__ void read() {
    q = sequence_of(p.seq, s);
    tiles = max(1, kt.count(q.length));
  }
  // behind the last tile of a key head, to the next one's first (the call has another tile)
  __device__ __forceinline__ void wrap() {
    if (t < tiles) return;
    t = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    ++s;
    read();
  }
};

// The tiles of a call and, of CTA `cta` of its deal, the first sequence and where that begins, from the sequences' lengths, by all threads of the block.
__device__ __forceinline__ Deal find_start(const AttentionParams &p, long long *shared, int cta, int &s, long long &base) {
  // shared: [0, 5) the warps' sums, 6: sequence, 7: base
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
  const Deal deal(total);
  const long long at = cta < deal.ctas ? deal.begin(cta) : -1;
  long long here = before + scan - sum;
  if (at >= here && at < here + sum) {
    int i = s0;
    if (per > 1)
      for (long long t = tiles(i); at >= here + t; t = tiles(i)) { here += t; ++i; }
    shared[6] = i;
    shared[7] = here;
  }
  __syncthreads();
  s = (int)shared[6];
  base = shared[7];
  return deal;
}

template <typename T, int CB, int MB>
__global__ void __launch_bounds__(THREADS, Smem<CB, MB>::CTAS) attention_token_kernel(const __grid_constant__ TokenLaunch g) {
  using L = Smem<CB, MB>;
  constexpr int STAGES = L::STAGES, NB = L::NB;                 // NB: blocks of 8 channels
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *qfull = empty + STAGES, *qempty = qfull + 2;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF);
  int *verdict = reinterpret_cast<int *>(smem + L::MISC_OFF + 4);
  long long *found = reinterpret_cast<long long *>(smem + L::MISC_OFF + 8);
  const AttentionParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    tma_prefetch_desc(&g.qmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], MB); }
    for (int i = 0; i < 2; ++i) { mbar_init(&qfull[i], 1); mbar_init(&qempty[i], WARPS); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  // rows of queries that no copy fills
  for (int i = threadIdx.x; i < 2 * L::Q_BYTES / 16; i += THREADS) reinterpret_cast<uint4 *>(smem + L::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  griddep_launch_dependents();
  griddep_wait();
  int s0;
  long long base0;
  const Deal deal = find_start(p, found, blockIdx.x, s0, base0);       // (its barriers order the initialisation above)
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
    uint8_t *dst = smem + which * BOX_BYTES + page_in_tile * kt.page * 128;
    // What this lane copies for a tile.  Tables are read some tiles ahead and looked at when the copies are issued: a read takes as long as a tile does.
    constexpr int AHEAD = 4;
    struct { int page, token, head, row; } next[AHEAD];           // row: of the queries, in front of a piece's first tile
    auto read = [&](int j, bool piece) {
      walk.wrap();
      next[j].head = walk.head;
      next[j].row = piece || walk.t == 0 ? walk.q.first : -1;
      next[j].token = 0;
      next[j].page = (int)p.seq.pages;                          // one outside the map: zeros
      if (!kt.page) {
        next[j].page = walk.s;
        next[j].token = walk.t * TILE;
      } else if (mine) {
        const int i = kt.pages ? walk.t * kt.pages + page_in_tile : walk.t / kt.parts;
        if (!kt.pages) next[j].token = walk.t % kt.parts * TILE;
        if ((long long)i * kt.page < walk.q.length) next[j].page = p.seq.table[walk.s * p.seq.width + i];
        else next[j].token = -1;                                // behind the sequence's end
      }
      ++walk.t;
    };
    int stage = 0, issued = 0, pieces = 0;
    uint32_t phase = 1;
    const int tiles = (int)min(end - first, 0x7FFFFFFFll);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (j < tiles) read(j, j == 0);
    bool ok = true;
    for (int i = 0; i < tiles && ok; i += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i + j >= tiles || !ok) break;
        if (next[j].row >= 0) {
          uint64_t *bar = &qfull[pieces & 1];
          if (!mbar_poll_warp(&qempty[pieces & 1], ((pieces >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(bar, CB * g.box * group * 128);
          __syncwarp();
          if (lane < CB) tma_tile_3d(smem + L::Q_OFF + (pieces & 1) * L::Q_BYTES + lane * MB * 16 * 128, &g.qmap, lane * 64, next[j].head * group, next[j].row, bar);
          ++pieces;
        }
        if (!mbar_poll_warp(&empty[stage], phase, abort_flag)) { ok = false; break; }
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
        __syncwarp();
        if (mine) {
          int page = next[j].page;
          if ((unsigned)page >= (unsigned)p.seq.pages && kt.page) {
            if (next[j].token >= 0) report_status(p.status, ST_BAD_PAGE);
            page = (int)p.seq.pages;
          }
          tma_tile_4d(dst + stage * L::STAGE, map, cb * 64, max(next[j].token, 0), next[j].head, page, &full[stage]);
        }
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        if (i + j + AHEAD < tiles) read(j, false);
        ++issued;
      }
    }
    if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
    // no copy is in flight when the block ends, however its other warps end
    for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1, abort_flag);
    for (int i = max(0, pieces - 2); i < pieces; ++i) mbar_wait_warp(&qfull[i & 1], (i >> 1) & 1, abort_flag);
  } else {
    // ---- the consumers.  Accumulators of a lane: rows lane / 4 and lane / 4 + 8 of a block, channels 2 * (lane % 4) and the next of eight
    const int quad = lane & 3, ksteps = (p.head_dim + 15) / 16, block = warp % MB, turn = warp / MB;
    const float c = fabsf(p.scale) * 1.4426950408889634f;
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;    // a negative scale goes to the queries, so that the largest product has the largest score
    float4 *merge = reinterpret_cast<float4 *>(smem + L::MERGE_OFF);
    float2 *ml = reinterpret_cast<float2 *>(smem + L::ML_OFF);
    const int kid = lane >> 3, krow = lane & 7;
    const uint32_t k_off = ((kid >> 1) * 8 + krow) * 128, v_off = ((kid & 1) * 8 + krow) * 128;
    int index = 0, pieces = 0;                                  // index: of a piece's first tile among this CTA's
    for (long long at = first; at < end; ++pieces) {
      walk.wrap();
      const int t0 = walk.t, t1 = (int)min((long long)walk.tiles, t0 + (end - at)), rows = walk.q.n * group, length = walk.q.length;
      const long long item = at - t0, item_end = item + walk.tiles;
      at += t1 - t0;
      int seen[2];                                              // the first key that a row does not see
#pragma unroll
      for (int half = 0; half < 2; ++half) seen[half] = p.causal ? length - walk.q.n + (block * 16 + half * 8 + (lane >> 2)) / group + 1 : length;
      const int seen_by_all = p.causal ? length - walk.q.n + 1 : length;
      // Q of this key head's rows, in the products' own order
      uint32_t q[CB * 4][4];
      if (!mbar_poll_warp(&qfull[pieces & 1], (pieces >> 1) & 1, abort_flag)) fail_code = ST_WAIT_TIMEOUT_MMA;
      const uint32_t qb = smem_u32(smem + L::Q_OFF + (pieces & 1) * L::Q_BYTES) + (block * 16 + (kid & 1) * 8 + krow) * 128;
#pragma unroll
      for (int k = 0; k < CB * 4; ++k) {
        ldmatrix4(q[k], qb + (k >> 2) * MB * 16 * 128 + ((((k & 3) * 2 + (kid >> 1)) ^ krow) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) q[k][i] ^= flip;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&qempty[pieces & 1]);
      float o[NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
      for (int t = t0 + ((turn - index) & (L::TURNS - 1)); t < t1; t += L::TURNS) {
        const int i = index + t - t0, stage = i % STAGES;
        if (!mbar_poll_warp(&full[stage], (i / STAGES) & 1, abort_flag)) fail_code = ST_WAIT_TIMEOUT_MMA;
        const int key0 = kt.first(t), here = kt.held(t, length);
        const uint32_t kb = smem_u32(smem + stage * L::STAGE), vb = kb + CB * BOX_BYTES;
        float sc[4][4];
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i >> 2][i & 3] = 0.0f;
#pragma unroll
        for (int k = 0; k < CB * 4; ++k) {
          if (k < ksteps) {
            const uint32_t at_k = kb + (k >> 2) * BOX_BYTES + k_off + ((((k & 3) * 2 + (kid & 1)) ^ krow) << 4);
            uint32_t k0[4], k1[4];
            ldmatrix4(k0, at_k);
            ldmatrix4(k1, at_k + 16 * 128);
            mma16816<T>(sc[0], q[k], k0[0], k0[1]);
            mma16816<T>(sc[1], q[k], k0[2], k0[3]);
            mma16816<T>(sc[2], q[k], k1[0], k1[1]);
            mma16816<T>(sc[3], q[k], k1[2], k1[3]);
          }
        }
        const bool part = here < TILE;
        if (part || key0 + TILE > seen_by_all) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = (i >> 2) * 8 + quad * 2 + (i & 1);
            if (key >= here || key0 + key >= seen[(i >> 1) & 1]) sc[i >> 2][i & 3] = -INFINITY;
          }
        }
        float keep[2], from[2];
        bool moved = false;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float top = m[half];
#pragma unroll
          for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(sc[n][half * 2], sc[n][half * 2 + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
          from[half] = top == -INFINITY ? 0.0f : top * c;
          keep[half] = exp2_approx(m[half] * c - from[half]);
          moved |= top > m[half];
          m[half] = top;
        }
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
          for (int half = 0; half < 2; ++half) l[half] *= keep[half];
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= keep[i >> 1];
        }
        uint32_t pf[2][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float w0 = exp2_approx(fmaf(sc[n][half * 2], c, -from[half])), w1 = exp2_approx(fmaf(sc[n][half * 2 + 1], c, -from[half]));
            l[half] += w0 + w1;                                 // (of this lane's keys: the four lanes of a row meet at the end)
            pf[n >> 1][half + 2 * (n & 1)] = pack2<T>(w0, w1);  // the second product's operand has 16 bits
          }
        // values of places that hold no keys may be anything, and 0 times anything is not always 0
        uint32_t mask[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = j * 8 + quad * 2;
          mask[j] = (key < here ? 0xFFFFu : 0u) | (key + 1 < here ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int n = 0; n < NB; n += 2) {
          const uint32_t at_v = vb + (n >> 3) * BOX_BYTES + v_off + ((((n & 7) + (kid >> 1)) ^ krow) << 4);
          uint32_t v0[4], v1[4];
          ldmatrix4_trans(v0, at_v);
          ldmatrix4_trans(v1, at_v + 16 * 128);
          if (part) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v0[i] &= mask[i & 1]; v1[i] &= mask[2 + (i & 1)]; }
          }
          mma16816<T>(o[n], pf[0], v0[0], v0[1]);
          mma16816<T>(o[n + 1], pf[0], v0[2], v0[3]);
          mma16816<T>(o[n], pf[1], v1[0], v1[1]);
          mma16816<T>(o[n + 1], pf[1], v1[2], v1[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      index += t1 - t0;
      // ---- The warps' results together: the second two hand theirs to the first two, whose results all four then join, a quarter of the channels each.
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 1);
        l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 2);
        m[half] *= c;
      }
      constexpr int HALF = WARPS / 2;
      if (warp >= HALF) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (quad == 0) ml[warp * 16 + half * 8 + (lane >> 2)] = make_float2(m[half], l[half]);
#pragma unroll
        for (int n = 0; n < NB; ++n) merge[((warp - HALF) * NB + n) * 32 + lane] = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
      }
      named_bar_sync(1, WARPS * 32);
      if (warp < HALF) {
        float mine[2], theirs[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float2 x = ml[(warp + HALF) * 16 + half * 8 + (lane >> 2)];
          const float top = fmaxf(m[half], x.x), from = top == -INFINITY ? 0.0f : top;
          mine[half] = exp2_approx(m[half] - from);
          theirs[half] = exp2_approx(x.x - from);
          if (quad == 0) ml[warp * 16 + half * 8 + (lane >> 2)] = make_float2(top, l[half] * mine[half] + x.y * theirs[half]);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float4 &at = merge[(warp * NB + n) * 32 + lane];
          const float4 x = at;
          at = make_float4(o[n][0] * mine[0] + x.x * theirs[0], o[n][1] * mine[0] + x.y * theirs[0], o[n][2] * mine[1] + x.z * theirs[1],
                           o[n][3] * mine[1] + x.w * theirs[1]);
        }
      }
      named_bar_sync(1, WARPS * 32);
      // A warp takes every fourth block of channels.  Piece of a whole item: out; otherwise to the workspace, and the last one there joins all of them.
      const int c0 = deal.owner(item), c1 = deal.owner(item_end - 1);
      const bool alone = c0 == c1;
      constexpr int PER = NB / WARPS, COPIES = HALF / MB;
      auto part = [&](int cta) { return g.w.partial + ((size_t)cta * 2 + (cta == c0 ? 1 : 0)) * L::PARTIAL; };     // (its last piece, or its first)
      float *mine = part(blockIdx.x);
      float4 sum[MB][PER];
      float lsum[MB][2];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        float weight[COPIES][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = half * 8 + (lane >> 2);
          float2 x[COPIES];
          float top = -INFINITY;
          lsum[b][half] = 0.0f;
#pragma unroll
          for (int w = 0; w < COPIES; ++w) { x[w] = ml[(MB > 1 ? b : w) * 16 + r]; top = fmaxf(top, x[w].x); }
          const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
          for (int w = 0; w < COPIES; ++w) {
            weight[w][half] = exp2_approx(x[w].x - from);
            lsum[b][half] += x[w].y * weight[w][half];
          }
          if (!alone && warp == 0 && quad == 0 && b * 16 + r < rows)
            *reinterpret_cast<float2 *>(mine + MB * 16 * CB * 64 + (b * 16 + r) * 2) = make_float2(top, lsum[b][half]);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int n = i * WARPS + warp;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < COPIES; ++w) {
            const float4 x = merge[((MB > 1 ? b : w) * NB + n) * 32 + lane];
            v.x += x.x * weight[w][0]; v.y += x.y * weight[w][0];
            v.z += x.z * weight[w][1]; v.w += x.w * weight[w][1];
          }
          sum[b][i] = v;
          if (!alone && b * 16 + (lane >> 2) < rows) reinterpret_cast<float4 *>(mine)[(b * NB + n) * 32 + lane] = v;
        }
      }
      bool write = alone;
      if (!alone) {
        named_bar_sync(1, WARPS * 32);
        // (released and acquired by one thread for the block, whose other threads are ordered by the barriers)
        if (threadIdx.x == 0) {
          int before;
          asm volatile("atom.acq_rel.gpu.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(g.w.arrived + c0) : "memory");
          if (before == c1 - c0) g.w.arrived[c0] = 0;
          *verdict = before == c1 - c0;
        }
        named_bar_sync(1, WARPS * 32);
        write = *verdict != 0;
        if (write) {
#pragma unroll
          for (int b = 0; b < MB; ++b) {
            if (b * 16 + (lane >> 2) >= rows) continue;
            float top[2] = {-INFINITY, -INFINITY};
            auto stats = [&](int cta, int half) {
              const int r = min(b * 16 + half * 8 + (lane >> 2), rows - 1);
              return __ldcg(reinterpret_cast<const float2 *>(part(cta) + MB * 16 * CB * 64 + r * 2));
            };
#pragma unroll 8
            for (int cta = c0; cta <= c1; ++cta)
#pragma unroll
              for (int half = 0; half < 2; ++half) top[half] = fmaxf(top[half], stats(cta, half).x);
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[b][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            lsum[b][0] = lsum[b][1] = 0.0f;
#pragma unroll 8
            for (int cta = c0; cta <= c1; ++cta) {
              const float *from = part(cta);
              float weight[2];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float2 x = stats(cta, half);
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
            const int r = b * 16 + half * 8 + (lane >> 2), token = r / group;
            if (r >= rows) continue;
            const float total = lsum[b][half], inv = total == 0.0f ? 0.0f : 1.0f / total;
            T *out = static_cast<T *>(p.out) + (long long)(walk.q.first + token) * p.ld_out + (long long)(walk.head * group + r - token * group) * p.head_dim;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int ch = (i * WARPS + warp) * 8 + quad * 2;
              const float4 v = sum[b][i];
              if (ch < p.head_dim) *reinterpret_cast<uint32_t *>(out + ch) = half ? pack2<T>(v.z * inv, v.w * inv) : pack2<T>(v.x * inv, v.y * inv);
            }
          }
      }
      walk.t = t1;
      named_bar_sync(1, WARPS * 32);                            // the merge area may be written again
    }
  }
  if (fail_code != 0 && lane == 0) report_status(p.status, fail_code);
}

template <typename T, int CB, int MB>
cudaError_t go(TokenLaunch &g, cudaStream_t s) {
  using L = Smem<CB, MB>;
  static_assert(L::CTAS <= TOKEN_CTAS && L::CTAS * L::PARTIAL <= TOKEN_PARTIAL, "");
  return launch_overlapped(attention_token_kernel<T, CB, MB>, dim3(g.p.num_sms * L::CTAS), dim3(THREADS), L::TOTAL, s, g);
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

bool encode_queries(CUtensorMap *m, const AttentionParams &p, int heads, int tokens) {
  PFN_encodeTiled fn = get_encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.heads, (cuuint64_t)p.seq.rows};
  const cuuint64_t strides[2] = {(cuuint64_t)p.head_dim * 2, (cuuint64_t)p.ld_q * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens}, one[3] = {1, 1, 1};
  return fn(m, p.et == ET_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(p.q), dims, strides, box, one,
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
  const int rows = KeyTiles<TILE>(p.page_size).box(), group = p.heads / p.kv_heads;
  g.box = (int)most_rows(p) / group;
  if (!encode_keys(&g.kmap, p, p.k, rows) || !encode_keys(&g.vmap, p, p.v, rows) || !encode_queries(&g.qmap, p, group, g.box)) return cudaErrorInvalidValue;
  return p.et == ET_BF16 ? go<__nv_bfloat16>(g, (int)most_rows(p), s) : go<__half>(g, (int)most_rows(p), s);
}

}  // namespace elb
