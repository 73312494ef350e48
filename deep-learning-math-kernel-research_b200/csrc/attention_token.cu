// Attention of few new tokens over long keys: a step of answers.
//
// What it is made of is reading K and V once.  All rows of a key head (its g heads times the sequence's new tokens) share a tile of
// 32 keys; the call's tiles, of all sequences and key heads in order, are dealt out evenly to two or three CTAs per SM, whatever their lengths, so a
// sequence's length is split wherever that falls.  Four warps of a CTA take a tile each, in turns, with a running maximum, sum and result of their own, so
// that they meet only at the end of a piece; four others bring the tiles, in turns too, since each takes about 1100 cycles to issue one.  Then their results are joined,
// written out if the piece is all of its key head's keys, and left in the workspace otherwise, where the last CTA of those that share it joins
// them in the order of the keys: no result depends on timing.  While one CTA of an SM does that, the others read.
//
// Products are mma.sync m16n8k16: 16 rows are the least a matrix instruction takes, and at HBM's rate (23 bytes per SM and cycle) one of them is wanted
// every 22 cycles, far below what it can do; tcgen05 would pad 128 rows and bring each score through tensor memory.
//
// 64 x 1 tokens of 32 heads of 128 over 8 behind 500 to 16000: 334 to 350 us, 6.2 to 6.6 TB/s, a copy's rate.  Smaller calls wait: some 5 us until the first tiles are there (lengths, table,
// copies, one after the other), 3 to 6 for the join.
#include <cmath>
#include <type_traits>

#include "attention.cuh"
#include "elb_common.cuh"
#include "umma.cuh"

namespace elb {

namespace {

constexpr int TILE = 32, WARPS = 4, PRODUCERS = 4, THREADS = (WARPS + PRODUCERS) * 32;
constexpr int BOX_BYTES = TILE * 128;                           // the keys of a tile, 64 channels each

// CB: boxes of 64 channels; MB: blocks of 16 rows, each a warp's.  The warps of a block take turns in TURNS.
template <int CB, int MB>
struct Smem {
  static constexpr int CTAS = CB == 1 ? 3 : 2;                  // per SM (64 channels with 2: 24 x 1 token of 12 heads 29 -> 31.5 us, 64 x 1 of 16 140 -> 155)
  static constexpr int REGS = CB == 1 ? 112 : 208, REGS_PRODUCER = 48;      // of threads, together the (80 or 128) * 256 that a CTA has
  static constexpr int TURNS = WARPS / MB, NB = CB * 8;
  static constexpr int STAGE = 2 * CB * BOX_BYTES;
  // A multiple of the turns, also of the producers: the same warps then come back to a stage, and see each of its phases.  (One bit of parity does not tell a stage that has
  // not been filled from one that has been twice.)
  static constexpr int STAGES = 4;
  static_assert(STAGES % TURNS == 0 && STAGES % PRODUCERS == 0, "");
  static constexpr int Q_BYTES = CB * MB * 16 * 128, Q_OFF = STAGES * STAGE;       // two slots, of a piece's queries and the next one's
  static constexpr int PITCH = CB * 64 + 8;                     // floats of a warp's row among the results (8: its lanes' banks)
  static constexpr int MERGE_OFF = Q_OFF + 2 * Q_BYTES;
  static constexpr int COPIES = MB > 1 ? 1 : WARPS;             // results of a block that lie there at the end; two blocks: a warp's, joined with its partner's
  static constexpr int MERGE = COPIES * MB * 16 * PITCH * 4;
  static constexpr int ML_OFF = MERGE_OFF + MERGE;              // maxima and sums, [WARPS][16]
  static constexpr int BAR_OFF = ML_OFF + WARPS * 16 * 8;       // full[S], empty[S], landed[S], qfull[2]
  static constexpr int MISC_OFF = BAR_OFF + (3 * STAGES + 2) * 8;
  // The pieces in whose values some were cleared, each at its number modulo SPOILT (copies are a ring of tiles ahead, and a piece has one at least), as the number's lower
  // bits and 1.  (A piece that is taken for another has none to add.)
  static constexpr int SPOILT = 8, PIECE_BITS = 0x7FFF;
  static_assert(SPOILT > STAGES, "");
  static constexpr int TOTAL = MISC_OFF + 8 + SPOILT * 4 + 1024;       // (room to align)
  static constexpr int PARTIAL = MB * 16 * (CB * 64 + 2);       // floats of a partial result: rows, then their maxima and sums
  static_assert(CTAS * (TOTAL + 1024) <= 228 * 1024, "");
};

struct alignas(64) TokenLaunch {
  CUtensorMap kmap, vmap, qmap;
  AttentionParams p;
  AttentionWorkspace w;
  int box;                          // new tokens of a copy of queries
};

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

// A key head's tiles: one at least, so that every row is written, and no more for sequences without new tokens
__device__ __forceinline__ int tiles_of(const KeyTiles<TILE> &kt, const Sequence &q) { return q.n > 0 ? max(1, kt.count(q.length)) : 1; }
// The call's tiles lie in order: sequences, their key heads, their tiles.
// Their deal and where this CTA starts, from the sequences' lengths, by a warp.
struct Start { Sequence q; long long base; int s; };
__device__ __forceinline__ Deal find_start(const AttentionParams &p, int cta, Start &start) {
  const KeyTiles<TILE> kt(p.page_size);
  const int lane = threadIdx.x & 31, per = (int)((p.seq.seqs + 31) / 32), s0 = lane * per, s1 = (int)min((long long)s0 + per, p.seq.seqs);
  auto tiles = [&](const Sequence &q) { return (long long)tiles_of(kt, q) * p.kv_heads; };
  Sequence q = {0, 0, 0};
  long long sum = 0;
  if (per == 1) {
    if (s0 < s1) {
      q = sequence_of(p.seq, s0);
      sum = tiles(q);
    }
  } else {
#pragma unroll 4
    for (int i = s0; i < s1; ++i) sum += tiles(sequence_of(p.seq, i));
  }
  long long scan = sum;
#pragma unroll
  for (int b = 1; b < 32; b <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, scan, b);
    if (lane >= b) scan += v;
  }
  // (a CTA takes no longer for a tile of each warp than for one)
  const long long total = __shfl_sync(0xFFFFFFFFu, scan, 31);
  const Deal deal(total, min((long long)gridDim.x, (total + WARPS - 1) / WARPS));
  const long long at = cta < deal.ctas ? deal.begin(cta) : 0;
  long long here = scan - sum;
  const int mine = __ffs(__ballot_sync(0xFFFFFFFFu, at >= here && at < here + sum)) - 1;
  int i = s0;
  if (per > 1 && lane == mine) {
    q = sequence_of(p.seq, i);
    for (long long t = tiles(q); at >= here + t; t = tiles(q)) { here += t; q = sequence_of(p.seq, ++i); }
  }
  start.s = __shfl_sync(0xFFFFFFFFu, i, mine);
  start.base = __shfl_sync(0xFFFFFFFFu, here, mine);
  start.q.first = __shfl_sync(0xFFFFFFFFu, q.first, mine);
  start.q.n = __shfl_sync(0xFFFFFFFFu, q.n, mine);
  start.q.length = __shfl_sync(0xFFFFFFFFu, q.length, mine);
  return deal;
}

// Where a CTA is: tile t of `tiles` of key head `head` of sequence s
struct Walk {
  const AttentionParams &p;
  const KeyTiles<TILE> kt;
  Sequence q;
  int s, head, tiles, t;
  __device__ __forceinline__ Walk(const AttentionParams &p, long long at, const Start &start) : p(p), kt(p.page_size), q(start.q), s(start.s) {
    tiles = tiles_of(kt, q);
    head = (int)quotient(at - start.base, tiles);
    t = (int)(at - start.base - (long long)head * tiles);
  }
  // from behind the last tile of a key head to the next one (the call has more)
  __device__ __forceinline__ void wrap() {
    t -= tiles;
    if (++head < p.kv_heads) return;
    head = 0;
    q = sequence_of(p.seq, ++s);
    tiles = tiles_of(kt, q);
  }
};

template <typename T, int CB, int MB>
__global__ void __launch_bounds__(THREADS, Smem<CB, MB>::CTAS) attention_token_kernel(const __grid_constant__ TokenLaunch g) {
  using L = Smem<CB, MB>;
  constexpr int STAGES = L::STAGES, NB = L::NB;                 // NB: blocks of 8 channels
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *landed = empty + STAGES, *qfull = landed + STAGES;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF);
  int *verdict = reinterpret_cast<int *>(smem + L::MISC_OFF + 4);
  volatile int *spoilt = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 8);
  const AttentionParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    tma_prefetch_desc(&g.qmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], MB); mbar_init(&landed[i], 1); }
    for (int i = 0; i < 2; ++i) mbar_init(&qfull[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x >= 32 && threadIdx.x < 32 + L::SPOILT) spoilt[threadIdx.x - 32] = 0;
  // rows of queries that no copy fills
  for (int i = threadIdx.x; i < 2 * L::Q_BYTES / 16; i += THREADS) reinterpret_cast<uint4 *>(smem + L::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  griddep_launch_dependents();
  griddep_wait();
  Start start;
  const Deal deal = find_start(p, blockIdx.x, start);
  if ((int)blockIdx.x >= deal.ctas) return;
  const long long first = deal.begin(blockIdx.x), end = deal.begin(blockIdx.x + 1);
  Walk walk(p, first, start);
  const KeyTiles<TILE> &kt = walk.kt;
  int fail_code = 0;

  if (warp >= WARPS) {
    // ---- a producer: a lane per copy, [K or V][64 channels][page of the tile]
    reg_dealloc<L::REGS_PRODUCER>();
    const int boxes = kt.pages ? kt.pages : 1, bytes = 2 * CB * boxes * kt.box() * 128;
    const int which = lane / boxes, page_in_tile = lane - which * boxes, cb = which % CB;
    const bool mine = lane < 2 * CB * boxes, values = which >= CB;
    const CUtensorMap *map = values ? &g.vmap : &g.kmap;
    uint8_t *dst = smem + which * BOX_BYTES + page_in_tile * kt.page * 128;
    // What this lane copies for a tile.  Tables are read a tile ahead and looked at when the copies are issued.
    constexpr int AHEAD = 2;
    struct { int page, token, head, look; } next[AHEAD];
    int piece = 0;
    auto read = [&](int j) {
      for (; walk.t >= walk.tiles; ++piece) walk.wrap();
      next[j].head = walk.head;
      next[j].look = 0;                                         // or the tile's rows that some of the new tokens do not see, [lowest byte, the next) of a piece
      if (p.causal && walk.q.n > 1) {
        const int from = max(walk.q.length - walk.q.n + 1 - kt.first(walk.t), 0), to = kt.held(walk.t, walk.q.length);
        if (from < to) next[j].look = from | to << 8 | (piece & L::PIECE_BITS) << 16;
      }
      next[j].token = 0;
      next[j].page = (int)p.seq.pages;                          // one outside the map: zeros
      if (!kt.page) {
        next[j].page = walk.s;
        next[j].token = walk.t * TILE;
      } else if (mine) {
        int i = walk.t * kt.pages + page_in_tile;
        if (!kt.pages) {
          i = kt.page_of(walk.t);
          next[j].token = (walk.t - i * kt.parts) * TILE;
        }
        if ((long long)i * kt.page < walk.q.length && walk.q.n > 0) next[j].page = p.seq.table[walk.s * p.seq.width + i];
        else next[j].token = -1;                                // behind the sequence's end, or of one that nobody asks for
      }
      walk.t += PRODUCERS;
    };
    const int tiles = (int)min(end - first, 0x7FFFFFFFll);
    int i = warp - WARPS;
    walk.t += i;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j * PRODUCERS < tiles) read(j);
    bool ok = true;
    uint32_t landed_phase = 0;
    while (i < tiles && ok) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i >= tiles || !ok) break;
        const int stage = i % STAGES;
        if (!mbar_poll_warp(&empty[stage], ((i / STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
        const int look = next[j].look;
        uint64_t *bar = look != 0 ? &landed[stage] : &full[stage];
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
        __syncwarp();
        if (mine) {
          int page = next[j].page;
          if ((unsigned)page >= (unsigned)p.seq.pages && kt.page) {
            if (next[j].token >= 0) report_status(p.status, ST_BAD_PAGE);
            page = (int)p.seq.pages;
          }
          tma_tile_4d(dst + stage * L::STAGE, map, cb * 64, max(next[j].token, 0), next[j].head, page, bar);
        }
        if (look != 0) {                                        // their values are looked at before the tile is handed on
          ok = mbar_poll_warp(bar, landed_phase, abort_flag);
          landed_phase ^= 1;
          if (clear_not_finite<T, CB, BOX_BYTES, 1>(smem + stage * L::STAGE + CB * BOX_BYTES, look & 255, look >> 8 & 255))
            spoilt[look >> 16 & (L::SPOILT - 1)] = (look >> 16) + 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        }
        if (i + AHEAD * PRODUCERS < tiles) read(j);
        i += PRODUCERS;
      }
    }
    if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
    // no copy is in flight when the block ends, however its other warps end
    static_assert(STAGES == PRODUCERS, "a stage is one producer's");
    if (i >= PRODUCERS) mbar_wait_warp(&full[(i - PRODUCERS) % STAGES], ((i - PRODUCERS) / STAGES) & 1, abort_flag);
  } else {
    reg_alloc<L::REGS>();
    // ---- the consumers.  Accumulators of a lane: rows lane / 4 and lane / 4 + 8 of a block, channels 2 * (lane % 4) and the next of eight
    const int quad = lane & 3, ksteps = (p.head_dim + 15) / 16, block = warp % MB, turn = warp / MB;
    const float c = fabsf(p.scale) * 1.4426950408889634f;
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;    // a negative scale goes to the queries, so that the largest product has the largest score
    float *merge = reinterpret_cast<float *>(smem + L::MERGE_OFF);     // [WARPS][16][PITCH]
    float2 *ml = reinterpret_cast<float2 *>(smem + L::ML_OFF);
    const int kid = lane >> 3, krow = lane & 7;
    const uint32_t k_off = ((kid >> 1) * 8 + krow) * 128, v_off = ((kid & 1) * 8 + krow) * 128;
    // the queries of the next piece are on their way while one is worked on: its slot was read in the piece before, which all warps have left
    auto fetch = [&](int piece, int head, int row) {
      if (lane == 0) mbar_arrive_expect_tx(&qfull[piece & 1], CB * g.box * group * 128);
      __syncwarp();
      if (lane < CB) tma_tile_3d(smem + L::Q_OFF + (piece & 1) * L::Q_BYTES + lane * MB * 16 * 128, &g.qmap, lane * 64, head * group, row, &qfull[piece & 1]);
    };
    if (warp == 0) fetch(0, walk.head, walk.q.first);
    int index = 0, pieces = 0;                                  // index: of a piece's first tile among this CTA's
    for (long long at = first; at < end; ++pieces) {
      if (walk.t >= walk.tiles) walk.wrap();
      const int t0 = walk.t, t1 = (int)min((long long)walk.tiles, t0 + (end - at)), rows = walk.q.n * group, length = walk.q.length;
      const long long item = at - t0, item_end = item + walk.tiles;
      at += t1 - t0;
      if (warp == 0 && at < end) {
        if (walk.head + 1 < p.kv_heads) fetch(pieces + 1, walk.head + 1, walk.q.first);
        else fetch(pieces + 1, 0, sequence_of(p.seq, walk.s + 1).first);
      }
      int seen[2];                                              // the first key that a row does not see
#pragma unroll
      for (int half = 0; half < 2; ++half) seen[half] = p.causal ? length - walk.q.n + (block * 16 + half * 8 + (lane >> 2)) / group + 1 : length;
      const int seen_by_all = p.causal ? length - walk.q.n + 1 : length;
      // Q of this key head's rows, in the products' own order
      uint32_t q[CB * 4][4];
      const int slot = pieces & 1;
      if (!mbar_poll_warp(&qfull[slot], (pieces >> 1) & 1, abort_flag)) fail_code = ST_WAIT_TIMEOUT_MMA;
      const uint32_t qb = smem_u32(smem + L::Q_OFF + slot * L::Q_BYTES) + (block * 16 + (kid & 1) * 8 + krow) * 128;
#pragma unroll
      for (int k = 0; k < CB * 4; ++k) {
        ldmatrix4(q[k], qb + (k >> 2) * MB * 16 * 128 + ((((k & 3) * 2 + (kid >> 1)) ^ krow) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) q[k][i] ^= flip;
      }
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
        float keep[2], base[2];
        bool moved = false;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float top = m[half];
#pragma unroll
          for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(sc[n][half * 2], sc[n][half * 2 + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
          base[half] = top == -INFINITY ? 0.0f : top;
          keep[half] = exp2_approx((m[half] - base[half]) * c);
          moved |= top > m[half];
          m[half] = top;
        }
        // (Their distances from the largest, then times c: products of large scores with c are rounded, by more than one from 2^25 on, and past 2^128 none of fp32's numbers.)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i >> 2][i & 3] -= base[(i >> 1) & 1];
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
            const float w0 = exp2_approx(sc[n][half * 2] * c), w1 = exp2_approx(sc[n][half * 2 + 1] * c);
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
        // The next tile's copy, of the other proxy, comes behind the last read of this one.  (Without the fence some of the values' ldmatrix were found behind the arrival: in two
        // calls of 100 of 64 x 1 tokens behind 500 to 16000 a few of a tile's values were those of the tile that comes to the same stage next.)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      index += t1 - t0;
      // ---- The warps' results together.  From here on a row is a warp's, a lane has 2 * CB of its channels.
      float own[2] = {1.0f, 1.0f}, add[2] = {0.0f, 0.0f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 1);
        l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 2);
      }
      float *place = merge + ((MB > 1 ? block : warp) * 16 + (lane >> 2)) * L::PITCH + quad * 2;
      auto leave_rows = [&](bool joining) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = half * 8 + (lane >> 2);
          if (joining) {
            const float2 x = ml[(warp + MB) * 16 + r];
            const float top = fmaxf(m[half], x.x), from = top == -INFINITY ? 0.0f : top;
            own[half] = exp2_approx((m[half] - from) * c);
            add[half] = exp2_approx((x.x - from) * c);
            m[half] = top;
            l[half] = l[half] * own[half] + x.y * add[half];
          }
          if (quad == 0) ml[warp * 16 + r] = make_float2(m[half], l[half]);
          if (block * 16 + r < rows) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              float2 &at = *reinterpret_cast<float2 *>(place + half * 8 * L::PITCH + n * 8);
              float2 v = make_float2(o[n][half * 2] * own[half], o[n][half * 2 + 1] * own[half]);
              if (joining) { v.x += at.x * add[half]; v.y += at.y * add[half]; }
              at = v;
            }
          }
        }
      };
      if (MB == 1 || turn > 0) leave_rows(false);
      named_bar_sync(1, WARPS * 32);
      if (MB > 1) {
        if (turn == 0) leave_rows(true);
        named_bar_sync(1, WARPS * 32);
      }
      // of the values that were cleared those that a row sees, to one of its results, by the lanes that will join these
      if (spoilt[pieces & (L::SPOILT - 1)] == (pieces & L::PIECE_BITS) + 1) {
#pragma unroll 1
        for (int r = warp; r < rows; r += WARPS) {
          const int end = min(length, length - walk.q.n + r / group + 1);
#pragma unroll 1
          for (int j = max(seen_by_all, 0); j < end; ++j) {
            const long long at = place_of_key(p, walk.s, j);
            const T *v = static_cast<const T *>(p.v) + at + walk.head * p.ld_head;
            for (int ch = lane * 2 * CB; ch < (at < 0 ? 0 : min((lane + 1) * 2 * CB, p.head_dim)); ++ch)
              if (!isfinite(to_f32(v[ch]))) merge[r * L::PITCH + ch] += to_f32(v[ch]);
          }
        }
      }
      const int c0 = deal.owner(item), c1 = deal.owner(item_end - 1), sharers = c1 - c0 + 1;
      constexpr int PER = 2 * CB, WIDE = CB * 64, GROUP = 32;
      struct Row { float v[PER], top, l; };
      auto part = [&](int cta) { return g.w.partial + (cta * 2 + (cta == c0 ? 1 : 0)) * L::PARTIAL; };     // (its last piece, or its first)
      auto base_of = [](float top) { return top == -INFINITY ? 0.0f : top; };
      // a row of all of the warps that had its block
      auto row_here = [&](int r) {
        Row x;
        float2 y[L::COPIES];
        x.top = -INFINITY;
        x.l = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) x.v[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < L::COPIES; ++w) { y[w] = ml[w * 16 + r]; x.top = fmaxf(x.top, y[w].x); }
#pragma unroll
        for (int w = 0; w < L::COPIES; ++w) {
          const float k = exp2_approx((y[w].x - base_of(x.top)) * c);
          const float *src = merge + (w * 16 + r) * L::PITCH + lane * PER;
          x.l += y[w].y * k;
#pragma unroll
          for (int i = 0; i < PER; ++i) x.v[i] += src[i] * k;
        }
        return x;
      };
      // Rows of n CTAs' results, in their order.  R rows of a warp at once, WARPS apart (where there are as many, otherwise the first again): each is little work
      // behind two round trips to L2.
      auto nth = [&](int r, int a) { return r + a * WARPS < rows ? r + a * WARPS : r; };
      auto rows_of = [&](auto &x, int r, auto cta_of, int n) {
        constexpr int R = sizeof(x) / sizeof(Row);
#pragma unroll
        for (int a = 0; a < R; ++a) {
          x[a].top = -INFINITY;
          x[a].l = 0.0f;
#pragma unroll
          for (int i = 0; i < PER; ++i) x[a].v[i] = 0.0f;
        }
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += 32) {                    // a lane looks at one maximum and sum
          const int here = min(32, n - k0);
          float2 y[R];
          float weight[R];
#pragma unroll
          for (int a = 0; a < R; ++a)
            y[a] = lane < here ? __ldcg(reinterpret_cast<const float2 *>(part(cta_of(k0 + lane)) + MB * 16 * WIDE) + nth(r, a)) : make_float2(-INFINITY, 0.0f);
#pragma unroll
          for (int a = 0; a < R; ++a) {
            float top = fmaxf(x[a].top, y[a].x);
#pragma unroll
            for (int b = 16; b > 0; b >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, b));
            const float keep = exp2_approx((x[a].top - base_of(top)) * c);
            weight[a] = exp2_approx((y[a].x - base_of(top)) * c);
            float sum = y[a].y * weight[a];
#pragma unroll
            for (int b = 16; b > 0; b >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, b);
            x[a].top = top;
            x[a].l = x[a].l * keep + sum;
#pragma unroll
            for (int i = 0; i < PER; ++i) x[a].v[i] *= keep;
          }
          constexpr int BATCH = 16 / R;                         // results on their way at once, of each row
#pragma unroll 1
          for (int k = 0; k < here; k += BATCH) {
            float z[R][BATCH][PER];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
#pragma unroll
              for (int a = 0; a < R; ++a) {
                const float *src = part(cta_of(k0 + min(k + j, here - 1))) + nth(r, a) * WIDE + lane * PER;
                if constexpr (CB == 2) *reinterpret_cast<float4 *>(z[a][j]) = __ldcg(reinterpret_cast<const float4 *>(src));
                else *reinterpret_cast<float2 *>(z[a][j]) = __ldcg(reinterpret_cast<const float2 *>(src));
              }
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
#pragma unroll
              for (int a = 0; a < R; ++a) {
                const float w = k + j < here ? __shfl_sync(0xFFFFFFFFu, weight[a], k + j) : 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i) x[a].v[i] += k + j < here ? z[a][j][i] * w : 0.0f;
              }
          }
        }
      };
      auto leave = [&](int cta, int r, const Row &x) {
        float *dst = part(cta);
        if constexpr (CB == 2) *reinterpret_cast<float4 *>(dst + r * WIDE + lane * PER) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        else *reinterpret_cast<float2 *>(dst + r * WIDE + lane * PER) = make_float2(x.v[0], x.v[1]);
        if (lane == 0) reinterpret_cast<float2 *>(dst + MB * 16 * WIDE)[r] = make_float2(x.top, x.l);
      };
      // whether this CTA is the last of n that have left their rows; the others' can then be read
      auto last_of = [&](int *arrived, int n) {
        named_bar_sync(1, WARPS * 32);
        // (released and acquired by one thread for the block, whose other threads are ordered by the barriers)
        if (threadIdx.x == 0) {
          int before;
          asm volatile("atom.acq_rel.gpu.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(arrived) : "memory");
          if (before == n - 1) *arrived = 0;
          *verdict = before == n - 1;
        }
        named_bar_sync(1, WARPS * 32);
        return *verdict != 0;
      };
      auto write = [&](int r, const Row &x) {
        const float inv = x.l == 0.0f ? 0.0f : 1.0f / x.l;
        const int token = r / group, ch = lane * PER;
        T *out = static_cast<T *>(p.out) + (long long)(walk.q.first + token) * p.ld_out + (long long)(walk.head * group + r - token * group) * p.head_dim + ch;
        if (ch >= p.head_dim) return;
        if constexpr (CB == 2) *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<T>(x.v[0] * inv, x.v[1] * inv), pack2<T>(x.v[2] * inv, x.v[3] * inv));
        else *reinterpret_cast<uint32_t *>(out) = pack2<T>(x.v[0] * inv, x.v[1] * inv);
      };
      // Piece of a whole item: out; otherwise to the workspace, where the last one there joins all of them.  Where more than two groups of CTAs share an
      // item, the last of each group joins that first, and the last of these the groups.
      auto finish = [&](auto of_warp) {
        constexpr int R = decltype(of_warp)::value;
        Row x[R];
#pragma unroll 1
        for (int r = warp; r < rows; r += R * WARPS) {
#pragma unroll
          for (int a = 0; a < R; ++a) x[a] = row_here(nth(r, a));
#pragma unroll
          for (int a = 0; a < R; ++a) leave(blockIdx.x, nth(r, a), x[a]);
        }
        int *arrived = g.w.arrived + c0, n = sharers, stride = 1, at = c0;
        if (sharers > 2 * GROUP) {
          const int begin = c0 + ((int)blockIdx.x - c0) / GROUP * GROUP, final = min(begin + GROUP - 1, c1);
          if (!last_of(g.w.arrived + gridDim.x + final, final - begin + 1)) return;
#pragma unroll 1
          for (int r = warp; r < rows; r += R * WARPS) {
            rows_of(x, r, [&](int k) { return begin + k; }, final - begin + 1);
#pragma unroll
            for (int a = 0; a < R; ++a) leave(final, nth(r, a), x[a]);
          }
          n = (sharers + GROUP - 1) / GROUP;
          stride = GROUP;
          at = c0 + GROUP - 1;
        }
        if (!last_of(arrived, n)) return;
#pragma unroll 1
        for (int r = warp; r < rows; r += R * WARPS) {
          rows_of(x, r, [&](int k) { return min(at + k * stride, c1); }, n);
#pragma unroll
          for (int a = 0; a < R; ++a)
            if (r + a * WARPS < rows) write(r + a * WARPS, x[a]);
        }
      };
      if (sharers == 1) {
#pragma unroll 1
        for (int r = warp; r < rows; r += WARPS) write(r, row_here(r));
      } else if (rows <= WARPS) {
        finish(std::integral_constant<int, 1>());
      } else {
        finish(std::integral_constant<int, 4>());
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

// Up to 16 rows to a key head a warp's matrix instruction is as long whatever they are; with up to 32 two warps share a tile of keys.  (32 heads of 128 over 8, us
// here / with the prompts' kernel: 1 x 1 token behind 4000 15/33, 64 x 1 175/219, 8 x 4 36/42, 8 x 8 43/42, 24 x 8 84/113, 64 x 8 196/221, 8 x 5 of 40 heads behind 1000 to
// 7000 46/62; behind 1000, where that starts and joins sooner, 8 x 8 25/19, 64 x 8 69/78.)
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
