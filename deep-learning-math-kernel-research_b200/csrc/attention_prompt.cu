// Attention of prompts on tensor cores.
//
// An item is one key head and two tiles of 128 rows: a tile's rows are the g heads that share the key head, of 128 / g tokens, so that K and V are brought in
// once for all of them.  Keys come in tiles of 128.  With S = Q K^T in tensor memory, a warpgroup per row tile holds a row per thread: its maximum m and
// sum l of e^(s - m); the terms go back to tensor memory as P, 16 bits, over the scores, and O += P V.  One thread issues all products in the order
// O0 S0' O1 S1', so that one tile's products run while the other's softmax does.  With 128 channels a tile's products take the tensor cores 512 cycles each,
// its 16384 exponentials the SM's 16 special-function lanes 1024, and the way round of scores, softmax and results about 3400 a tile: 8192 tokens of 32 heads
// over 8, causal, 448 us, 1230 TFLOP/s.
//
// A CTA per SM goes over the items, each the next that nobody has taken, those of the longest sequences first; one warp does nothing but find them (3 to 8 k cycles
// between items when every role did it).  The next one's queries, keys and scores are on their way while the last one's results are written, exchanged among
// four lanes first, since a row per thread makes 32 lines of each store.  Where there are fewer items than half of the SMs, their keys are split, and the last CTA
// of those that share a tile joins the results in the order of the keys.
//
// The maximum that the terms are relative to may stay 8 powers of two behind: P then reaches 256, O and l are in 32 bits, and scaling O again, a round trip
// through registers, is left out for nearly every tile.  When the scores of a tile are there, so is O's last product: both are the same thread's, in order.
//
// Measured and not taken (the same prompt): two warpgroups a row tile 468 us; an issuer for each row tile 589; P handed over in quarters 520, whole 462; 1 to 4 of 8
// exponentials from a polynomial on the multiply-add pipe 453 to 500.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"
#include "umma.cuh"

namespace elb {

namespace {

constexpr int TILE = 128, THREADS = 384;                        // four warps: copies, products; two warpgroups of rows
constexpr int BOX_BYTES = TILE * 128;                           // 128 rows of 64 channels
constexpr int REGS_ROWS = 216, REGS_OTHERS = 72;                // (2 * 216 + 72) * 128 = 168 * 384
constexpr float SLACK = 8.0f;                                   // powers of two

template <int CB>
struct Smem {
  static constexpr int Q_BYTES = CB * BOX_BYTES, STAGE = CB * BOX_BYTES;
  static constexpr int STAGES = CB == 1 ? 8 : 5;                // of K or V
  static constexpr int RING_OFF = 2 * Q_BYTES;
  static constexpr int BAR_OFF = RING_OFF + STAGES * STAGE;     // full[S], empty[S], qfull[2], qempty[2], sfull[2], phalf[2], pfull[2], ofull[2], oempty[2], ifull[2], iempty[2]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 18) * 8;
  static constexpr int ITEMS_OFF = (MISC_OFF + 16 + 63) / 64 * 64;             // (misc: tmem slot, abort flag, verdicts)
  static constexpr int TOTAL = ITEMS_OFF + 2 * 64 + 1024;       // (room to align)
};

struct alignas(64) PromptLaunch {
  CUtensorMap kmap, vmap, qmap;
  AttentionParams p;
  AttentionWorkspace w;
  int tokens;                       // of a row tile
  int splits;                       // CTAs that share an item's keys; above 1: no CTA has two items
};

// Two 32-bit values side by side, which the fused multiply-add takes together
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A matrix descriptor whose low word, the address and the distance along M or N, is worked out in 32 bits
__device__ __forceinline__ uint64_t with_low(uint64_t desc, uint32_t low) { return (desc & 0xFFFFFFFF00000000ull) | low; }

// An item, and of its tiles of keys those that this CTA has: [t0, t1), of which row tile i sees those below end[i].  place: of its partial result in the
// workspace, where those of an item that is split begin at `places`.  s: -1 behind the last item
struct alignas(64) Item {
  int s, head, first, n, length, row0, t0, t1, end[2], place, places;
};

// The items of a call in order, by one warp: sequences (up to 32 of them the longest first), their blocks of two row tiles from the last, which sees the most keys,
// their key heads, their splits.
struct Finder {
  const PromptLaunch &g;
  const KeyTiles<TILE> kt;
  const int lane, per_block;
  int total;                        // items
  int own, upto;                    // sequence of this lane (of the first of several); blocks of the call up to the end of this lane's sequences
  __device__ __forceinline__ int blocks_of(int s) const { return (sequence_of(g.p.seq, s).n + per_block - 1) / per_block; }
  __device__ __forceinline__ Finder(const PromptLaunch &g) : g(g), kt(g.p.page_size), lane(threadIdx.x & 31), per_block(2 * g.tokens) {
    const int seqs = (int)g.p.seq.seqs, per = (seqs + 31) / 32;
    own = lane * per;
    int blocks = 0;
    if (per == 1) {
      int length = lane < seqs ? sequence_of(g.p.seq, lane).length : -1, rank = 0;
      for (int j = 0; j < seqs; ++j) {
        const int other = __shfl_sync(0xFFFFFFFFu, length, j);
        rank += other > length || (other == length && j < lane);
      }
      for (int j = 0; j < seqs; ++j) {
        const int at = __shfl_sync(0xFFFFFFFFu, rank, j);
        if (at == lane) own = j;
      }
      if (lane < seqs) blocks = blocks_of(own);
    } else {
      for (int s = own; s < min(own + per, seqs); ++s) blocks += blocks_of(s);
    }
    upto = blocks;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, upto, k);
      if (lane >= k) upto += v;
    }
    total = __shfl_sync(0xFFFFFFFFu, upto, 31) * g.p.kv_heads * g.splits;
  }
  __device__ __forceinline__ void find(int at, Item &it) const {
    const AttentionParams &p = g.p;
    const int item = at / g.splits, split = at - item * g.splits, block_at = item / p.kv_heads;
    it.head = item - block_at * p.kv_heads;
    it.places = item * g.splits;
    it.place = at;
    const int mine = __ffs(__ballot_sync(0xFFFFFFFFu, block_at < upto)) - 1;
    int s = __shfl_sync(0xFFFFFFFFu, own, mine), before = mine > 0 ? __shfl_sync(0xFFFFFFFFu, upto, mine > 0 ? mine - 1 : 0) : 0;
    int blocks = blocks_of(s);
    while (block_at >= before + blocks) { before += blocks; blocks = blocks_of(++s); }        // (several sequences a lane)
    const Sequence q = sequence_of(p.seq, s);
    it.s = s;
    it.first = q.first;
    it.n = q.n;
    it.length = q.length;
    it.row0 = (blocks - 1 - (block_at - before)) * per_block;
    int seen[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = it.row0 + i * g.tokens, last = min(from + g.tokens, q.n) - 1;
      seen[i] = from >= q.n ? 0 : kt.count(max(0, p.causal ? min(q.length, q.length - q.n + last + 1) : q.length));
    }
    const long long most = max(seen[0], seen[1]);
    it.t0 = (int)quotient(most * split, g.splits);
    it.t1 = (int)quotient(most * (split + 1), g.splits);
#pragma unroll
    for (int i = 0; i < 2; ++i) it.end[i] = max(it.t0, min(it.t1, seen[i]));
  }
};

template <typename T, int CB>
__global__ void __launch_bounds__(THREADS, 1) attention_prompt_kernel(const __grid_constant__ PromptLaunch g) {
  using L = Smem<CB>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t S_COL = 0, O_COL = 256, COLS = 512;        // scores 2 x 128 columns, P in their first 64; results 2 x 64 CB
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *qfull = empty + STAGES, *qempty = qfull + 2, *sfull = qempty + 2,
           *phalf = sfull + 2, *pfull = phalf + 2, *ofull = pfull + 2, *oempty = ofull + 2, *ifull = oempty + 2, *iempty = ifull + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::MISC_OFF);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 4);
  volatile int *verdict = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 8);
  Item *slots = reinterpret_cast<Item *>(smem + L::ITEMS_OFF);
  const AttentionParams &p = g.p;
  // (from lane 0: what is known to be the same in all lanes goes to the tensor cores without a move each)
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    tma_prefetch_desc(&g.qmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&qfull[i], 1);
      mbar_init(&qempty[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&phalf[i], 4);
      mbar_init(&pfull[i], 4);
      mbar_init(&ofull[i], 1);
      mbar_init(&oempty[i], 4);
      mbar_init(&ifull[i], 1);
      mbar_init(&iempty[i], 10);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  const KeyTiles<TILE> kt(p.page_size);
  if (kt.rows < TILE) {                                         // rows of a tile that no copy fills: zeros, as values that nothing is multiplied with
    for (int i = threadIdx.x; i < STAGES * L::STAGE / 16; i += THREADS) reinterpret_cast<uint4 *>(smem + L::RING_OFF)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  griddep_wait();
  if (warp == 1) tmem_alloc(tmem_slot, COLS);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  griddep_launch_dependents();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
  int fail_code = 0;
  // the next item of a role, which the finding warp has put down; false: there is none
  auto done_item = [&](uint32_t &count) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&iempty[count & 1]);
    ++count;
  };
  auto next_item = [&](uint32_t &count, Item &it) {
    if (!mbar_wait_uniform(&ifull[count & 1], (count >> 1) & 1, abort_flag)) return false;
    it = slots[count & 1];
    done_item(count);
    return it.s >= 0;
  };

  if (warp < 4) {
    reg_dealloc<REGS_OTHERS>();
    if (warp == 0) {
      // ---- copies: queries, then K and V of each tile, a lane per copy, [64 channels][page of the tile]
      const int boxes = kt.pages ? kt.pages : 1, cb = lane / boxes, page_in_tile = lane - cb * boxes;
      const bool mine = lane < CB * boxes;
      const uint32_t bytes = CB * boxes * kt.box() * 128;
      uint8_t *dst = smem + L::RING_OFF + cb * BOX_BYTES + page_in_tile * kt.page * 128;
      int issued = 0, stage = 0, queries[2] = {0, 0};
      uint32_t phase = 1;
      bool ok = true;
      uint32_t count = 0;
      for (Item it; ok && next_item(count, it);) {
        if (it.t1 == it.t0) continue;
        // (the queries' place is free when the item in front has had its last scores: until then they come as far as L2)
        if (lane < 2 * CB && it.end[lane / CB] > it.t0) tma_prefetch_3d(&g.qmap, lane % CB * 64, it.head * group, it.first + it.row0 + lane / CB * g.tokens);
        int next_page = 0, next_token = 0;
        auto read = [&](int t) {
          next_page = (int)p.seq.pages;                         // one outside the map: zeros
          next_token = 0;
          if (!kt.page) {
            next_page = it.s;
            next_token = t * TILE;
          } else if (mine) {
            int i = t * kt.pages + page_in_tile;
            if (!kt.pages) {
              i = t / kt.parts;
              next_token = (t - i * kt.parts) * TILE;
            }
            if ((long long)i * kt.page < it.length) next_page = p.seq.table[it.s * p.seq.width + i];
            else next_token = -1;                               // behind the sequence's end
          }
        };
        read(it.t0);
        for (int t = it.t0; t < it.t1 && ok; ++t) {
          int page = next_page;
          const int token = max(next_token, 0);
          if ((unsigned)page >= (unsigned)p.seq.pages && kt.page) {
            if (mine && next_token >= 0) report_status(p.status, ST_BAD_PAGE);
            page = (int)p.seq.pages;
          }
          if (t + 1 < it.t1) read(t + 1);
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            if (!mbar_wait_uniform(&empty[stage], phase, abort_flag)) { ok = false; break; }
            if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
            __syncwarp();
            if (mine) tma_tile_4d(dst + stage * L::STAGE, v ? &g.vmap : &g.kmap, cb * 64, token, it.head, page, &full[stage]);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
            ++issued;
            if (t > it.t0 || v > 0) continue;
            // (behind the first keys: a tile's place is free when the item in front has had its last scores)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (it.end[i] == it.t0 || !ok) continue;
              if (!mbar_wait_uniform(&qempty[i], (queries[i] & 1) ^ 1, abort_flag)) { ok = false; continue; }
              if (lane == 0) mbar_arrive_expect_tx(&qfull[i], CB * group * g.tokens * 128);
              __syncwarp();
              if (lane < CB) tma_tile_3d(smem + i * L::Q_BYTES + lane * BOX_BYTES, &g.qmap, lane * 64, it.head * group, it.first + it.row0 + i * g.tokens, &qfull[i]);
              ++queries[i];
            }
          }
        }
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
      // no copy is in flight when the block ends, however its other warps end
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1, abort_flag);
      for (int i = 0; i < 2; ++i)
        if (queries[i] > 0) mbar_wait_warp(&qfull[i], (queries[i] - 1) & 1, abort_flag);
    } else if (warp == 1) {
      // ---- products.  Issued by a converged warp, addresses in 32 bits, the next tile's K and V waited for behind this one's products: what the warp waits and works
      // out between two products the tensor cores wait for.
      const uint32_t el = elect_one();
      const int ksteps = (p.head_dim + 15) / 16, bf = p.et == ET_BF16;
      const uint32_t s_idesc = umma_idesc(1, bf, bf, TILE, TILE) | (p.scale < 0.0f ? UMMA_NEGATE_A : 0u);
      const uint32_t o_idesc = umma_idesc(1, bf, bf, TILE, ksteps * 16) | UMMA_B_ROWS_ARE_K;
      const uint32_t ring = smem_u32(smem) + L::RING_OFF;
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem)), k_desc = umma_desc_sw128(ring), v_desc = umma_desc_sw128_rows_k(ring, BOX_BYTES);
      const uint32_t q_low = (uint32_t)q_desc, k_low = (uint32_t)k_desc, v_low = (uint32_t)v_desc;
      int stage = 0;                                            // the next of the ring to be looked at
      uint32_t phase = 0, items[2] = {0, 0}, terms[2] = {0, 0};
      bool ok = true;
      auto next_full = [&]() {
        ok = ok && mbar_wait_uniform(&full[stage], phase, abort_flag);
        const int here = stage;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        return here;
      };
      auto scores = [&](int i, int from, bool last) {
        const uint32_t ql = q_low + i * (L::Q_BYTES >> 4), kl = k_low + from * (L::STAGE >> 4);
#pragma unroll
        for (int k = 0; k < CB * 4; ++k) {
          const uint32_t at = (k >> 2) * (BOX_BYTES >> 4) + (k & 3) * 2;
          if (k < ksteps) umma_f16_el(tmem + S_COL + i * TILE, with_low(q_desc, ql + at), with_low(k_desc, kl + at), s_idesc, k != 0, el);
        }
        umma_commit_el(&sfull[i], el);
        if (last) umma_commit_el(&qempty[i], el);
      };
      uint32_t count = 0;
      for (Item it; ok && next_item(count, it);) {
        it.t0 = __shfl_sync(0xFFFFFFFFu, it.t0, 0);
        it.t1 = __shfl_sync(0xFFFFFFFFu, it.t1, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) it.end[i] = __shfl_sync(0xFFFFFFFFu, it.end[i], 0);
        if (it.t1 == it.t0) continue;
        // the tile in which the sequence ends: values behind its end may be anything, and 0 times anything is not always 0
        const int last = kt.count(it.length) - 1, held = kt.held(last, it.length);
        auto next_values = [&](int t) {
          const int at = next_full();
          if (t == last && held < TILE && ok) {
            uint8_t *rows = smem + L::RING_OFF + at * L::STAGE;
            for (int j = held * 8 + lane; j < TILE * 8; j += 32)
#pragma unroll
              for (int c = 0; c < CB; ++c) reinterpret_cast<uint4 *>(rows + c * BOX_BYTES)[j] = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
          return at;
        };
        int keys_at = next_full();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (it.end[i] == it.t0) continue;
          ok = ok && mbar_wait_uniform(&qfull[i], items[i] & 1, abort_flag);
          if (!ok) break;
          tc_fence_after_sync();
          scores(i, keys_at, it.t0 + 1 == it.end[i]);
        }
        if (!ok) break;
        umma_commit_el(&empty[keys_at], el);
        int values_at = next_values(it.t0);
        if (it.t0 + 1 < it.t1) keys_at = next_full();
        for (int t = it.t0; t < it.t1 && ok; ++t) {
          const uint32_t vl = v_low + values_at * (L::STAGE >> 4);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (t >= it.end[i]) continue;
            // (the item in front has had its results read)
            if (t == it.t0) ok = ok && mbar_wait_uniform(&oempty[i], (items[i] & 1) ^ 1, abort_flag);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && mbar_wait_uniform(half ? &pfull[i] : &phalf[i], terms[i] & 1, abort_flag);
              if (!ok) break;
              tc_fence_after_sync();
#pragma unroll
              for (int k = half * 4; k < half * 4 + 4; ++k)
                umma_f16_ts_el(tmem + O_COL + i * CB * 64, tmem + S_COL + i * TILE + k * 8, with_low(v_desc, vl + k * 128), o_idesc, k > 0 || t > it.t0, el);
            }
            if (!ok) break;
            ++terms[i];
            if (t + 1 < it.end[i]) {
              scores(i, keys_at, t + 2 == it.end[i]);
            } else {
              umma_commit_el(&ofull[i], el);
              ++items[i];
            }
          }
          if (!ok) break;
          umma_commit_el(&empty[values_at], el);
          if (t + 1 < it.t1) {
            umma_commit_el(&empty[keys_at], el);
            values_at = next_values(t + 1);
            if (t + 2 < it.t1) keys_at = next_full();
          }
        }
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_MMA;
    } else if (warp == 2) {
      // ---- items: the CTA's own first one, then the next that nobody has taken.  Every CTA counts once past the last, so the counter sees as many
      // counts as there are items, and the last of them leaves it at zero.
      const Finder finder(g);
      const int ctas = gridDim.x;
      uint32_t count = 0;
      bool ok = true;
      for (int at = blockIdx.x;;) {
        Item it;
        if (at < finder.total) finder.find(at, it);
        else it.s = -1;
        if (ok) {                                               // (on, where the others have given up: the counter has to come to its end)
          ok = mbar_wait_uniform(&iempty[count & 1], ((count >> 1) & 1) ^ 1, abort_flag);
          if (ok && lane == 0) {
            slots[count & 1] = it;
            mbar_arrive(&ifull[count & 1]);
          }
          ++count;
        }
        if (at >= finder.total) break;
        at = finder.total;
        if (finder.total > ctas) {
          int taken = 0;
          if (lane == 0) {
            taken = atomicAdd(g.w.next, 1);
            if (taken == finder.total - 1) *g.w.next = 0;
          }
          at = ctas + __shfl_sync(0xFFFFFFFFu, taken, 0);
        }
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
    }
  } else {
    // ---- rows
    reg_alloc<REGS_ROWS>();
    const int i = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, in_tile = r / group;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, s_at = tmem + lanes + S_COL + i * TILE, o_at = tmem + lanes + O_COL + i * CB * 64;
    const float c = fabsf(p.scale) * 1.4426950408889634f, slack = SLACK / c;
    uint32_t items = 0, terms = 0, count = 0;
    // (an item is read again where its results are written, which keeps it out of the registers of the loop)
    for (; mbar_wait_uniform(&ifull[count & 1], (count >> 1) & 1, abort_flag) && slots[count & 1].s >= 0; done_item(count)) {
      volatile Item &it = slots[count & 1];
      const int length = it.length, t0 = it.t0, end = it.end[i], tiles = end - t0;
      if (it.row0 + i * g.tokens >= it.n) continue;             // no rows in this tile
      const int seen = p.causal ? min(length, length - it.n + it.row0 + i * g.tokens + in_tile + 1) : length;
      float m = -INFINITY, l = 0.0f;
      for (int t = t0; t < end; ++t, ++terms) {
        if (!mbar_wait_uniform(&sfull[i], terms & 1, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_EPILOGUE; break; }
        tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s_at + q * 32, s[q]);
        const int limit = min(kt.held(t, length), seen - kt.first(t));
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_arrived32(s[q]);
        if (!__all_sync(0xFFFFFFFFu, limit >= TILE)) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (q * 32 + k >= limit) s[q][k] = 0xFF800000u;   // -inf
        }
        float top4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top4[q] = __uint_as_float(s[q][0]);
#pragma unroll
          for (int k = 1; k < 32; ++k) top4[q] = fmaxf(top4[q], __uint_as_float(s[q][k]));
        }
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        if (__any_sync(0xFFFFFFFFu, top > m + slack)) {
          const float to = top > m + slack ? top : m, scale = m == -INFINITY ? 0.0f : exp2_approx((m - to) * c);
          if (t > t0) {
#pragma unroll 1
            for (int q = 0; q < 2 * CB; ++q) {
              uint32_t o[32];
              tmem_ld32(o_at + q * 32, o);
              tmem_ld_wait();
              tmem_arrived32(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * scale);
              tmem_st32(o_at + q * 32, o);
            }
          }
          l *= scale;
          m = to;
        }
        const float from = m == -INFINITY ? 0.0f : m * c;
        const uint64_t c2 = pair(c, c), from2 = pair(-from, -from);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const uint64_t z = fma2(pair(__uint_as_float(s[q][2 * k]), __uint_as_float(s[q][2 * k + 1])), c2, from2);
            float a, b;
            unpair(z, a, b);
            a = exp2_approx(a);
            b = exp2_approx(b);
            sum[k & 1] = add2(sum[k & 1], pair(a, b));
            w[k] = pack2<T>(a, b);                              // the second product's operand has 16 bits
          }
          tmem_st16(s_at + q * 16, w);
          if (q & 1) {                                          // half of the keys can be multiplied with their values
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q == 1 ? &phalf[i] : &pfull[i]);
          }
        }
        float l4[4];
        unpair(sum[0], l4[0], l4[1]);
        unpair(sum[1], l4[2], l4[3]);
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      }
      if (tiles > 0 && !mbar_wait_uniform(&ofull[i], items & 1, abort_flag)) fail_code = ST_WAIT_TIMEOUT_EPILOGUE;
      tc_fence_after_sync();
      const int token = it.row0 + i * g.tokens + in_tile;
      const bool mine = in_tile < g.tokens && token < it.n;
      T *out = static_cast<T *>(p.out) + (long long)(it.first + token) * p.ld_out + (long long)(it.head * group + r - in_tile * group) * p.head_dim;
      const uint32_t rows_here = __ballot_sync(0xFFFFFFFFu, mine);
      // 32 channels of a row are four words of 16 bytes; four lanes exchange theirs, so that a store has 64 bytes of each of eight rows
      auto write = [&](const float (&v)[32], int q, float inv) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = make_uint4(pack2<T>(v[k * 8] * inv, v[k * 8 + 1] * inv), pack2<T>(v[k * 8 + 2] * inv, v[k * 8 + 3] * inv),
                            pack2<T>(v[k * 8 + 4] * inv, v[k * 8 + 5] * inv), pack2<T>(v[k * 8 + 6] * inv, v[k * 8 + 7] * inv));
        auto trade = [&](uint4 &a, uint4 &b, int with) {        // the lane whose bit is clear gives b and takes the other's a in its place
          const bool upper = (lane & with) != 0;
          uint4 x = upper ? a : b;
          x.x = __shfl_xor_sync(0xFFFFFFFFu, x.x, with);
          x.y = __shfl_xor_sync(0xFFFFFFFFu, x.y, with);
          x.z = __shfl_xor_sync(0xFFFFFFFFu, x.z, with);
          x.w = __shfl_xor_sync(0xFFFFFFFFu, x.w, with);
          if (upper) a = x;
          else b = x;
        };
        trade(w[0], w[1], 1);
        trade(w[2], w[3], 1);
        trade(w[0], w[2], 2);
        trade(w[1], w[3], 2);
        const int ch = q * 32 + (lane & 3) * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int y = (lane & ~3) + k;
          T *to = reinterpret_cast<T *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(out), y));
          if (((rows_here >> y) & 1) && ch < p.head_dim) *reinterpret_cast<uint4 *>(to + ch) = w[k];
        }
      };
      // a partial result: [4 channels][row], then the rows' maxima and sums
      constexpr int WIDE = CB * 64;
      auto part = [&](int place) { return g.w.partial + ((size_t)place * 2 + i) * (TILE * (WIDE + 2)); };
      float *mine_part = part(it.place);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int q = 0; q < 2 * CB; ++q) {
        uint32_t o[32];
        if (tiles > 0) {
          tmem_ld32(o_at + q * 32, o);
          tmem_ld_wait();
          tmem_arrived32(o);
        }
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = tiles > 0 ? __uint_as_float(o[k]) : 0.0f;
        if (g.splits == 1) {
          write(v, q, inv);
        } else if (mine) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            reinterpret_cast<float4 *>(mine_part)[(q * 8 + k) * TILE + r] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
      }
      if (tiles > 0) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&oempty[i]);
        ++items;
      }
      if (g.splits > 1) {
        if (mine) reinterpret_cast<float2 *>(mine_part + TILE * WIDE)[r] = make_float2(m * c, l);
        named_bar_sync(1 + i, 128);
        // (released and acquired by one thread for the row tile's four warps, which the barriers order)
        if (r == 0) {
          int before, *arrived = g.w.arrived + it.places * 2 + i;
          asm volatile("atom.acq_rel.gpu.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(arrived) : "memory");
          if (before == g.splits - 1) *arrived = 0;
          verdict[i] = before == g.splits - 1;
        }
        named_bar_sync(1 + i, 128);
        if (verdict[i] != 0) {                                  // (rows that are not there read what others left and write nothing)
          const int places = it.places;
          float top = -INFINITY, whole = 0.0f;
          for (int k = 0; k < g.splits; ++k) top = fmaxf(top, __ldcg(reinterpret_cast<const float2 *>(part(places + k) + TILE * WIDE) + r).x);
          const float from = top == -INFINITY ? 0.0f : top;
          for (int k = 0; k < g.splits; ++k) {
            const float2 x = __ldcg(reinterpret_cast<const float2 *>(part(places + k) + TILE * WIDE) + r);
            whole += x.y * exp2_approx(x.x - from);
          }
          const float inv = whole == 0.0f ? 0.0f : 1.0f / whole;
#pragma unroll 1
          for (int q = 0; q < 2 * CB; ++q) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = 0.0f;
#pragma unroll 2
            for (int k = 0; k < g.splits; ++k) {
              const float w = exp2_approx(__ldcg(reinterpret_cast<const float2 *>(part(places + k) + TILE * WIDE) + r).x - from);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(part(places + k)) + (q * 8 + j) * TILE + r);
                v[4 * j] += x.x * w; v[4 * j + 1] += x.y * w; v[4 * j + 2] += x.z * w; v[4 * j + 3] += x.w * w;
              }
            }
            write(v, q, inv);
          }
        }
      }
    }
  }
  if (fail_code != 0 && lane == 0) report_status(p.status, fail_code);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, COLS);
}

template <typename T, int CB>
cudaError_t go(const PromptLaunch &g, long long items, cudaStream_t s) {
  static_assert(2 * TILE * (CB * 64 + 2) <= PROMPT_PARTIAL, "");
  return launch_overlapped(attention_prompt_kernel<T, CB>, dim3((unsigned)(items < g.p.num_sms ? items : g.p.num_sms)), dim3(THREADS), Smem<CB>::TOTAL, s, g);
}
template <typename T>
cudaError_t go(const PromptLaunch &g, long long items, cudaStream_t s) { return g.p.head_dim <= 64 ? go<T, 1>(g, items, s) : go<T, 2>(g, items, s); }
template <typename K>
cudaError_t allow(K kern, int smem) { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }

// Items before splitting; of ragged sequences the most that there can be
long long items_of(const AttentionParams &p) {
  const long long block = 2 * (TILE / (p.heads / p.kv_heads)), blocks = p.seq.starts ? p.seq.rows / block + p.seq.seqs : p.seq.seqs * ((p.seq.each + block - 1) / block);
  return blocks * p.kv_heads;
}

}  // namespace

cudaError_t init_attention_prompt() {
  cudaError_t e = allow(attention_prompt_kernel<__nv_bfloat16, 1>, Smem<1>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_prompt_kernel<__nv_bfloat16, 2>, Smem<2>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_prompt_kernel<__half, 1>, Smem<1>::TOTAL);
  if (e == cudaSuccess) e = allow(attention_prompt_kernel<__half, 2>, Smem<2>::TOTAL);
  return e;
}

bool attention_prompt_takes(const AttentionParams &p) {
  const int group = p.heads / p.kv_heads;
  return p.words && p.head_dim <= 128 && group <= TILE && p.page_size % 8 == 0 && p.seq.width > 0 && p.seq.pages > 0 && items_of(p) <= INT32_MAX;
}

// Keys are split where that fills the SMs, into no fewer than three tiles each of what the sequences can hold.
cudaError_t launch_attention_prompt(const AttentionParams &p, const AttentionWorkspace &w, cudaStream_t s) {
  PromptLaunch g;
  const int rows = KeyTiles<TILE>(p.page_size).box(), group = p.heads / p.kv_heads;
  g.p = p;
  g.tokens = TILE / group;
  g.w = w;
  const long long items = items_of(p), fit = p.num_sms / items, worth = p.seq.capacity / (3 * TILE);
  g.splits = (int)(fit < worth ? fit : worth);
  if (g.splits < 1) g.splits = 1;
  if (!encode_keys(&g.kmap, p, p.k, rows) || !encode_keys(&g.vmap, p, p.v, rows) || !encode_queries(&g.qmap, p, group, g.tokens)) return cudaErrorInvalidValue;
  return p.et == ET_BF16 ? go<__nv_bfloat16>(g, items * g.splits, s) : go<__half>(g, items * g.splits, s);
}

}  // namespace elb
