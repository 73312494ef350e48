// Attention of prompts on tensor cores.
//
// A CTA takes one key head and two tiles of 128 rows: a tile's rows are the g heads that share the key head, of 128 / g tokens, so that K and V are brought in
// once for all of them.  Keys come in tiles of 128.  With S = Q K^T in tensor memory, a warpgroup per row tile holds a row per thread: its maximum m and
// sum l of e^(s - m); the terms go back to tensor memory as P, 16 bits, over the scores, and O += P V.  One thread issues all products in the order
// O0 S0' O1 S1', so that one tile's products run while the other's softmax does.  With 128 channels a tile's products take the tensor cores 512 cycles each,
// its 16384 exponentials the SM's 16 special-function lanes 1024, and the way round of scores, softmax and results some 3400 for both tiles.
//
// Blocks of up to 32 sequences come in the order of their work, those of the longest first and of each the last, which see the most keys.  Where there are fewer of them than
// half of the SMs, their keys are split, and the last CTA of those that share a tile joins the results in the order of the keys.
//
// The maximum that the terms are relative to may stay 8 powers of two behind: P then reaches 256, O and l are in 32 bits, and scaling O again, a round trip
// through registers, is left out for nearly every tile.  When the scores of a tile are there, so is O's last product: both are the same thread's, in order.
//
// Measured and not taken (8192 tokens of 32 heads over 8, causal: 450 us so): two warpgroups a row tile 468 us; an issuer for each row tile 589; P handed over in
// quarters 520, whole 462; 1 to 4 of 8 exponentials from a polynomial on the multiply-add pipe 453 to 500; a CTA per SM that goes over the blocks, the next one's
// first scores beside the last one's results, 469, with tiles of keys dealt out evenly over the CTAs 478.
// With 64 channels (377 us so): P beside the scores, so that the next ones wait for nothing, 381; a row tile a CTA, two CTAs an SM, 410.
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
  static constexpr int BAR_OFF = RING_OFF + STAGES * STAGE;     // full[S], empty[S], qfull, sfull[2], phalf[2], pfull[2], ofull[2], clean[4]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 13) * 8;
  static constexpr int TOTAL = MISC_OFF + 32 + 1024;            // tmem slot, abort flag, verdicts, whether values were left out; room to align
};

struct alignas(64) PromptLaunch {
  CUtensorMap kmap, vmap, qmap;
  AttentionParams p;
  AttentionWorkspace w;
  int tokens;                       // of a row tile
  int blocks;                       // of two row tiles, of all sequences (ragged: at most)
  int splits;                       // CTAs that share a block's keys
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
// What a row's terms are relative to, once its maximum so far is m: 2^(s c - m c), c the scale in powers of two, is one fused multiply-add of s, `step` = c and -`from` =
// -m c.  m c is rounded, by up to 2^-25 of it, for all terms alike, and past 2^128 none of fp32's numbers.  From 2^27 on the next smaller score's term is below 2^-7, most are
// below 2^-126, and `step` is the power of two above c, with which nothing is rounded.
struct Reference { float step, from; };
__device__ __forceinline__ float power_above(float c) { return __uint_as_float((__float_as_uint(c) + 0x007FFFFFu) & 0x7F800000u); }
__device__ __forceinline__ bool is_large(const Reference &r) { return !(fabsf(r.from) < 0x1p27f); }
__device__ __forceinline__ Reference reference(float m, float c) { return {c, m == -INFINITY ? 0.0f : __fmul_rn(m, c)}; }
__device__ __forceinline__ Reference large_reference(float m, float c) {
  const float step = power_above(c), from = m * step;
  return isinf(from) ? Reference{1.0f, m} : Reference{step, from};
}
// The factor of what is relative to the old maximum
__device__ __forceinline__ float to_reference(float old, float m, float c) {
  const Reference was = reference(old, c), is = reference(m, c);
  return old == -INFINITY ? 0.0f : exp2_approx(is_large(was) || is_large(is) ? (old - m) * c : was.from - is.from);
}
// What a partial result says that it is relative to, in powers of two times unit_of(c), which rounds nothing and keeps it in fp32's range; or -inf.
__device__ __forceinline__ float unit_of(float c) { return fmaxf(power_above(c), 1.0f); }
__device__ __forceinline__ float left_reference(float m, float c) {
  const Reference r = reference(m, c);
  return m == -INFINITY ? m : is_large(r) ? m * fminf(power_above(c), 1.0f) : r.from / unit_of(c);
}
// A matrix descriptor whose low word, the address and the distance along M or N, is worked out in 32 bits
__device__ __forceinline__ uint64_t with_low(uint64_t desc, uint32_t low) { return (desc & 0xFFFFFFFF00000000ull) | low; }

// The `at`-th block of two row tiles of a call, by a warp.  false: there is none.  Of up to 32 sequences the longest come first; of more, each has as many places as it has blocks,
// or one more: the first at its first row over a block's, plus its number, so that it is found by a search.  Of each sequence the last block is the first.
struct Block { int s, index; Sequence q; };
__device__ __forceinline__ bool find_block(const PromptLaunch &g, int at, Block &b) {
  const Sequences &batch = g.p.seq;
  const int lane = threadIdx.x & 31, per_block = 2 * g.tokens, seqs = (int)batch.seqs;
  auto blocks_of = [&](const Sequence &q) { return (q.n + per_block - 1) / per_block; };
  if (seqs > 32) {
    const int each = (batch.each + per_block - 1) / per_block;
    auto place = [&](long long s) { return batch.starts ? min(max(batch.starts[s], 0), (int)batch.rows) / per_block + (int)s : (int)s * each; };
    b.s = batch.starts ? (int)last_up_to(seqs, at, lane, place) : at / each;
    if (b.s < 0) return false;
    b.q = sequence_of(batch, b.s);
    const int behind = at - place(b.s), blocks = blocks_of(b.q);
    b.index = blocks - 1 - behind;
    return behind >= 0 && behind < blocks;                      // (whatever starts hold)
  }
  const Sequence own = lane < seqs ? sequence_of(batch, lane) : Sequence{0, 0, -1};
  int rank = 0, s = lane;
  for (int j = 0; j < seqs; ++j) {
    const int other = __shfl_sync(0xFFFFFFFFu, own.length, j);
    rank += other > own.length || (other == own.length && j < lane);
  }
  for (int j = 0; j < seqs; ++j)
    if (__shfl_sync(0xFFFFFFFFu, rank, j) == lane) s = j;
  const Sequence q = {__shfl_sync(0xFFFFFFFFu, own.first, s), __shfl_sync(0xFFFFFFFFu, own.n, s), __shfl_sync(0xFFFFFFFFu, own.length, s)};
  const int blocks = lane < seqs ? blocks_of(q) : 0;
  int upto = blocks;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, k);
    if (lane >= k) upto += v;
  }
  const uint32_t who = __ballot_sync(0xFFFFFFFFu, at < upto);
  if (who == 0) return false;
  const int mine = __ffs(who) - 1;
  b.s = __shfl_sync(0xFFFFFFFFu, s, mine);
  b.index = __shfl_sync(0xFFFFFFFFu, upto - 1 - at, mine);
  b.q = {__shfl_sync(0xFFFFFFFFu, q.first, mine), __shfl_sync(0xFFFFFFFFu, q.n, mine), __shfl_sync(0xFFFFFFFFu, q.length, mine)};
  return true;
}

template <typename T, int CB>
__global__ void __launch_bounds__(THREADS, 1) attention_prompt_kernel(const __grid_constant__ PromptLaunch g) {
  using L = Smem<CB>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t S_COL = 0, O_COL = 256, COLS = 512;        // scores 2 x 128 columns, P in their first 64; results 2 x 64 CB
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *qfull = empty + STAGES, *sfull = qfull + 1, *phalf = sfull + 2,
           *pfull = phalf + 2, *ofull = pfull + 2, *clean = ofull + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::MISC_OFF);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 4), *verdict = abort_flag + 1, *spoilt = abort_flag + 3;
  const AttentionParams &p = g.p;
  // (from lane 0: what is known to be the same in all lanes goes to the tensor cores without a move each)
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    tma_prefetch_desc(&g.qmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(qfull, 1);
    for (int i = 0; i < 4; ++i) mbar_init(&clean[i], 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&sfull[i], 1); mbar_init(&phalf[i], 4); mbar_init(&pfull[i], 4); mbar_init(&ofull[i], 2); }
    *abort_flag = *spoilt = 0;
    fence_barrier_init();
  }
  const KeyTiles<TILE> kt(p.page_size);
  if (kt.rows < TILE) {                                         // rows of a tile that no copy fills: zeros, as values that nothing is multiplied with
    for (int i = threadIdx.x; i < STAGES * L::STAGE / 16; i += THREADS) reinterpret_cast<uint4 *>(smem + L::RING_OFF)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncthreads();
  griddep_wait();
  const int item = blockIdx.x / g.splits, split = blockIdx.x - item * g.splits, head = item % p.kv_heads;
  Block block;
  if (!find_block(g, item / p.kv_heads, block)) return;         // (the same for all warps)
  // (the copies start without tensor memory, which is taken when the kernel in front has ended; the kernel behind may start when it has been)
  if (warp == 1 || warp >= 4) {
    if (warp == 1) {
      tmem_alloc(tmem_slot, COLS);
      griddep_launch_dependents();
    }
    tc_fence_before_sync();
    named_bar_sync(3, 9 * 32);
    tc_fence_after_sync();
  }
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);        // (nothing yet in the other warps)
  // The tiles of keys that this CTA has, [t0, t1), of which the row tiles see those below n0 and n1
  const int length = block.q.length, n = block.q.n, row0 = block.index * 2 * g.tokens;
  auto seen_by = [&](int i) {
    const int first = row0 + i * g.tokens, last = min(first + g.tokens, n) - 1;
    return __shfl_sync(0xFFFFFFFFu, first >= n ? 0 : kt.count(max(0, p.causal ? min(length, length - n + last + 1) : length)), 0);
  };
  const int seen0 = seen_by(0), seen1 = seen_by(1), all = max(seen0, seen1);
  const int t0 = g.splits > 1 ? (int)((long long)all * split / g.splits) : 0, t1 = g.splits > 1 ? (int)((long long)all * (split + 1) / g.splits) : all;
  const int n0 = max(t0, min(t1, seen0)), n1 = max(t0, min(t1, seen1));
  const int edge = p.causal ? max(length - n + row0 + 1, 0) : length;      // the first key that not all rows see
  // Values behind the sequence's end may be anything, and 0 times anything is not always 0; those of keys that not all rows see may not be finite (clear_not_finite).
  // The tile in which the sequence ends and those from the edge on, a few of a block's, are looked at by the warp that copies: it has nothing else to do by then.
  const int last = kt.count(length) - 1, looked_at = edge < length ? kt.count(edge + 1) - 1 : kt.held(last, length) < TILE ? last : INT32_MAX;
  int fail_code = 0;

  if (warp < 4) {
    reg_dealloc<REGS_OTHERS>();
    if (warp == 0) {
      // ---- copies: queries, then K and V of each tile, a lane per copy, [64 channels][page of the tile]
      const int boxes = kt.pages ? kt.pages : 1, cb = lane / boxes, page_in_tile = lane - cb * boxes;
      const bool mine = lane < CB * boxes;
      const uint32_t bytes = CB * boxes * kt.box() * 128;
      int next_page = 0, next_token = 0;
      auto read = [&](int t) {
        next_page = (int)p.seq.pages;                           // one outside the map: zeros
        next_token = 0;
        if (!kt.page) {
          next_page = block.s;
          next_token = t * TILE;
        } else if (mine) {
          int i = t * kt.pages + page_in_tile;
          if (!kt.pages) {
            i = kt.page_of(t);
            next_token = (t - i * kt.parts) * TILE;
          }
          if ((long long)i * kt.page < length) next_page = p.seq.table[block.s * p.seq.width + i];
          else next_token = -1;                                 // behind the sequence's end
        }
      };
      if (t1 > t0) {
        read(t0);
        if (lane == 0) mbar_arrive_expect_tx(qfull, 2 * CB * group * g.tokens * 128);
        __syncwarp();
        if (lane < 2 * CB)                                      // (rows that are not there: others', or zeros)
          tma_tile_3d(smem + lane * BOX_BYTES, &g.qmap, lane % CB * 64, head * group, block.q.first + row0 + lane / CB * g.tokens, qfull);
      }
      int issued = 0;
      bool ok = true;
      auto look_at = [&](int t) {
        const int fill = (t - t0) * 2 + 1, begin = max(edge - kt.first(t), 0), end = kt.held(t, length);
        uint8_t *rows = smem + L::RING_OFF + fill % STAGES * L::STAGE;
        ok = ok && mbar_wait_uniform(&full[fill % STAGES], (fill / STAGES) & 1, abort_flag);
        if (ok && t == last)
          for (int j = end * 8 + lane; j < TILE * 8; j += 32)
#pragma unroll
            for (int c = 0; c < CB; ++c) reinterpret_cast<uint4 *>(rows + c * BOX_BYTES)[j] = make_uint4(0, 0, 0, 0);
        if (ok && begin < end && clear_not_finite<T, CB, BOX_BYTES, 4>(rows, begin, end)) *spoilt = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&clean[(t - max(looked_at, t0)) & 3]);
      };
      for (int t = t0; t < t1 && ok; ++t) {
        int page = next_page;
        const int token = max(next_token, 0);
        if ((unsigned)page >= (unsigned)p.seq.pages && kt.page) {
          if (mine && next_token >= 0) report_status(p.status, ST_BAD_PAGE);
          page = (int)p.seq.pages;
        }
        if (t + 1 < t1) read(t + 1);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int stage = issued % STAGES;
          if (!mbar_wait_uniform(&empty[stage], ((issued / STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          __syncwarp();
          if (mine)
            tma_tile_4d(smem + L::RING_OFF + stage * L::STAGE + cb * BOX_BYTES + page_in_tile * kt.page * 128, v ? &g.vmap : &g.kmap, cb * 64, token, head, page,
                        &full[stage]);
          ++issued;
        }
        if (ok && t > t0 && t - 1 >= looked_at) look_at(t - 1);   // (behind the copies of the next tile, in front of those that wait for the products with this one)
      }
      if (ok && t1 > t0 && t1 - 1 >= looked_at) look_at(t1 - 1);
      if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
      // no copy is in flight when the block ends, however its other warps end
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1, abort_flag);
      if (t1 > t0) mbar_wait_warp(qfull, 0, abort_flag);
    } else if (warp == 1 && t1 > t0) {
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
      uint32_t phase = 0;
      bool ok = mbar_wait_uniform(qfull, 0, abort_flag);
      auto next_full = [&]() {
        ok = ok && mbar_wait_uniform(&full[stage], phase, abort_flag);
        const int here = stage;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        return here;
      };
      auto scores = [&](int i, int from) {
        const uint32_t ql = q_low + i * (L::Q_BYTES >> 4), kl = k_low + from * (L::STAGE >> 4);
#pragma unroll
        for (int k = 0; k < CB * 4; ++k) {
          const uint32_t at = (k >> 2) * (BOX_BYTES >> 4) + (k & 3) * 2;
          if (k < ksteps) umma_f16_el(tmem + S_COL + i * TILE, with_low(q_desc, ql + at), with_low(k_desc, kl + at), s_idesc, k != 0, el);
        }
        umma_commit_el(&sfull[i], el);
      };
      // (four barriers in turns: tile t + 4's values are not copied before tile t's have been multiplied)
      static_assert(STAGES <= 8, "");
      auto next_values = [&](int t) {
        const int at = next_full(), k = t - max(looked_at, t0);
        if (k >= 0) ok = ok && mbar_wait_uniform(&clean[k & 3], (k >> 2) & 1, abort_flag);
        return at;
      };
      int keys_at = next_full();
      if (ok) {
        tc_fence_after_sync();
        if (n0 > t0) scores(0, keys_at);
        if (n1 > t0) scores(1, keys_at);
        umma_commit_el(&empty[keys_at], el);
      }
      int values_at = next_values(t0);
      uint32_t parity = 0;
      if (t0 + 1 < t1) keys_at = next_full();
      for (int t = t0; t < t1 && ok; ++t, parity ^= 1) {
        const uint32_t vl = v_low + values_at * (L::STAGE >> 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int end = i ? n1 : n0;
          if (t < end) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && mbar_wait_uniform(half ? &pfull[i] : &phalf[i], parity, abort_flag);
              if (!ok) break;
              tc_fence_after_sync();
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int k = half * 4 + j;
                umma_f16_ts_el(tmem + O_COL + i * CB * 64, tmem + S_COL + i * TILE + k * 8, with_low(v_desc, vl + k * 128), o_idesc, k > 0 || t > t0, el);
              }
            }
            if (!ok) break;
            if (t + 1 < end) scores(i, keys_at);
            else {
              umma_commit_el(&ofull[i], el);
              if (lane == 0) mbar_arrive(&ofull[i]);            // (and what this warp has written)
            }
          }
        }
        umma_commit_el(&empty[values_at], el);
        if (t + 1 < t1) {
          umma_commit_el(&empty[keys_at], el);
          values_at = next_values(t + 1);
          if (t + 2 < t1) keys_at = next_full();
        }
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_MMA;
    }
  } else {
    // ---- rows
    reg_alloc<REGS_ROWS>();
    const int i = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, in_tile = r / group, token = row0 + i * g.tokens + in_tile, end = i ? n1 : n0, tiles = end - t0;
    const bool mine = in_tile < g.tokens && token < n;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, s_at = tmem + lanes + S_COL + i * TILE, o_at = tmem + lanes + O_COL + i * CB * 64;
    const float c = fabsf(p.scale) * 1.4426950408889634f, slack = fminf(SLACK / c, 3e38f);
    const int seen = p.causal ? min(length, length - n + token + 1) : length;
    float l = 0.0f;
    float m = -INFINITY;
    Reference ref = reference(m, c);
    uint32_t parity = 0;
    for (int t = t0; t < end; ++t, parity ^= 1) {
      if (!mbar_wait_uniform(&sfull[i], parity, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_EPILOGUE; break; }
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
            if (q * 32 + k >= limit) s[q][k] = 0xFF800000u;     // -inf
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
        const float to = top > m + slack ? top : m, scale = to_reference(m, to, c);
        m = to;
        ref = reference(m, c);
        if (is_large(ref)) ref = large_reference(m, c);
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
      }
      const uint64_t step2 = pair(ref.step, ref.step), from2 = pair(-ref.from, -ref.from);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint64_t z = fma2(pair(__uint_as_float(s[q][2 * k]), __uint_as_float(s[q][2 * k + 1])), step2, from2);
          float a, b;
          unpair(z, a, b);
          a = exp2_approx(a);
          b = exp2_approx(b);
          sum[k & 1] = add2(sum[k & 1], pair(a, b));
          w[k] = pack2<T>(a, b);                                // the second product's operand has 16 bits
        }
        tmem_st16(s_at + q * 16, w);
        if (q == 1) {                                           // the first half of the keys can be multiplied with their values
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&phalf[i]);
        }
      }
      float l4[4];
      unpair(sum[0], l4[0], l4[1]);
      unpair(sum[1], l4[2], l4[3]);
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[i]);
    }
    if (tiles > 0 && fail_code == 0 && !mbar_wait_uniform(&ofull[i], 0, abort_flag)) fail_code = ST_WAIT_TIMEOUT_EPILOGUE;
    // (the queries' place is written below: where nothing was computed, their copy has to have landed first)
    if (tiles == 0 && t1 > t0 && !mbar_wait_uniform(qfull, 0, abort_flag)) fail_code = ST_WAIT_TIMEOUT_EPILOGUE;
    tc_fence_after_sync();
    if (__any_sync(0xFFFFFFFFu, tiles > 0 && *spoilt != 0)) {     // values that are not finite: those that the row sees
#pragma unroll 1
      for (int q = 0; q < 2 * CB; ++q) {
        uint32_t o[32];
        tmem_ld32(o_at + q * 32, o);
        tmem_ld_wait();
        tmem_arrived32(o);
#pragma unroll 1
        for (int j = edge; j < (mine ? seen : 0); ++j) {
          const long long at = place_of_key(p, block.s, j);
          const T *v = static_cast<const T *>(p.v) + at + head * p.ld_head + q * 32;
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float x = at >= 0 && q * 32 + k < p.head_dim ? to_f32(v[k]) : 0.0f;
            if (!isfinite(x)) o[k] = __float_as_uint(__uint_as_float(o[k]) + x);
          }
        }
        __syncwarp();
        tmem_st32(o_at + q * 32, o);
      }
      tmem_st_wait();
    }
    T *out = static_cast<T *>(p.out) + (long long)(block.q.first + token) * p.ld_out + (long long)(head * group + r - in_tile * group) * p.head_dim;
    const uint32_t rows_here = __ballot_sync(0xFFFFFFFFu, mine);
    // A row per thread would make 32 lines of each store: 64 channels of a warp's rows go through the place of its queries, which nothing reads any more, 16-byte word x
    // of row y at x ^ (y & 7), and on to memory eight lanes to a row.
    uint4 *stage = reinterpret_cast<uint4 *>(smem + i * L::Q_BYTES + (warp & 3) * 32 * 128);
    auto write = [&](const float (&v)[32], int q, float inv) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        stage[lane * 8 + (((q & 1) * 4 + k) ^ (lane & 7))] =
            make_uint4(pack2<T>(v[k * 8] * inv, v[k * 8 + 1] * inv), pack2<T>(v[k * 8 + 2] * inv, v[k * 8 + 3] * inv),
                       pack2<T>(v[k * 8 + 4] * inv, v[k * 8 + 5] * inv), pack2<T>(v[k * 8 + 6] * inv, v[k * 8 + 7] * inv));
      if ((q & 1) == 0) return;
      __syncwarp();
      const int word = lane & 7, ch = (q >> 1) * 64 + word * 8;
#pragma unroll
      for (int y0 = 0; y0 < 32; y0 += 4) {
        const int y = y0 + (lane >> 3);
        T *to = reinterpret_cast<T *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(out), y));
        const uint4 x = stage[y * 8 + (word ^ (y & 7))];
        if (((rows_here >> y) & 1) && ch < p.head_dim) *reinterpret_cast<uint4 *>(to + ch) = x;
      }
      __syncwarp();
    };
    // a partial result: [4 channels][row], then the rows' maxima and sums
    constexpr int WIDE = CB * 64;
    auto part = [&](int k) { return g.w.partial + ((size_t)(item * g.splits + k) * 2 + i) * (TILE * (WIDE + 2)); };
    if (row0 + i * g.tokens < n) {                              // (a row tile with rows: the same for its four warps)
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
            reinterpret_cast<float4 *>(part(split))[(q * 8 + k) * TILE + r] =
                make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
      }
      if (g.splits > 1) {
        if (mine) reinterpret_cast<float2 *>(part(split) + TILE * WIDE)[r] = make_float2(left_reference(m, c), l);
        named_bar_sync(1 + i, 128);
        // (released and acquired by one thread for the row tile's four warps, which the barriers order)
        if (r == 0) {
          int before, *arrived = g.w.arrived + item * 2 + i;
          asm volatile("atom.acq_rel.gpu.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(arrived) : "memory");
          if (before == g.splits - 1) *arrived = 0;
          verdict[i] = before == g.splits - 1;
        }
        named_bar_sync(1 + i, 128);
        if (verdict[i] != 0) {                                  // (rows that are not there read what others left, and write nothing)
          const float unit = unit_of(c);
          float top = -INFINITY, whole = 0.0f;
          for (int k = 0; k < g.splits; ++k) top = fmaxf(top, __ldcg(reinterpret_cast<const float2 *>(part(k) + TILE * WIDE) + r).x);
          const float from = top == -INFINITY ? 0.0f : top;
          for (int k = 0; k < g.splits; ++k) {
            const float2 x = __ldcg(reinterpret_cast<const float2 *>(part(k) + TILE * WIDE) + r);
            whole += x.y * exp2_approx((x.x - from) * unit);
          }
          const float inv = whole == 0.0f ? 0.0f : 1.0f / whole;
#pragma unroll 1
          for (int q = 0; q < 2 * CB; ++q) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = 0.0f;
#pragma unroll 2
            for (int k = 0; k < g.splits; ++k) {
              const float w = exp2_approx((__ldcg(reinterpret_cast<const float2 *>(part(k) + TILE * WIDE) + r).x - from) * unit);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(part(k)) + (q * 8 + j) * TILE + r);
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
cudaError_t go(const PromptLaunch &g, cudaStream_t s) {
  static_assert(2 * TILE * (CB * 64 + 2) <= PROMPT_PARTIAL, "");
  return launch_overlapped(attention_prompt_kernel<T, CB>, dim3((unsigned)(g.blocks * g.p.kv_heads * g.splits)), dim3(THREADS), Smem<CB>::TOTAL, s, g);
}
template <typename T>
cudaError_t go(const PromptLaunch &g, cudaStream_t s) { return g.p.head_dim <= 64 ? go<T, 1>(g, s) : go<T, 2>(g, s); }
template <typename K>
cudaError_t allow(K kern, int smem) { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }

long long blocks_of(const AttentionParams &p, int tokens) {
  if (!p.seq.starts) return p.seq.seqs * ((p.seq.each + 2ll * tokens - 1) / (2 * tokens));
  return p.seq.rows / (2 * tokens) + p.seq.seqs;
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
  return p.words && p.head_dim <= 128 && group <= TILE && p.page_size % 8 == 0 && p.seq.width > 0 && p.seq.pages > 0 &&
         blocks_of(p, TILE / group) * p.kv_heads <= INT32_MAX;
}

// Keys are split where that fills the SMs, into no fewer than three tiles each of what the sequences can hold; the workspace has a place for each SM.
// (512 tokens behind 15488, 32 heads over 8: 221 us whole, 132 split in two.)
cudaError_t launch_attention_prompt(const AttentionParams &p, const AttentionWorkspace &w, cudaStream_t s) {
  PromptLaunch g;
  const int rows = KeyTiles<TILE>(p.page_size).box(), group = p.heads / p.kv_heads;
  g.p = p;
  g.tokens = TILE / group;
  g.blocks = (int)blocks_of(p, g.tokens);
  g.w = w;
  const int fit = p.num_sms / (g.blocks * p.kv_heads), worth = p.seq.capacity / (3 * TILE);
  g.splits = fit < worth ? fit : worth;
  if (g.splits < 1) g.splits = 1;
  if (!encode_keys(&g.kmap, p, p.k, rows) || !encode_keys(&g.vmap, p, p.v, rows) || !encode_queries(&g.qmap, p, group, g.tokens)) return cudaErrorInvalidValue;
  return p.et == ET_BF16 ? go<__nv_bfloat16>(g, s) : go<__half>(g, s);
}

}  // namespace elb
