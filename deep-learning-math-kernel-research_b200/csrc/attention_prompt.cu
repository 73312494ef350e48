// Attention of prompts on tensor cores.
//
// A CTA takes one key head and two tiles of 128 rows: a tile's rows are the g heads that share the key head, of 128 / g tokens, so that K and V are brought in
// once for all of them.  Keys come in tiles of 128.  With S = Q K^T in tensor memory, a warpgroup per row tile holds a row per thread: its maximum m and
// sum l of e^(s - m); the terms go back to tensor memory as P, 16 bits, over the scores, and O += P V.  One thread issues all products in the order
// O0 S0' O1 S1', so that one tile's products run while the other's softmax does.  A tile of 128 x 128 x 128 takes the tensor cores 512 cycles, twice, and its
// 16384 exponentials the SM's 16 special-function lanes 1024.
//
// The maximum that the terms are relative to may stay 8 powers of two behind: P then reaches 256, O and l are in 32 bits, and scaling O again, a round trip
// through registers, is left out for nearly every tile.  When the scores of a tile are there, so is O's last product: both are the same thread's, in order.
#include <cmath>

#include "attention.cuh"
#include "elb_common.cuh"
#include "umma.cuh"

namespace elb {

namespace {

constexpr int TILE = 128, THREADS = 384;                        // four warps: copies, products; two warpgroups of rows
constexpr int BOX_BYTES = TILE * 128;                           // 128 rows of 64 channels
constexpr int REGS_ROWS = 224, REGS_OTHERS = 56;                // (2 * 224 + 56) * 128 = 168 * 384
constexpr float SLACK = 8.0f;                                   // powers of two

template <int CB>
struct Smem {
  static constexpr int Q_BYTES = CB * BOX_BYTES, STAGE = CB * BOX_BYTES;
  static constexpr int STAGES = CB == 1 ? 8 : 5;                // of K or V
  static constexpr int RING_OFF = 2 * Q_BYTES;
  static constexpr int BAR_OFF = RING_OFF + STAGES * STAGE;     // full[S], empty[S], qfull, sfull[2], pfull[2], ofull[2]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 7) * 8;
  static constexpr int TOTAL = MISC_OFF + 16 + 1024;            // tmem slot, abort flag; room to align
};

struct alignas(64) PromptLaunch {
  CUtensorMap kmap, vmap, qmap;
  AttentionParams p;
  int tokens;                       // of a row tile
  int blocks;                       // of two row tiles, of all sequences (ragged: at most)
};

// The block of two row tiles that a CTA has, by a warp: the last blocks first, which see the most keys
struct Block { int s, index; Sequence q; };
__device__ __forceinline__ bool find_block(const PromptLaunch &g, int at, Block &b) {
  const Sequences &q = g.p.seq;
  const int per_block = 2 * g.tokens;
  if (!q.starts) {
    const int per = (q.each + per_block - 1) / per_block;
    b.index = (int)(per - 1 - at / q.seqs);
    b.s = (int)(at % q.seqs);
    b.q = sequence_of(q, b.s);
    return true;
  }
  const int lane = threadIdx.x & 31, per = (int)((q.seqs + 31) / 32), s0 = lane * per, s1 = (int)min((long long)s0 + per, q.seqs);
  auto blocks = [&](int s) { return (sequence_of(q, s).n + per_block - 1) / per_block; };
  int sum = 0;
#pragma unroll 4
  for (int s = s0; s < s1; ++s) sum += blocks(s);
  int scan = sum;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, scan, k);
    if (lane >= k) scan += v;
  }
  int here = scan - sum;
  const uint32_t who = __ballot_sync(0xFFFFFFFFu, at >= here && at < scan);
  if (who == 0) return false;
  int s = s0, n = 0;
  if (at >= here && at < scan) {
    for (n = blocks(s); at >= here + n; n = blocks(s)) { here += n; ++s; }
  }
  const int mine = __ffs(who) - 1;
  b.s = __shfl_sync(0xFFFFFFFFu, s, mine);
  b.index = __shfl_sync(0xFFFFFFFFu, n - 1 - (at - here), mine);
  b.q = sequence_of(q, b.s);
  return true;
}

template <typename T, int CB>
__global__ void __launch_bounds__(THREADS, 1) attention_prompt_kernel(const __grid_constant__ PromptLaunch g) {
  using L = Smem<CB>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t S_COL = 0, O_COL = 256, COLS = 512;        // scores 2 x 128 columns, P in their first 64; results 2 x 64 CB
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *qfull = empty + STAGES, *sfull = qfull + 1, *pfull = sfull + 2,
           *ofull = pfull + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::MISC_OFF);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 4);
  const AttentionParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.kmap);
    tma_prefetch_desc(&g.vmap);
    tma_prefetch_desc(&g.qmap);
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(qfull, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&sfull[i], 1); mbar_init(&pfull[i], 4); mbar_init(&ofull[i], 1); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  const KeyTiles<TILE> kt(p.page_size);
  if (kt.rows < TILE) {                                         // rows of a tile that no copy fills: zeros, as values that nothing is multiplied with
    for (int i = threadIdx.x; i < STAGES * L::STAGE / 16; i += THREADS) reinterpret_cast<uint4 *>(smem + L::RING_OFF)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncthreads();
  griddep_wait();
  const int head = blockIdx.x % p.kv_heads;
  Block block;
  const bool there = find_block(g, blockIdx.x / p.kv_heads, block);
  if (!there) return;                                           // (the same for all warps)
  if (warp == 1) tmem_alloc(tmem_slot, COLS);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  // the tiles of keys that each row tile sees
  const int length = block.q.length, n = block.q.n, row0 = block.index * 2 * g.tokens;
  auto keys_of = [&](int i) {
    const int first = row0 + i * g.tokens, last = min(first + g.tokens, n) - 1;
    return first >= n ? 0 : max(0, p.causal ? min(length, length - n + last + 1) : length);
  };
  const int n0 = kt.count(keys_of(0)), n1 = kt.count(keys_of(1)), most = max(n0, n1);
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
            i = t / kt.parts;
            next_token = (t - i * kt.parts) * TILE;
          }
          if ((long long)i * kt.page < length) next_page = p.seq.table[block.s * p.seq.width + i];
          else next_token = -1;                                 // behind the sequence's end
        }
      };
      if (most > 0) {
        read(0);
        const int tiles = n1 > 0 ? 2 : 1;
        if (lane == 0) mbar_arrive_expect_tx(qfull, tiles * CB * group * g.tokens * 128);
        __syncwarp();
        if (lane < tiles * CB)
          tma_tile_3d(smem + lane * BOX_BYTES, &g.qmap, lane % CB * 64, head * group, block.q.first + row0 + lane / CB * g.tokens, qfull);
      }
      int issued = 0;
      bool ok = true;
      for (int t = 0; t < most && ok; ++t) {
        int page = next_page;
        const int token = max(next_token, 0);
        if ((unsigned)page >= (unsigned)p.seq.pages && kt.page) {
          if (mine && next_token >= 0) report_status(p.status, ST_BAD_PAGE);
          page = (int)p.seq.pages;
        }
        if (t + 1 < most) read(t + 1);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int stage = issued % STAGES;
          if (!mbar_poll_warp(&empty[stage], ((issued / STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          __syncwarp();
          if (mine)
            tma_tile_4d(smem + L::RING_OFF + stage * L::STAGE + cb * BOX_BYTES + page_in_tile * kt.page * 128, v ? &g.vmap : &g.kmap, cb * 64, token, head, page,
                        &full[stage]);
          ++issued;
        }
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_PRODUCER;
      // no copy is in flight when the block ends, however its other warps end
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1, abort_flag);
      if (most > 0) mbar_wait_warp(qfull, 0, abort_flag);
    } else if (warp == 1 && most > 0) {
      // ---- products
      const uint32_t el = elect_one();
      const int ksteps = (p.head_dim + 15) / 16, bf = p.et == ET_BF16;
      const uint32_t s_idesc = umma_idesc(1, bf, bf, TILE, TILE) | (p.scale < 0.0f ? UMMA_NEGATE_A : 0u);
      const uint32_t o_idesc = umma_idesc(1, bf, bf, TILE, ksteps * 16) | UMMA_B_ROWS_ARE_K;
      const uint32_t qb = smem_u32(smem), ring = qb + L::RING_OFF;
      bool ok = true;
      auto wait = [&](uint64_t *bar, uint32_t parity) {
        ok = ok && mbar_poll_warp(bar, parity, abort_flag);
        return ok;
      };
      auto scores = [&](int i, int t) {
        const uint64_t qd = umma_desc_sw128(qb + i * L::Q_BYTES), kd = umma_desc_sw128(ring + 2 * t % STAGES * L::STAGE);
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t at = (k >> 2) * (BOX_BYTES >> 4) + (k & 3) * 2;
          umma_f16_el(tmem + S_COL + i * TILE, qd + at, kd + at, s_idesc, k != 0, el);
        }
        umma_commit_el(&sfull[i], el);
      };
      auto has = [&](int i, int t) { return t < (i ? n1 : n0); };
      auto full_stage = [&](int item) { return wait(&full[item % STAGES], (item / STAGES) & 1); };
      // the tile in which the sequence ends: values behind its end may be anything, and 0 times anything is not always 0
      const int last = kt.count(length) - 1, held = kt.held(last, length);
      if (wait(qfull, 0) && full_stage(0)) {
        tc_fence_after_sync();
        for (int i = 0; i < 2; ++i) if (has(i, 0)) scores(i, 0);
        umma_commit_el(&empty[0], el);
      }
      for (int t = 0; t < most && ok; ++t) {
        const int v = 2 * t + 1;
        if (!full_stage(v)) break;
        if (t == last && held < TILE) {
          uint8_t *rows = smem + L::RING_OFF + v % STAGES * L::STAGE;
          for (int j = held * 8 + lane; j < TILE * 8; j += 32)
#pragma unroll
            for (int c = 0; c < CB; ++c) reinterpret_cast<uint4 *>(rows + c * BOX_BYTES)[j] = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (t + 1 < most && !full_stage(v + 1)) break;
        for (int i = 0; i < 2; ++i) {
          if (has(i, t)) {
            if (!wait(&pfull[i], t & 1)) break;
            tc_fence_after_sync();
            const uint64_t vd = umma_desc_sw128_rows_k(ring + v % STAGES * L::STAGE, BOX_BYTES);
#pragma unroll
            for (int k = 0; k < TILE / 16; ++k) umma_f16_ts_el(tmem + O_COL + i * CB * 64, tmem + S_COL + i * TILE + k * 8, vd + k * 128, o_idesc, (t | k) != 0, el);
            if (!has(i, t + 1)) umma_commit_el(&ofull[i], el);
          }
          if (has(i, t + 1)) scores(i, t + 1);
        }
        umma_commit_el(&empty[v % STAGES], el);
        if (t + 1 < most) umma_commit_el(&empty[(v + 1) % STAGES], el);
      }
      if (!ok) fail_code = ST_WAIT_TIMEOUT_MMA;
    }
  } else {
    // ---- rows
    reg_alloc<REGS_ROWS>();
    const int i = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, in_tile = r / group, token = row0 + i * g.tokens + in_tile, tiles = i ? n1 : n0;
    const bool mine = in_tile < g.tokens && token < n;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, s_at = tmem + lanes + S_COL + i * TILE, o_at = tmem + lanes + O_COL + i * CB * 64;
    const float c = fabsf(p.scale) * 1.4426950408889634f, slack = SLACK / c;
    const int seen = p.causal ? min(length, length - n + token + 1) : length;
    float m = -INFINITY, l = 0.0f;
    for (int t = 0; t < tiles; ++t) {
      if (!mbar_poll_warp(&sfull[i], t & 1, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_EPILOGUE; break; }
      tc_fence_after_sync();
      uint32_t s[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(s_at + q * 32, s[q]);
      tmem_ld_wait();
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_arrived32(s[q]);
      const int limit = min(kt.held(t, length), seen - kt.first(t));
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
        const float to = top > m + slack ? top : m, scale = m == -INFINITY ? 0.0f : exp2_approx((m - to) * c);
        if (t > 0) {
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
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float a = exp2_approx(fmaf(__uint_as_float(s[q][2 * k]), c, -from)), b = exp2_approx(fmaf(__uint_as_float(s[q][2 * k + 1]), c, -from));
          sum[k & 3] += a + b;
          w[k] = pack2<T>(a, b);                                // the second product's operand has 16 bits
        }
        tmem_st16(s_at + q * 16, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[i]);
    }
    if (tiles > 0 && fail_code == 0 && !mbar_poll_warp(&ofull[i], 0, abort_flag)) fail_code = ST_WAIT_TIMEOUT_EPILOGUE;
    tc_fence_after_sync();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = static_cast<T *>(p.out) + (long long)(block.q.first + token) * p.ld_out + (long long)(head * group + r - in_tile * group) * p.head_dim;
#pragma unroll 1
    for (int q = 0; q < 2 * CB; ++q) {
      uint32_t o[32];
      if (tiles > 0) tmem_ld32(o_at + q * 32, o);
      tmem_ld_wait();
      tmem_arrived32(o);
      if (mine) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (q * 32 + k * 8 >= p.head_dim) break;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = tiles > 0 ? pack2<T>(__uint_as_float(o[k * 8 + 2 * j]) * inv, __uint_as_float(o[k * 8 + 2 * j + 1]) * inv) : 0u;
          *reinterpret_cast<uint4 *>(out + q * 32 + k * 8) = make_uint4(w[0], w[1], w[2], w[3]);
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
  return launch_overlapped(attention_prompt_kernel<T, CB>, dim3((unsigned)(g.blocks * g.p.kv_heads)), dim3(THREADS), Smem<CB>::TOTAL, s, g);
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

cudaError_t launch_attention_prompt(const AttentionParams &p, cudaStream_t s) {
  PromptLaunch g;
  const int rows = KeyTiles<TILE>(p.page_size).box(), group = p.heads / p.kv_heads;
  g.p = p;
  g.tokens = TILE / group;
  g.blocks = (int)blocks_of(p, g.tokens);
  if (!encode_keys(&g.kmap, p, p.k, rows) || !encode_keys(&g.vmap, p, p.v, rows) || !encode_queries(&g.qmap, p, group, g.tokens)) return cudaErrorInvalidValue;
  return p.et == ET_BF16 ? go<__nv_bfloat16>(g, s) : go<__half>(g, s);
}

}  // namespace elb
