// Matrix products of the transformer operators, dense and grouped by expert, on packed weights (ops.cuh).
#include <cmath>

#include "elb_common.cuh"
#include "gemm_epilogue.cuh"
#include "ops.cuh"
#include "umma.cuh"

namespace elb {

// Bytes of the operand rings.  The kernel of few tiles with few tokens and shared channels leaves room for a second CTA on its
// SM (the next launch's weights arrive while this one ends, and a cluster finds its SMs); a CTA that streams a whole row tile
// wants all of the SM's memory for loads in flight (24 x 4096 -> 16384 23.4 us, 29.0 with the small ring).
//
// Clusters on several streams: a CTA of one that holds tensor memory while its partner elsewhere waits for some must not meet a CTA of another in the
// reverse position.  Kernels of the small ring take 32 columns, two of them on an SM; every other cluster's kernel fills an SM by its
// shared memory or registers; the nearest to leaving room is the fp32 direct convolution (all 512 columns), whose 512 threads of 80 registers and
// 320 of 80 here would be 66560 of 65536.  Whoever changes these counts has to look at that again.
constexpr int SMALL_RING = 110 * 1024, LARGE_RING = 224 * 1024;
constexpr int TILES_RING = 192 * 1024;

namespace {

// One thread per 16-byte chunk of the packed image.
__global__ void pack_weights_kernel(uint4 *dst, const uint16_t *src, int rows, int ic, int kt, int row_tiles, int gated, int hwio,
                                    long long chunks, long long per_expert) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < chunks; i += (long long)gridDim.x * blockDim.x) {
    const long long e = i / per_expert;
    long long r = i - e * per_expert;
    const int slot = (int)(r & 7);
    r >>= 3;
    const int in_tile = (int)(r & (GT_ROWS - 1));
    r >>= 7;
    const int k_tile = (int)(r % kt), row_tile = (int)(r / kt);
    const int p = row_tile * GT_ROWS + in_tile;                          // packed row
    const int row = packed_source(p, rows, gated);                       // row of the source
    const int k0 = k_tile * GT_K + ((slot ^ (in_tile & 7)) << 3);
    uint16_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = k0 + j;
      v[j] = 0;
      if (row < rows && k < ic)
        v[j] = hwio ? src[(e * ic + k) * rows + row] : src[(e * rows + row) * (long long)ic + k];
    }
    dst[i] = *reinterpret_cast<uint4 *>(v);
  }
}

__global__ void pack_bias_kernel(float *dst, const void *src, int et, int rows, int padded, int gated) {
  const int p = blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= padded) return;
  float v = 0.0f;
  const int row = packed_source(p, rows, gated);
  if (row < rows) {
    v = et == ET_F32 ? static_cast<const float *>(src)[row]
      : et == ET_BF16 ? to_f32(static_cast<const __nv_bfloat16 *>(src)[row]) : to_f32(static_cast<const __half *>(src)[row]);
  }
  dst[p] = v;
}

// ---------------------------------------------------------------------------------------------
// The tensor-core kernels.  Left operand (128 rows, tensor memory lanes): a tile of packed weights, one contiguous bulk copy of
// 16 KB per 64 channels.  Right operand (BN columns): BN tokens, one tiled copy with the 128-byte swizzle from the caller's
// tensor (rows and channels outside it arrive as zeros).  Few tokens then cost a narrow MMA and not a padded one, and the
// weights, which are what a small call is made of, stream through shared memory once.
// ---------------------------------------------------------------------------------------------
// Few tiles: warp 0 produces, 1 issues the MMAs, 2 to 9 are the epilogue's.  Many tiles: 0 and 2 produce, 1 issues, 3 idles, 4 to
// 15 are the epilogue's.
constexpr int SPLIT_WARPS = 8, TILES_WARPS = 12;

template <int BN, bool PAIR, int RING, int EPI_WARPS>
struct GemmSmem {
  static constexpr int X_BYTES = (PAIR ? BN / 2 : BN) * 128;
  static constexpr int STAGE = GT_BYTES + X_BYTES;
  static constexpr int STAGES = RING / STAGE;
  static constexpr int EPI_OFF = STAGES * STAGE;                     // staging of the epilogue, where it runs beside the ring
  static constexpr int BAR_OFF = EPI_OFF + EPI_WARPS * EPI_STAGE;    // full[S], empty[S], tfull[2], tempty[2]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 4) * 8;
  static constexpr int TOTAL = MISC_OFF + 16 + 1024;          // tmem slot, abort flag; room to align
};

struct alignas(64) GemmLaunch {
  CUtensorMap xmap, wmap;      // tokens; packed weights as rows of 128 bytes (pairs only)
  GemmParams p;
  int splits;                  // CTAs of a cluster that share a tile's channels
  int token_tiles, tile_tokens;
  int band;                    // token tiles that neighbouring tiles of the walk share weights over
  int box;                     // tokens of one tiled copy
  int early;                   // the tiles are known before the kernel in front of this one has ended
};

__device__ __forceinline__ uint8_t *smem_1k(uint8_t *base) { return base + ((1024u - (smem_u32(base) & 1023u)) & 1023u); }

struct EpilogueTile {
  const Epilogue &e;
  uint8_t *stage;
  uint32_t taddr;
  int part, parts, lane, prow0;
  long long tok0;
  int ntok;
};
template <typename W, typename F>
struct EpilogueCall : EpilogueTile {
  W wait;
  F release;
  template <typename OT, bool GATED>
  __device__ __forceinline__ bool operator()() {
    return epilogue_tile_as<OT, GATED>(e, stage, taddr, part, parts, lane, prow0, tok0, ntok, wait, release);
  }
};
template <typename W, typename F>
__device__ __forceinline__ bool epilogue_tile(const EpilogueTile &t, W wait, F release) { return by_kind(t.e, EpilogueCall<W, F>{t, wait, release}); }

// The partial sums of a tile, brought together over the CTAs of a cluster in the order of their ranks: blocks of 16 tokens go round the
// CTAs, those of one CTA round its two halves of warps.  A thread's accumulators lie in the same place everywhere.
struct JoinCall {
  const Epilogue &e;
  uint8_t *stage;
  uint32_t part;          // of this thread's first accumulators in its own CTA's shared memory
  int half, lane, prow0, rank, splits;
  long long tok0;
  int ntok;
  template <typename OT, bool GATED>
  __device__ __forceinline__ bool operator()() {
    EpilogueWarp<OT, GATED> w(e, stage, lane, prow0);
#pragma unroll 1
    for (int k = rank + half * splits; k * 16 < ntok; k += 2 * splits) {
      w.fetch(tok0 + k * 16, ntok - k * 16);
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.0f;
#pragma unroll 2
      for (int r = 0; r < splits; ++r) {
        uint32_t from;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(part + k * 4 * (GT_ROWS * 16)), "r"(r));
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(x[i].x), "=f"(x[i].y), "=f"(x[i].z), "=f"(x[i].w) : "r"(from + i * (GT_ROWS * 16)) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[4 * i] += x[i].x; v[4 * i + 1] += x[i].y; v[4 * i + 2] += x[i].z; v[4 * i + 3] += x[i].w; }
      }
      uint32_t a[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) a[i] = __float_as_uint(v[i]);
      w.block(a, tok0 + k * 16, ntok - k * 16, 0, 0);
    }
    return true;
  }
};

// ---- Few tiles: each belongs to a cluster of CTAs that share its channels.  The partial sums are brought together through
// distributed shared memory in the order of the ranks, each CTA finishing a part of the tokens.
template <int BN, int RING>
__global__ void __launch_bounds__(64 + SPLIT_WARPS * 32) gemm_split_kernel(const __grid_constant__ GemmLaunch g) {
  using L = GemmSmem<BN, false, RING, 0>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t COLS = BN < 32 ? 32 : BN;
  constexpr int PART = BN * GT_ROWS * 4;                      // the epilogue runs when the ring has done: partial sums and staging lie in it
  static_assert(PART + SPLIT_WARPS * EPI_STAGE <= L::STAGES * L::STAGE, "");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_1k(smem_raw);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *tfull = empty + STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::MISC_OFF);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 4);
  const GemmParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = g.splits, rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / splits, row_tile = tile % p.row_tiles, tt = tile / p.row_tiles;
  const int k0 = (int)((long long)p.kt * rank / splits), k1 = (int)((long long)p.kt * (rank + 1) / splits), steps = k1 - k0;
  const int tok0 = tt * BN, ntok = min(BN, p.rows - tok0);
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.xmap);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  if (warp >= 1) {
    // Tensor memory is taken when the kernel before this one has ended, and the kernel behind may start when it has been
    // taken: of two kernels on an SM, one that holds tensor memory never waits for one that still wants some.
    griddep_wait();
    if (warp == 1) {
      tmem_alloc(tmem_slot, COLS);
      griddep_launch_dependents();
    }
    tc_fence_before_sync();
    named_bar_sync(1, (1 + SPLIT_WARPS) * 32);
    tc_fence_after_sync();
  }
  const uint32_t tmem = warp == 0 ? 0u : *tmem_slot;
  int fail_code = 0;
  if (warp == 0) {
    const uint32_t el = elect_one();
    const uint8_t *w = p.w + ((size_t)row_tile * p.kt + k0) * GT_BYTES;
    // The weights are the plan's own: their first copies need not wait for the kernel before this one.  Issuing a copy takes a
    // thread some 250 cycles, lanes side by side take them together: the first stages are a lane's each.
    const int ahead = min(STAGES, steps);
    if (lane < ahead) {
      mbar_arrive_expect_tx(&full[lane], L::STAGE);
      tma_bulk_g2s(smem + lane * L::STAGE, w + (size_t)lane * GT_BYTES, GT_BYTES, &full[lane]);
    }
    griddep_wait();
    if (lane < ahead) tma_tile_2d(smem + lane * L::STAGE + GT_BYTES, &g.xmap, (k0 + lane) * GT_K, tok0, &full[lane]);
    __syncwarp();
    for (int i = ahead; i < steps; ++i) {
      const int s = i % STAGES;
      if (!mbar_poll_warp(&empty[s], ((i / STAGES) & 1) ^ 1, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_PRODUCER; break; }
      if (el) {
        mbar_arrive_expect_tx(&full[s], L::STAGE);
        tma_bulk_g2s(smem + s * L::STAGE, w + (size_t)i * GT_BYTES, GT_BYTES, &full[s]);
        tma_tile_2d(smem + s * L::STAGE + GT_BYTES, &g.xmap, (k0 + i) * GT_K, tok0, &full[s]);
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_one();
    const uint32_t idesc = umma_idesc(1, p.in_et == ET_BF16, p.in_et == ET_BF16, GT_ROWS, BN);
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const int s = i % STAGES;
      if (!mbar_poll_warp(&full[s], (i / STAGES) & 1, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_MMA; ok = false; break; }
      tc_fence_after_sync();
      const uint32_t a = smem_u32(smem + s * L::STAGE);
      const uint64_t ad = umma_desc_sw128(a), bd = umma_desc_sw128(a + GT_BYTES);
#pragma unroll
      for (int k = 0; k < GT_K / 16; ++k) umma_f16_el(tmem, ad + k * 2, bd + k * 2, idesc, (i | k) != 0, el);
      umma_commit_el(&empty[s], el);
    }
    if (ok) umma_commit_el(tfull, el);
  }
  const int quarter = warp & 3, half = (warp - 2) >> 2, prow0 = row_tile * GT_ROWS + quarter * 32;
  uint8_t *stage = smem + PART + (warp - 2) * EPI_STAGE;
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  float4 *part = reinterpret_cast<float4 *>(smem) + quarter * 32 + lane;     // [block of 16 tokens][4][128 threads]
  bool ok = true;
  if (warp >= 2) {
    auto wait = [&] {
      const bool done = mbar_wait_warp(tfull, 0, abort_flag);
      tc_fence_after_sync();
      return done;
    };
    ok = splits > 1 ? wait() : epilogue_tile({p.epi, stage, taddr, half, SPLIT_WARPS / 4, lane, prow0, tok0, ntok}, wait, [] {});
    if (!ok) fail_code = ST_WAIT_TIMEOUT_EPILOGUE;
    if (ok && splits > 1) {
#pragma unroll 1
      for (int k = half; k < (ntok + 15) / 16; k += 2) {
        uint32_t a[16];
        tmem_ld_block(taddr + k * 16, a);
        tmem_ld_wait16(a);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          part[(k * 4 + i) * GT_ROWS] =
              make_float4(__uint_as_float(a[4 * i]), __uint_as_float(a[4 * i + 1]), __uint_as_float(a[4 * i + 2]), __uint_as_float(a[4 * i + 3]));
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && ok) by_kind(p.epi, JoinCall{p.epi, stage, smem_u32(part), half, lane, prow0, rank, splits, tok0, ntok});
    __syncwarp();
    cluster_sync_all();                                       // nobody leaves while its partial sums are read
  }
  if (fail_code != 0) report_status(p.status, fail_code);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, COLS);
}

// ---- Many tiles: persistent CTAs, or pairs of them (PAIR: one tcgen05.mma.cta_group::2 for 256 packed rows, each CTA
// holding its 128 and half of the tokens), two accumulators, so that a tile's epilogue runs beside the next one's products.
template <int BN, bool PAIR, bool GROUPED>
__global__ void __launch_bounds__(128 + TILES_WARPS * 32, 1) gemm_tiles_kernel(const __grid_constant__ GemmLaunch g) {
  using L = GemmSmem<BN, PAIR, TILES_RING, TILES_WARPS>;
  constexpr int STAGES = L::STAGES, CTAS = PAIR ? 2 : 1;
  constexpr uint32_t ACC = BN < 32 ? 32 : BN, COLS = 2 * ACC;       // columns of an accumulator
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_1k(smem_raw);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF), *empty = full + STAGES, *tfull = empty + STAGES, *tempty = tfull + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::MISC_OFF);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC_OFF + 4);
  const GemmParams &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int row_steps = (p.row_tiles + CTAS - 1) / CTAS;      // tiles along the rows, of one or two row tiles
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&g.xmap);
    if (PAIR) tma_prefetch_desc(&g.wmap);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], CTAS * TILES_WARPS); }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  if (PAIR) cluster_sync_all();                               // the barriers exist in both CTAs
  // The producer of the weights starts at once, where these and the tiles are known before the kernel in front has ended.  The others
  // wait for that; tensor memory is taken behind it, and the kernel behind may start when it has been (see gemm_split_kernel).
  if (warp == 0 || warp == 2) {
    if (PAIR) cluster_arrive();                               // (its wait is at the end)
    if (warp == 2 || !g.early) griddep_wait();
  } else {
    griddep_wait();
    if (warp == 1) { if (PAIR) tmem_alloc2(tmem_slot, COLS); else tmem_alloc(tmem_slot, COLS); }
    tc_fence_before_sync();
    if (PAIR) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    } else if (warp != 3) {
      named_bar_sync(1, (1 + TILES_WARPS) * 32);
    }
    tc_fence_after_sync();
    if (warp == 1) griddep_launch_dependents();
  }
  const uint32_t tmem = warp == 0 || warp == 2 ? 0u : *tmem_slot;
  // (from L2: a block that is early may meet lines of an earlier call in its SM's cache)
  const int token_tiles = GROUPED ? __ldcg(p.n_tiles) : g.token_tiles;
  const int total = token_tiles * row_steps;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  struct Tile { int expert, row_tile, tok0, ntok; };
  auto tile_of = [&](int i) {
    Tile t;
    if (GROUPED) {
      const int4 q = __ldcg(reinterpret_cast<const int4 *>(p.tiles + i / row_steps));     // a GroupTile
      t.expert = q.x;
      t.tok0 = q.y;
      t.ntok = q.z;
      t.row_tile = (i % row_steps) * CTAS + rank;
    } else {
      // bands of token tiles: inside one the walk goes down the rows, so that the CTAs at work share tokens and weights in L2
      const int per = g.band * row_steps, b = i / per, in = i - b * per;
      const int width = min(g.band, token_tiles - b * g.band);
      t.expert = 0;
      t.row_tile = in / width * CTAS + rank;
      t.tok0 = (b * g.band + in % width) * g.tile_tokens;
      t.ntok = min(g.tile_tokens, p.rows - t.tok0);
    }
    return t;
  };
  // Only as many columns as a tile has tokens are multiplied, in steps of 16 per CTA; CTA 1 of a pair holds the second half.
  auto columns = [](int ntok) { return (ntok + 16 * CTAS - 1) / (16 * CTAS) * (16 * CTAS); };
  int fail_code = 0;
  if (warp == 0 || warp == 2) {
    // Two producers, of the weights and of the tokens: issuing a stage's copies from one thread took 500 cycles, as long as the
    // stage's MMAs.
    const bool weights = warp == 0;
    const uint32_t el = elect_one();
    int s = 0, free_stages = weights && g.early ? STAGES : -1;
    uint32_t phase = 1;
    bool ok = true;
    for (int i = first; i < total && ok; i += step) {
      const Tile t = tile_of(i);
      const int rt = min(t.row_tile, p.row_tiles - 1);         // (the second of a pair may lie past the last tile)
      const uint8_t *w = p.w + t.expert * p.w_stride + (size_t)rt * p.kt * GT_BYTES;
      const int wrow = PAIR ? (int)((t.expert * p.w_stride / GT_BYTES + (size_t)rt * p.kt) * GT_ROWS) : 0;
      const int mine = columns(t.ntok) / CTAS, boxes = (mine + g.box - 1) / g.box, x0 = t.tok0 + rank * mine;
      const uint32_t bytes = CTAS * (GT_BYTES + boxes * g.box * 128);
      for (int k = 0; k < p.kt; ++k) {
        // (a full ring empties when the kernel in front has ended, however long that takes; the wait behind this one has a limit)
        if (free_stages == 0) griddep_wait();
        --free_stages;
        if (!mbar_poll_warp(&empty[s], phase, abort_flag)) { ok = false; fail_code = ST_WAIT_TIMEOUT_PRODUCER; break; }
        uint8_t *dst = smem + s * L::STAGE;
        if (weights) {
          if (el) {
            if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
            if (PAIR) tma_tile_2d_pair(dst, &g.wmap, 0, wrow + k * GT_ROWS, mapa_u32(&full[s], 0));
            else tma_bulk_g2s(dst, w + (size_t)k * GT_BYTES, GT_BYTES, &full[s]);
          }
        } else if (lane < boxes) {                             // (a lane per box)
          uint8_t *to = dst + GT_BYTES + lane * g.box * 128;
          if (PAIR) tma_tile_2d_pair(to, &g.xmap, k * GT_K, x0 + lane * g.box, mapa_u32(&full[s], 0));
          else tma_tile_2d(to, &g.xmap, k * GT_K, x0 + lane * g.box, &full[s]);
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t el = elect_one();
      uint32_t count = 0, phase = 0;
      int s = 0;
      bool ok = true;
      for (int i = first; i < total && ok; i += step, ++count) {
        const uint32_t b = count & 1;
        const uint32_t idesc = umma_idesc(1, p.in_et == ET_BF16, p.in_et == ET_BF16, GT_ROWS * CTAS, columns(tile_of(i).ntok));
        if (!mbar_poll_warp(&tempty[b], ((count >> 1) & 1) ^ 1, abort_flag)) { fail_code = ST_WAIT_TIMEOUT_MMA; break; }
        tc_fence_after_sync();
        const uint32_t d = tmem + b * ACC;
        for (int k = 0; k < p.kt; ++k) {
          if (!mbar_poll_warp(&full[s], phase, abort_flag)) { ok = false; fail_code = ST_WAIT_TIMEOUT_MMA; break; }
          tc_fence_after_sync();
          const uint32_t a = smem_u32(smem + s * L::STAGE);
          const uint64_t ad = umma_desc_sw128(a), bd = umma_desc_sw128(a + GT_BYTES);
#pragma unroll
          for (int j = 0; j < GT_K / 16; ++j) {
            if (PAIR) umma_f16_2cta_el(d, ad + j * 2, bd + j * 2, idesc, (k | j) != 0, el);
            else umma_f16_el(d, ad + j * 2, bd + j * 2, idesc, (k | j) != 0, el);
          }
          if (PAIR) umma_commit_2cta_el(&empty[s], el);
          else umma_commit_el(&empty[s], el);
          if (++s == STAGES) { s = 0; phase ^= 1; }
        }
        if (ok) { if (PAIR) umma_commit_2cta_el(&tfull[b], el); else umma_commit_el(&tfull[b], el); }
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    uint32_t count = 0;
    for (int i = first; i < total; i += step, ++count) {
      const Tile t = tile_of(i);
      const uint32_t b = count & 1;
      const int prow0 = t.row_tile * GT_ROWS + quarter * 32;
      const bool ok = epilogue_tile({p.epi, smem + L::EPI_OFF + (warp - 4) * EPI_STAGE, tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * ACC, part,
                                     TILES_WARPS / 4, lane, prow0, t.tok0, t.ntok},
                                    [&] {
                                      const bool done = mbar_wait_warp(&tfull[b], (count >> 1) & 1, abort_flag);
                                      tc_fence_after_sync();
                                      return done;
                                    },
                                    [&] {
                                      tc_fence_before_sync();
                                      __syncwarp();
                                      if (lane == 0) { if (PAIR) mbar_arrive_cluster(mapa_u32(&tempty[b], 0)); else mbar_arrive(&tempty[b]); }
                                    });
      if (!ok) { fail_code = ST_WAIT_TIMEOUT_EPILOGUE; break; }
    }
  }
  __syncwarp();
  if (fail_code != 0) report_status(p.status, fail_code);
  if (PAIR && (warp == 0 || warp == 2)) cluster_wait();
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after_sync();
  if (warp == 1) { if (PAIR) tmem_dealloc2(tmem, COLS); else tmem_dealloc(tmem, COLS); }
}

// Rows of any alignment -> rows that a tiled copy can read
__global__ void align_rows_kernel(uint16_t *dst, long long pitch, const uint16_t *src, long long ld, int rows, int n) {
  griddep_launch_dependents();
  griddep_wait();
  for (long long r = blockIdx.x; r < rows; r += gridDim.x)
    for (int i = threadIdx.x; i < n; i += blockDim.x) dst[r * pitch + i] = src[r * ld + i];
}

bool encode_rows(CUtensorMap *m, int et, const void *base, long long inner, long long rows, long long pitch_bytes, int box_inner, int box_rows,
                 bool swizzle) {
  PFN_encodeTiled fn = get_encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return fn(m, et == ET_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
cudaError_t launch_gemm_kernel(K kern, const GemmLaunch &g, int grid, int threads, int smem, int cluster, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0] = overlap_attribute();
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, g);
}

template <int BN, int RING>
cudaError_t go_split(GemmLaunch &g, cudaStream_t s) {
  using L = GemmSmem<BN, false, RING, 0>;
  if (!encode_rows(&g.xmap, g.p.in_et, g.p.x, g.p.ic, g.p.rows, g.p.ld_x * 2, GT_K, BN, true)) return cudaErrorInvalidValue;
  return launch_gemm_kernel(gemm_split_kernel<BN, RING>, g, g.p.row_tiles * g.token_tiles * g.splits, 64 + SPLIT_WARPS * 32, L::TOTAL, g.splits, s);
}

template <int BN, bool PAIR, bool GROUPED>
cudaError_t go_tiles(GemmLaunch &g, cudaStream_t s) {
  using L = GemmSmem<BN, PAIR, TILES_RING, TILES_WARPS>;
  const GemmParams &p = g.p;
  const int ctas = PAIR ? 2 : 1, row_steps = (p.row_tiles + ctas - 1) / ctas;
  // dense: one copy brings a CTA's tokens; grouped: tiles have any number of them, in boxes of up to 32
  g.box = p.tiles ? (BN / ctas < 32 ? BN / ctas : 32) : g.tile_tokens / ctas;
  if (!encode_rows(&g.xmap, p.in_et, p.x, p.ic, p.rows, p.ld_x * 2, GT_K, g.box, true)) return cudaErrorInvalidValue;
  if (PAIR && !encode_rows(&g.wmap, p.in_et, p.w, GT_K, p.w_rows, 128, GT_K, GT_ROWS, false)) return cudaErrorInvalidValue;
  const long long tiles = (long long)g.token_tiles * row_steps;
  const int most = PAIR ? p.max_pairs : p.num_sms;
  const int grid = (int)(tiles < most ? tiles : most) * ctas;
  return launch_gemm_kernel(gemm_tiles_kernel<BN, PAIR, GROUPED>, g, grid, 128 + TILES_WARPS * 32, L::TOTAL, ctas, s);
}

template <typename K>
cudaError_t allow(K kern, int smem) { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }

}  // namespace

cudaError_t launch_pack_weights(void *dst, const void *src, int experts, int rows, int ic, bool gated, bool hwio, cudaStream_t s) {
  const int kt = (ic + GT_K - 1) / GT_K, row_tiles = (packed_rows(gated ? rows / 2 : rows, gated) + GT_ROWS - 1) / GT_ROWS;
  const long long per = (long long)row_tiles * kt * GT_ROWS * 8, chunks = per * experts;
  const int blocks = (int)(chunks / 256 + 1 < 148 * 64 ? chunks / 256 + 1 : 148 * 64);
  pack_weights_kernel<<<blocks, 256, 0, s>>>(static_cast<uint4 *>(dst), static_cast<const uint16_t *>(src), rows, ic, kt, row_tiles,
                                             gated, hwio, chunks, per);
  return cudaGetLastError();
}

cudaError_t launch_pack_bias(float *dst, const void *src, int et, int rows, int padded, bool gated, cudaStream_t s) {
  pack_bias_kernel<<<(padded + 255) / 256, 256, 0, s>>>(dst, src, et, rows, padded, gated);
  return cudaGetLastError();
}

cudaError_t launch_align_rows(void *dst, long long pitch, const void *src, long long ld, int rows, int n, cudaStream_t s) {
  return launch_overlapped(align_rows_kernel, dim3(rows < 148 * 16 ? rows : 148 * 16), dim3(256), 0, s, static_cast<uint16_t *>(dst), pitch,
                           static_cast<const uint16_t *>(src), ld, rows, n);
}

// Kernel attributes are a device's: once for each of them.  max_pairs: the pairs of CTAs that the device holds at once (a
// persistent kernel with more would have them run one after the other).
cudaError_t init_gemm(int num_sms, int *max_pairs) {
  cudaError_t e = cudaSuccess;
  auto want = [&](cudaError_t r) { if (e == cudaSuccess) e = r; };
  want(allow(gemm_split_kernel<16, SMALL_RING>, GemmSmem<16, false, SMALL_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<32, SMALL_RING>, GemmSmem<32, false, SMALL_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<16, LARGE_RING>, GemmSmem<16, false, LARGE_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<32, LARGE_RING>, GemmSmem<32, false, LARGE_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<64, LARGE_RING>, GemmSmem<64, false, LARGE_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<128, LARGE_RING>, GemmSmem<128, false, LARGE_RING, 0>::TOTAL));
  want(allow(gemm_split_kernel<256, LARGE_RING>, GemmSmem<256, false, LARGE_RING, 0>::TOTAL));
  want(allow(gemm_tiles_kernel<256, true, false>, GemmSmem<256, true, TILES_RING, TILES_WARPS>::TOTAL));
  want(allow(gemm_tiles_kernel<16, false, true>, GemmSmem<16, false, TILES_RING, TILES_WARPS>::TOTAL));
  want(allow(gemm_tiles_kernel<32, false, true>, GemmSmem<32, false, TILES_RING, TILES_WARPS>::TOTAL));
  want(allow(gemm_tiles_kernel<64, false, true>, GemmSmem<64, false, TILES_RING, TILES_WARPS>::TOTAL));
  want(allow(gemm_tiles_kernel<128, false, true>, GemmSmem<128, false, TILES_RING, TILES_WARPS>::TOTAL));
  want(allow(gemm_tiles_kernel<256, true, true>, GemmSmem<256, true, TILES_RING, TILES_WARPS>::TOTAL));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_sms / 2 * 2);
  cfg.blockDim = dim3(128 + TILES_WARPS * 32);
  cfg.dynamicSmemBytes = GemmSmem<256, true, TILES_RING, TILES_WARPS>::TOTAL;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(max_pairs, gemm_tiles_kernel<256, true, false>, &cfg);
  if (e == cudaSuccess && *max_pairs < 1) e = cudaErrorInvalidConfiguration;
  return e;
}

int grouped_tile_tokens(int slots, int experts) {
  const int mean = (slots + experts - 1) / experts;
  return mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : mean <= 128 ? 128 : 256;
}

cudaError_t launch_gemm(const GemmParams &p, cudaStream_t s) {
  GemmLaunch g;
  g.p = p;
  g.splits = 1;
  g.band = 8;
  g.box = 0;
  g.early = !p.tiles || p.tiles_old;
  if (p.tiles) {
    g.token_tiles = p.max_tiles;
    g.tile_tokens = p.tile_tokens;
    switch (p.tile_tokens) {
      case 16: return go_tiles<16, false, true>(g, s);
      case 32: return go_tiles<32, false, true>(g, s);
      case 64: return go_tiles<64, false, true>(g, s);
      case 128: return go_tiles<128, false, true>(g, s);
      default: return go_tiles<256, true, true>(g, s);
    }
  }
  // Which kernel and tiles: the least of a model of their time in cycles, fitted to 25 shapes with every
  // choice measured (its choice costs up to 12 % over the best of them, mostly under 4).  A step of
  // 64 channels costs a CTA about the shared memory's traffic (operands in and out, at 134 bytes per cycle, 97 in a pair) or the
  // hand-overs of its roles; a launch the steps of its busiest SM, but no less than the weights at DRAM per cycle; sharing a tile's
  // channels costs the joining of the partial sums (two cluster barriers and the distributed reads).
  constexpr double DRAM = 3400.0, JOIN = 2500.0, JOIN_TOKEN = 30.0;
  const double weights = (double)p.row_tiles * p.kt * GT_BYTES / DRAM;
  double best = 1e30;
  bool pairs = false;
  for (int bn = 16; bn <= 256; bn *= 2) {
    if (bn > 16 && p.rows <= bn / 2) break;
    const int tt = (p.rows + bn - 1) / bn;
    const long long tiles = (long long)p.row_tiles * tt;
    const double step = fmax((GT_BYTES + bn * 128) * 2 / 134.0, 385.0);
    for (int splits = 1; splits <= 4; splits *= 2) {
      if (splits > 1 && (tiles * splits > p.num_sms || p.kt < splits * 2)) break;
      const double busy = (double)((tiles * splits + p.num_sms - 1) / p.num_sms);
      const double t = fmax(busy * ((p.kt + splits - 1) / splits) * step, weights) + (splits > 1 ? JOIN + JOIN_TOKEN * bn : 0.0) +
                       (busy - 1) * (3500.0 + bn * 10.0) + 6500.0 + bn * 10.0;
      if (t < best) { best = t; g.splits = splits; g.tile_tokens = bn; g.token_tiles = tt; }
    }
  }
  const int row_pairs = (p.row_tiles + 1) / 2;
  for (int most = 256; most >= 96 && p.rows > 64; most -= 32) {            // tiles of equal size, a multiple of 32 tokens
    const int tt = (p.rows + most - 1) / most, n = ((p.rows + tt - 1) / tt + 31) / 32 * 32, count = (p.rows + n - 1) / n;
    const double step = fmax((GT_BYTES + n * 64) * 2 / 97.0, 400.0);
    const double waves = (double)(((long long)row_pairs * count + p.max_pairs - 1) / p.max_pairs);
    const double t = fmax(waves * (fmax(p.kt * step, n * 20.0) + 2500.0), weights) + 5000.0 + n * 16.0;
    if (t < best) { best = t; pairs = true; g.splits = 1; g.tile_tokens = n; g.token_tiles = count; }
  }
  if (pairs) return go_tiles<256, true, false>(g, s);
  switch (g.tile_tokens) {
    case 16: return g.splits > 1 ? go_split<16, SMALL_RING>(g, s) : go_split<16, LARGE_RING>(g, s);
    case 32: return g.splits > 1 ? go_split<32, SMALL_RING>(g, s) : go_split<32, LARGE_RING>(g, s);
    case 64: return go_split<64, LARGE_RING>(g, s);
    case 128: return go_split<128, LARGE_RING>(g, s);
    default: return go_split<256, LARGE_RING>(g, s);
  }
}

// On CUDA cores the weights are read once for every two rows, from L2 at 5.3 TB/s behind a start of 1.5 us; on tensor cores once
// behind 3.6 us (up to 4 channel tiles) to 6.4 us (16).  Measured in us, here / there: 2 x 4096 -> 4096 9.2 / 11.2, 4 x
// 4096 -> 4096 15.4 / 11.3, 4 x 2048 -> 2048 5.4 / 8.4, 16 x 1024 -> 1024 5.2 / 6.5, 32 x 512 -> 512 2.9 / 5.3, 8 x 256 -> 8192 5.8 /
// 3.6, one row of 4096 -> 16384 23.5 / 23.5.
bool gemm_wants_gemv(long long rows, int row_tiles, int kt) {
  if (rows <= 1) return true;
  if (rows > 64) return false;
  const long long bytes = (long long)row_tiles * kt * GT_BYTES * ((rows + 1) / 2);
  return bytes <= (2ll << 20) * (kt < 20 ? kt : 20);
}

// The same choice for experts.  On CUDA cores each slot reads its expert's weights, at 4.9 TB/s behind 4 us; on tensor cores
// each expert that is hit is read once, at 7.5 TB/s behind 27 us.  Measured in us, here / there, 64 experts of 12.6 MB, 8 per
// token: 1 token 24.8 / 38.4, 2 tokens 41.5 / 54.9, 4 tokens 74.0 / 72.4, 8 tokens 138 / 92; 16 experts of 0.8 MB, 2 per
// token, 16 tokens 7.5 / 20.0; 4 experts of 3.1 MB, 4 per token, 16 tokens 30.9 / 24.3.
bool experts_want_gemv(int slots, int experts, double expert_bytes) {
  const double hit = experts * (1.0 - pow(1.0 - 1.0 / experts, slots)), mb = expert_bytes * 1e-6;
  return slots <= GEMV_SLOTS && 4.0 + slots * mb / 4.9 <= 27.0 + hit * mb / 7.5;
}

}  // namespace elb
