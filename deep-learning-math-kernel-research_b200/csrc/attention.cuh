// Parameter blocks and launchers of the attention operators (elb_rotary_*, elb_append_*, elb_attention_*).
#pragma once
#include <type_traits>

#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

// The sequences of a call: rows [first, first + n) of its new tokens, `length` tokens in all.  Whatever starts and lengths hold, rows lie in the
// call and the length in what table or tensor can hold.
struct Sequences {
  const int *table, *lengths, *starts;
  long long rows, seqs, width, pages;
  int each;                         // rows of every sequence, where starts is null
  int capacity;                     // tokens that a sequence can hold
};
struct Sequence { int first, n, length; };
__device__ __forceinline__ Sequence sequence_of(const Sequences &b, int s) {
  Sequence q;
  if (b.starts) {
    const int end = min(max(b.starts[s + 1], 0), (int)b.rows);
    q.first = min(max(b.starts[s], 0), (int)b.rows);
    q.n = max(end - q.first, 0);
  } else {
    q.first = s * b.each;
    q.n = b.each;
  }
  q.length = b.lengths ? min(max(b.lengths[s], 0), b.capacity) : b.capacity;
  return q;
}
// The last i of 0 .. n - 1 whose value(i) is not above x, by a warp, a lane a value: values do not fall.  (They are the caller's tensors': where they do, some i.)  -1: none
template <typename F>
__device__ __forceinline__ long long last_up_to(long long n, int x, int lane, F value) {
  long long at = 0;                                             // value(i) <= x below it; n more are not known
  while (n > 0) {
    const long long step = (n + 31) / 32, mine = (lane + 1) * step - 1;
    const int below = __popc(__ballot_sync(0xFFFFFFFFu, mine < n && value(at + mine) <= x));
    at += below * step;
    n = min(step - 1, n - below * step);                        // (of the step that ends above x, or of what is left behind the last whole one)
  }
  return at - 1;
}
// The sequence of a row, found by a warp.  seqs, or -1: none.
__device__ __forceinline__ int sequence_of_row(const Sequences &b, int row, int lane) {
  if (!b.starts) return row / b.each;
  return (int)last_up_to(b.seqs + 1, row, lane, [&](long long s) { return b.starts[s]; });
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// A call's tiles, dealt out in order: the first `more` CTAs take each + 1 of them, the others `each`.
struct Deal {
  long long each = 0, more = 0;
  int ctas = 0;
  Deal() = default;
  __device__ __forceinline__ Deal(long long total, long long most) : ctas((int)min(most, total)) {
    each = quotient(total, ctas);
    more = total - each * ctas;
  }
  __device__ __forceinline__ long long begin(int c) const { return c * each + min((long long)c, more); }
  __device__ __forceinline__ int owner(long long tile) const {
    const long long of_more = more * (each + 1);
    return (int)(tile < of_more ? quotient(tile, each + 1) : more + quotient(tile - of_more, each));
  }
};

struct RotaryParams {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;      // append: the caches
  const int *positions;             // null: of the sequences' tokens (append)
  Sequences seq;
  long long rows;
  long long ld_q, ld_k, ld_v, ld_q_out, ld_k_out;
  long long ld_page, ld_head, ld_token;
  const unsigned long long *steps;  // of each pair: turns per position, modulo 1, times 2^64
  int heads, kv_heads, head_dim, rotary, neighbours, inverse, page_size, et;
  float magnitude;
  int words;                        // everything lies in whole 16-byte words
  int num_sms;
  int *status;
};
cudaError_t launch_rotary(const RotaryParams &p, cudaStream_t s);

struct AttentionParams {
  void *out;
  const void *q, *k, *v;
  Sequences seq;
  long long ld_q, ld_out, ld_page, ld_head, ld_token;
  int heads, kv_heads, head_dim, et, page_size, causal;
  float scale;
  int words;                        // what tiled copies ask for: 16-byte aligned tensors, strides and head_dim of whole 16 bytes
  int num_sms;
  int *status;
};

// Where key j of sequence s lies in k and v (of key head 0); -1: in a page outside the pool
__device__ __forceinline__ long long place_of_key(const AttentionParams &p, int s, int j) {
  if (!p.page_size) return s * p.ld_page + j * p.ld_token;
  const int page = p.seq.table[s * p.seq.width + j / p.page_size];
  return page >= 0 && page < p.seq.pages ? page * p.ld_page + j % p.page_size * p.ld_token : -1;
}

// Values that are not finite, of keys that only some of a tile's rows see: 0, the term of a row that does not see them, times that would not be 0.  The products take
// 0 in their place, and the rows that see them add them when they are done.
// Here a warp looks at rows [from, to) of a tile as copies have brought it, CB boxes of 64 channels (UNROLL words of each at once).  Where there are such values it clears
// them: true.
template <typename T, int CB, int BOX_BYTES, int UNROLL>
__device__ __forceinline__ bool clear_not_finite(uint8_t *tile, int from, int to) {
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t EXPONENTS = BF ? 0x7F807F80u : 0x7C007C00u;
  const int begin = from * 8 + (threadIdx.x & 31), end = to * 8;
  uint32_t zeros[4] = {0, 0, 0, 0};                             // a value times 0, not 0 where it is not finite
  auto times_zero = [](uint32_t &sum, uint32_t w) {
    if (BF) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w), "r"(0));
    else asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w), "r"(0));
  };
#pragma unroll UNROLL
  for (int j = begin; j < end; j += 32)
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const uint4 x = reinterpret_cast<const uint4 *>(tile + c * BOX_BYTES)[j];
      times_zero(zeros[0], x.x);
      times_zero(zeros[1], x.y);
      times_zero(zeros[2], x.z);
      times_zero(zeros[3], x.w);
    }
  if (!__any_sync(0xFFFFFFFFu, ((zeros[0] | zeros[1] | zeros[2] | zeros[3]) & 0x7FFF7FFFu) != 0)) return false;
  auto cleared = [](uint32_t w) { return w & ~__vcmpeq2(w & EXPONENTS, EXPONENTS); };
#pragma unroll 1
  for (int j = begin; j < end; j += 32)
#pragma unroll 1
    for (int c = 0; c < CB; ++c) {
      uint4 &x = reinterpret_cast<uint4 *>(tile + c * BOX_BYTES)[j];
      x = make_uint4(cleared(x.x), cleared(x.y), cleared(x.z), cleared(x.w));
    }
  return true;
}

// Keys in tiles of up to TILE rows, as tiled copies bring them: whole pages where some fit, otherwise (and dense) parts of a page.
template <int TILE>
struct KeyTiles {
  int page;                         // tokens of a page; 0: dense, a sequence is one
  int pages;                        // whole pages of a tile; 0: parts of a page
  int rows;                         // tokens of a tile (of the last part of a page: at most)
  int parts;                        // of a page
  int shift;                        // parts are 1 << shift; -1: no power of two
  bool flat;                        // tile t holds keys t * TILE and on, as where pages and tiles are multiples of one another
  __host__ __device__ explicit KeyTiles(int page_size) : page(page_size) {
    pages = page_size > 0 && page_size <= TILE ? TILE / page_size : 0;
    rows = pages ? pages * page_size : TILE;
    parts = page_size > TILE ? (page_size + TILE - 1) / TILE : 1;
    flat = page_size > TILE ? page_size % TILE == 0 : rows == TILE;
    shift = -1;
    if ((parts & (parts - 1)) == 0)
      for (shift = 0; 1 << shift < parts;) ++shift;
  }
  __host__ __device__ int box() const { return pages ? page : TILE; }
  __host__ __device__ int count(int keys) const {
    if (flat) return (keys + TILE - 1) / TILE;
    return page > TILE ? keys / page * parts + (keys % page + TILE - 1) / TILE : (keys + rows - 1) / rows;
  }
  // the page that a tile is a part of
  __device__ __forceinline__ int page_of(int t) const { return shift >= 0 ? t >> shift : t / parts; }
  // the first key of a tile, and how many rows of it are keys, of `keys` in all
  __device__ __forceinline__ int first(int t) const {
    if (flat) return t * TILE;
    return page > TILE ? page_of(t) * page + (t - page_of(t) * parts) * TILE : t * rows;
  }
  __device__ __forceinline__ int held(int t, int keys) const {
    if (flat) return min(TILE, keys - t * TILE);
    const int here = page > TILE ? min(TILE, page - (t - page_of(t) * parts) * TILE) : rows;
    return min(here, keys - first(t));
  }
};

// A tiled copy's view of keys or values: 64 channels x `rows` tokens, with the 128-byte swizzle; what lies outside arrives as zeros
bool encode_keys(CUtensorMap *m, const AttentionParams &p, const void *base, int rows);

// and of the queries: 64 channels x `heads` heads that share a key head x `tokens` tokens
bool encode_queries(CUtensorMap *m, const AttentionParams &p, int heads, int tokens);

// Where a call's partial results lie, the counters of their joining (two of each CTA), zero between calls.  Per SM: for few
// tokens CTAs, and floats of one partial result of each; of which a CTA has up to two, its first
// piece's and its last's; for prompts floats of one.
struct AttentionWorkspace { float *partial; int *arrived; };
constexpr int TOKEN_CTAS = 3, TOKEN_PARTIAL = 2 * 32 * (128 + 2), PROMPT_PARTIAL = 2 * 128 * (128 + 2);
inline size_t attention_partial_floats(int num_sms) { return (size_t)num_sms * (2 * TOKEN_PARTIAL > PROMPT_PARTIAL ? 2 * TOKEN_PARTIAL : PROMPT_PARTIAL); }
inline size_t attention_workspace_bytes(int num_sms) { return (attention_partial_floats(num_sms) + (size_t)num_sms * TOKEN_CTAS * 2) * 4; }

// Few rows to a key head, over pages or dense tensors that tiled copies can read
bool attention_token_takes(const AttentionParams &p);
cudaError_t init_attention();                         // kernel attributes of the current device
cudaError_t launch_attention_token(const AttentionParams &p, const AttentionWorkspace &w, cudaStream_t s);
// Prompts, in tiles of 128 rows
bool attention_prompt_takes(const AttentionParams &p);
cudaError_t init_attention_prompt();
cudaError_t launch_attention_prompt(const AttentionParams &p, const AttentionWorkspace &w, cudaStream_t s);
cudaError_t launch_attention_any(const AttentionParams &p, cudaStream_t s);

}  // namespace elb
