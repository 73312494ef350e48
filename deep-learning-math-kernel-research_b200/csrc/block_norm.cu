// What lies between two blocks of a transformer: the norm behind a block, its gate and scale, the residual sum and the norm
// in front of the next block, in one pass over the data.
//
//   s = r + scale * gate * post(x);   y = pre(s)
//
// A row's values stay in registers from the load to the last store, so that each tensor is read or written once: the bound
// is HBM for long calls and the chain load -> reductions -> store for short ones.  Layer norm takes its variance around the
// mean, from the registers, not from a difference of sums.
//
// Rows of up to 1024 channels belong to a warp (no block barriers), longer ones to a block, which in long calls walks several.
// Rows that do not start at 16-byte boundaries (an odd number of channels) are taken in the aligned 8-element windows that cover
// them, the first and last of which are partly outside; the weights exist once for each of the eight places a row can
// start at (2500 x 1155, layer norms and gate, f16:
// 14.3 us, one element at a time 22.0; of 1152 channels 9.3).
#include "elb_common.cuh"
#include "ops.cuh"

namespace elb {

namespace {

// VEC consecutive elements, VEC = 8: at a 16-byte boundary.  lo .. hi: the elements that exist (others read as zero).
template <typename T, int VEC>
struct Raw {
  static constexpr int WORDS = VEC == 1 ? 1 : VEC * (int)sizeof(T) / 16;
  uint4 q[WORDS];
  T one;
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VEC == 1) one = *p;
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) q[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
  }
  __device__ __forceinline__ void load_part(const T *p, int lo, int hi) {
    if constexpr (VEC > 1) {
      T v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = i >= lo && i < hi ? p[i] : from_f32<T>(0.0f);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) q[i] = reinterpret_cast<uint4 *>(v)[i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (VEC == 1) v[0] = to_f32(one);
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) v[i * 4 + j] = __uint_as_float(w[j]);
          else {
            const float2 f = unpack2<T>(w[j]);
            v[i * 8 + 2 * j] = f.x;
            v[i * 8 + 2 * j + 1] = f.y;
          }
        }
      }
    }
  }
  __device__ __forceinline__ static void store(T *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = from_f32<T>(v[0]);
    else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[i * 4 + j]);
          else w[j] = pack2<T>(v[i * 8 + 2 * j], v[i * 8 + 2 * j + 1]);
        }
        reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  __device__ __forceinline__ static void store_part(T *p, const float (&v)[VEC], int lo, int hi) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= lo && i < hi) p[i] = from_f32<T>(v[i]);
  }
};

template <int VEC>
__device__ __forceinline__ void load_w(float (&w)[VEC], const float *p) {
  if constexpr (VEC == 1) w[0] = *p;
  else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 f = reinterpret_cast<const float4 *>(p)[i];
      w[4 * i] = f.x; w[4 * i + 1] = f.y; w[4 * i + 2] = f.z; w[4 * i + 3] = f.w;
    }
  }
}

// Sum over the threads of a row.  `slot`: another one for each call of a kernel, so that one barrier is enough.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float (&part)[4][32], int slot) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[slot][warp] = v;
    __syncthreads();
    v = lane < warps ? part[slot][lane] : 0.0f;
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  }
  return v;
}

constexpr int WARP_ROWS = 4;    // rows of a block whose rows belong to warps

// One row's arithmetic, on the values of its threads: v[i][j] is element c(i) + j, of which those outside the row are zero and stay
// out of the sums.  some(i) says whether an item has any inside; settle(i) clears those of a window's that lie outside.
template <int VEC, int ITEMS, bool WARP, bool WINDOW>
struct RowNorm {
  float (&v)[ITEMS][VEC];
  float (&part)[4][32];
  int c0, step, channels;
  __device__ __forceinline__ int c(int i) const { return c0 + i * step; }
  __device__ __forceinline__ bool some(int i) const { return c(i) < channels && (!WINDOW || c(i) + VEC > 0); }
  __device__ __forceinline__ void settle(int i) {
    if (WINDOW && (c(i) < 0 || c(i) + VEC > channels)) {          // (the first and the last of a row)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c(i) + j < 0 || c(i) + j >= channels) v[i][j] = 0.0f;
    }
  }
  // w, b: at element 0 (or, with a window, at the row's copy of the vectors)
  __device__ __forceinline__ void operator()(int kind, float eps, const float *w, const float *b, int slot) {
    float mean = 0.0f, sq = 0.0f;
    if (kind == 2) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[i][j];
      mean = row_sum<WARP>(s, part, slot) / channels;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (some(i)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] -= mean;
        if (kind == 2) settle(i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sq = fmaf(v[i][j], v[i][j], sq);
      }
    const float by = 1.0f / sqrtf(row_sum<WARP>(sq, part, slot + 1) / channels + eps);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (some(i)) {
        float wv[VEC];
        load_w<VEC>(wv, w + c(i));
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = v[i][j] * by * wv[j];
        if (b) {
          load_w<VEC>(wv, b + c(i));
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += wv[j];
        }
        settle(i);
      }
  }
};

// WINDOW: rows start anywhere, all at the same place of an 8-element window in each tensor but the gate
template <typename T, typename TR, int VEC, int ITEMS, bool WARP, bool WINDOW, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) block_norm_kernel(const NormParams p) {
  __shared__ float part[4][32];
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const long long row = WARP ? (long long)blockIdx.x * WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  if (WARP && row >= p.rows) return;
  const T *x = static_cast<const T *>(p.x) + row * p.ld_x;
  const int off = WINDOW ? (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) & (16 / sizeof(T) - 1)) : 0;
  const TR *r = static_cast<const TR *>(p.res) + row * p.ld_res;
  const T *g = static_cast<const T *>(p.gate) + (p.gate ? row / p.gate_rows * p.ld_gate : 0);
  float v[ITEMS][VEC];
  Raw<TR, VEC> res[ITEMS];
  Raw<T, VEC> gate[ITEMS];
  RowNorm<VEC, ITEMS, WARP, WINDOW> norm{v, part, lane * VEC - off, (WARP ? 32 : (int)blockDim.x) * VEC, p.channels};
  const long long shift = WINDOW ? off * p.w_pitch + off : 0;     // of a row's copy of the weights
  {
    Raw<T, VEC> raw[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = norm.c(i), lo = -c, hi = p.channels - c;
      if (norm.some(i)) {
        if (!WINDOW || (lo <= 0 && hi >= VEC)) {
          raw[i].load(x + c);
          if (p.res) res[i].load(r + c);
          if (p.gate) { if (WINDOW) gate[i].load_part(g + c, 0, VEC); else gate[i].load(g + c); }
        } else {
          raw[i].load_part(x + c, lo, hi);
          if (p.res) res[i].load_part(r + c, lo, hi);
          if (p.gate) gate[i].load_part(g + c, lo, hi);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (norm.some(i)) raw[i].get(v[i]);
      else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
      }
    }
  }
  if (p.post != 0) norm(p.post, p.post_eps, p.post_w + shift, p.post_b ? p.post_b + shift : nullptr, 0);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = norm.c(i);
    if (norm.some(i)) {
      float o[VEC];
      if (p.gate) {
        gate[i].get(o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= o[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= p.scale;
      if (p.res) {
        res[i].get(o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += o[j];
      }
      if (p.sum) {
        TR *to = static_cast<TR *>(p.sum) + row * p.ld_sum + c;
        if (!WINDOW || (c >= 0 && c + VEC <= p.channels)) Raw<TR, VEC>::store(to, v[i]);
        else Raw<TR, VEC>::store_part(to, v[i], -c, p.channels - c);
      }
    }
  }
  if (p.pre == 0 || !p.y) return;
  norm(p.pre, p.pre_eps, p.pre_w + shift, p.pre_b ? p.pre_b + shift : nullptr, 2);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = norm.c(i);
    if (norm.some(i)) {
      T *to = static_cast<T *>(p.y) + row * p.ld_y + c;
      if (!WINDOW || (c >= 0 && c + VEC <= p.channels)) Raw<T, VEC>::store(to, v[i]);
      else Raw<T, VEC>::store_part(to, v[i], -c, p.channels - c);
    }
  }
}

// Many aligned rows without a gate: blocks that walk them, a thread two vectors of each, the next row's input and residual on their
// way in registers while this row's sums are joined.  A block that has one row idles at each sum's barrier, and other blocks of its SM fill that only as
// far as registers go; with the loads in front it needs a third fewer threads for the same bytes in flight.  16384 x 4096 with two RMS
// norms and an fp32 residual: 135 us, 6.0 TB/s of 6.6 that a copy reaches (a block a row 149).  One row ahead, three blocks of 256
// threads on an SM: four leave too few registers (179), two too few warps (148), one vector a thread in 512 threads 145.
template <typename T, typename TR, int MOST, int BLOCKS>
__global__ void __launch_bounds__(MOST, BLOCKS) block_norm_walk_kernel(const NormParams p) {
  constexpr int ITEMS = 2, VEC = 8;
  __shared__ float part[2][4][32];                                // by the row's parity: one barrier lies between two rows' uses of a slot
  griddep_launch_dependents();
  griddep_wait();
  const int c0 = threadIdx.x * VEC;
  Raw<T, VEC> raw[ITEMS];
  Raw<TR, VEC> res[ITEMS];
  auto ask = [&](long long row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * (int)blockDim.x * VEC;
      if (c < p.channels) {
        raw[i].load(static_cast<const T *>(p.x) + row * p.ld_x + c);
        if (p.res) res[i].load(static_cast<const TR *>(p.res) + row * p.ld_res + c);
      }
    }
  };
  ask(blockIdx.x);
  int odd = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, odd ^= 1) {
    float v[ITEMS][VEC];
    Raw<TR, VEC> add[ITEMS];
    RowNorm<VEC, ITEMS, false, false> norm{v, part[odd], c0, (int)blockDim.x * VEC, p.channels};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (norm.some(i)) raw[i].get(v[i]);
      else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
      }
      add[i] = res[i];
    }
    if (row + gridDim.x < p.rows) ask(row + gridDim.x);
    if (p.post != 0) norm(p.post, p.post_eps, p.post_w, p.post_b, 0);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = norm.c(i);
      if (norm.some(i)) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= p.scale;
        if (p.res) {
          add[i].get(o);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += o[j];
        }
        if (p.sum) Raw<TR, VEC>::store(static_cast<TR *>(p.sum) + row * p.ld_sum + c, v[i]);
      }
    }
    if (p.pre != 0 && p.y) {
      norm(p.pre, p.pre_eps, p.pre_w, p.pre_b, 2);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (norm.some(i)) Raw<T, VEC>::store(static_cast<T *>(p.y) + row * p.ld_y + norm.c(i), v[i]);
    }
  }
}
template <typename T, typename TR, int MOST, int BLOCKS>
cudaError_t by_walk(const NormParams &p, int n, cudaStream_t s) {
  const int threads = (n + 63) / 64 * 32;
  const long long most = (long long)p.num_sms * (MOST * BLOCKS / threads);
  return launch_overlapped(block_norm_walk_kernel<T, TR, MOST, BLOCKS>, dim3((unsigned)(p.rows < most ? p.rows : most)), dim3(threads), 0, s, p);
}

// Copy a of a vector has element c at index a + c: eight places that a row's first element can have in its window, zeros around.
__global__ void norm_vector_kernel(float *dst, const void *src, int et, int n, long long pitch, float offset) {
  const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= 8 * pitch) return;
  const int c = (int)(i % pitch) - (int)(i / pitch);
  float v = 0.0f;
  if (c >= 0 && c < n)
    v = !src ? 1.0f
      : offset + (et == ET_F32 ? static_cast<const float *>(src)[c]
                  : et == ET_BF16 ? to_f32(static_cast<const __nv_bfloat16 *>(src)[c]) : to_f32(static_cast<const __half *>(src)[c]));
  dst[i] = v;
}

template <typename T, typename TR, int VEC, int ITEMS, bool WINDOW>
cudaError_t by_warps(const NormParams &p, cudaStream_t s) {
  return launch_overlapped(block_norm_kernel<T, TR, VEC, ITEMS, true, WINDOW, WARP_ROWS * 32, 1>, dim3((unsigned)((p.rows + WARP_ROWS - 1) / WARP_ROWS)),
                           dim3(WARP_ROWS * 32), 0, s, p);
}
// n: loads of a row
template <typename T, typename TR, int VEC, int ITEMS, bool WINDOW, int MOST = 1024, int BLOCKS = 1>
cudaError_t by_blocks(const NormParams &p, int n, cudaStream_t s) {
  const int threads = ((n + ITEMS - 1) / ITEMS + 31) / 32 * 32;
  return launch_overlapped(block_norm_kernel<T, TR, VEC, ITEMS, false, WINDOW, MOST, BLOCKS>, dim3((unsigned)p.rows), dim3(threads), 0, s, p);
}
template <typename T, typename TR, bool WINDOW>
cudaError_t by_vectors(const NormParams &p, int n, cudaStream_t s) {
  // Few rows: a block each with a load per thread, so that as little as possible lies behind one another (100 x 4096: 2.6 us, with
  // two 3.0).  Otherwise a warp each as long as its registers hold a row.
  const bool few = p.rows <= 2 * p.num_sms;
  if (n <= 32) return by_warps<T, TR, 8, 1, WINDOW>(p, s);
  if (few && n <= 1024) return by_blocks<T, TR, 8, 1, WINDOW>(p, n, s);
  if (n <= 64) return by_warps<T, TR, 8, 2, WINDOW>(p, s);
  if (n <= 128) return by_warps<T, TR, 8, 4, WINDOW>(p, s);
  // Walked: rows with two sums or more, where a barrier's wait is what the loads ahead hide (us, walked / a block a row: 16384 x 4096,
  // two RMS norms 102 / 113, a layer norm 78 / 92, but one RMS norm 91 / 82), and rows of more than 512 vectors, whose blocks are too
  // large for several on an SM (one RMS norm: 9000 x 8192 100 / 103, 2400 x 6144 21.2 / 26.6; two: 9000 x 8192 169 / 193).  From two
  // rows an SM on, behind `few` (300 x 4096 5.6 / 7.4, 500 8.6 / 7.9, 1100 15.1 / 16.7).  Not with a gate, whose rows are not loaded
  // ahead (8000 x 4096, layer norms 85 / 78; 4000 x 8192, one RMS norm 61 / 52), and not up to 256 vectors, where enough blocks are
  // resident (30000 x 1536 92.6 / 97.2, but 900 x 1600 5.5 / 5.2).
  const int sums = p.post + (p.y ? p.pre : 0);                    // (ELB_NORM_RMS is one, ELB_NORM_LAYER two)
  if (!WINDOW && !p.gate) {
    if (n > 256 && n <= 512 && sums >= 2) return by_walk<T, TR, 256, 3>(p, n, s);
    if (n > 512 && n <= 768) return by_walk<T, TR, 384, 2>(p, n, s);
    if (n > 768 && n <= 1024) return by_walk<T, TR, 512, 1>(p, n, s);
  }
  // (many short rows: ten blocks of 128 threads on an SM, 16384 x 1792 38.1 us, with one load per thread 43.4; 2500 x 1152 9.3 / 11.1)
  if (n <= 256) return p.rows < 32 * p.num_sms ? by_blocks<T, TR, 8, 1, WINDOW, 256>(p, n, s) : by_blocks<T, TR, 8, 2, WINDOW, 128, 10>(p, n, s);
  // (five blocks of 256 threads on an SM: 16384 x 4096 with one norm 80.9 us, with four 87.4)
  if (n <= 512) return by_blocks<T, TR, 8, 2, WINDOW, 256, 5>(p, n, s);
  if (n <= 1024) return by_blocks<T, TR, 8, 2, WINDOW, 512, 2>(p, n, s);
  if (n <= 2048) return by_blocks<T, TR, 8, 2, WINDOW>(p, n, s);
  return by_blocks<T, TR, 8, 4, WINDOW>(p, n, s);
}

template <typename T, typename TR>
cudaError_t launch_as(const NormParams &p, cudaStream_t s) {
  // where a tensor's rows start in units of 16 bytes, and whether all of them have the input's place there
  constexpr long long A = 16 / sizeof(T);
  auto place = [](const void *q, size_t size) { return (long long)(reinterpret_cast<uintptr_t>(q) / size); };
  auto like_x = [&](const void *q, long long ld, size_t size) {
    const long long m = 16 / (long long)size < A ? 16 / (long long)size : A;
    return !q || ((place(q, size) - place(p.x, sizeof(T))) % m == 0 && (ld - p.ld_x) % m == 0);
  };
  const bool alike = like_x(p.res, p.ld_res, sizeof(TR)) && like_x(p.sum, p.ld_sum, sizeof(TR)) && like_x(p.y, p.ld_y, sizeof(T));
  const bool whole = p.channels % 8 == 0 && place(p.x, sizeof(T)) % A == 0 && p.ld_x % A == 0 && like_x(p.gate, p.ld_gate, sizeof(T));
  if (alike && whole) return by_vectors<T, TR, false>(p, p.channels / 8, s);
  const int windows = (p.channels + (int)A + 6) / 8;
  if (alike && windows <= 4096) return by_vectors<T, TR, true>(p, windows, s);
  // anything else one element at a time
  const int n = p.channels;
  if (n <= 32) return by_warps<T, TR, 1, 1, false>(p, s);
  if (n <= 128) return by_warps<T, TR, 1, 4, false>(p, s);
  if (n <= 512) return by_warps<T, TR, 1, 16, false>(p, s);
  if (n <= 4096) return by_blocks<T, TR, 1, 8, false, 512>(p, n, s);
  return by_blocks<T, TR, 1, 32, false>(p, n, s);
}

}  // namespace

cudaError_t launch_norm_vector(float *dst, const void *src, int et, int n, long long pitch, float offset, cudaStream_t s) {
  norm_vector_kernel<<<(unsigned)((8 * pitch + 255) / 256), 256, 0, s>>>(dst, src, et, n, pitch, offset);
  return cudaGetLastError();
}

cudaError_t launch_block_norm(const NormParams &p, cudaStream_t s) {
  if (p.et == ET_F32) return launch_as<float, float>(p, s);
  if (p.et == ET_BF16) return p.et_res == ET_F32 ? launch_as<__nv_bfloat16, float>(p, s) : launch_as<__nv_bfloat16, __nv_bfloat16>(p, s);
  return p.et_res == ET_F32 ? launch_as<__half, float>(p, s) : launch_as<__half, __half>(p, s);
}

}  // namespace elb
