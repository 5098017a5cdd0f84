// Attention of queries to an encoder's states of another length: parameters, the grouping of regions by image, and the small
// kernels around the products (mvr_attn_fma.cuh: float arithmetic, every case; mvr_attn_tc.cuh: tensor cores).
//
//   s_j = scale q.k_j    p_j = exp(s_j - lse)    lse = log sum_j exp s_j    o = sum_j p_j v_j          over the states j allowed
//   delta = g.o    ds_j = p_j (g.v_j - delta)    dq = scale sum_j ds_j k_j    dk_j = scale sum ds_j q    dv_j = sum p_j g
//
// A query without allowed states gives 0, and 0 gradients.  States that are not allowed are never computed with: what they hold
// (NaN, infinities) has no effect.
//
// Rows.  A region r has T tokens with Hq heads; head h reads key head h / G.  The rows of a key head of an image are its regions'
// tokens with the G heads that share the key head, so that a tile of rows reads the states once for all of them.  With an index the
// regions are grouped by image first, in their order (attn_plan): `order` lists them image by image, `starts` says where each
// image's begin, and a last group holds those whose image is not in [0, N): no states, zero results.
#pragma once
#include "mvr_types.cuh"

namespace mvr {

// Division of numbers below 2^31 by a constant of the launch: a product and a shift.
struct Divisor {
  unsigned d, factor, shift;
  void set(unsigned divisor) {
    d = divisor;
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    factor = (unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int quotient(int n) const { return (int)((__umulhi((unsigned)n, factor) + (unsigned)n) >> shift); }
};

struct AttnParams {
  const void *q, *k, *v, *g;                     // g: gradient of the output (backward)
  void *out, *gq, *gk, *gv;                      // out, gq: (R, T, Hq, D); gk, gv: (N, L, Hk, D); all contiguous
  const void* o;                                 // the forward's output (backward)
  float *lse, *delta;                            // (R, T, Hq); lse in powers of two: log2 of the sum of 2^(s log2 e)
  float* norm;                                   // (R, T, Hq): |g| (float16 gradients)
  int* peaks;                                    // (N, Hk): largest |v| of the states that are read, float bits (float16 gradients)
  float2* row_peaks;                             // (tile of 128 rows, Hk): largest |g| and |delta| (float16 gradients)
  long long q_r, q_t, q_h, g_r, g_t, g_h;        // strides in elements; the last dimension is contiguous
  long long k_n, k_l, k_h, v_n, v_l, v_h;
  const int *order, *starts, *tiles;             // grouping by image, or null: region r reads image r
  const void* index;                             // set: no grouping; tile t is all rows of image t, found from the index (forward)
  int index_type;
  long long index_stride;
  const void* lengths;                           // (N) int32 or int64, or null
  int lengths64;
  const unsigned char* mask;                     // (N, L) or null
  int R, T, Hq, Hk, G, N, L, D;
  int W;                                         // columns of the operands in memory: D, or with pieces D rounded up to 8
  long long q_piece, g_piece;                    // elements from one piece of the queries (gradient) to the next
  Divisor by_T, by_G;
  float scale, scale_log2;
  int splits;                                    // parts of the states (forward, dq) or of the rows (dk, dv)
  float *part_o, *part_ml;                       // splits > 1: (split, row, D) and (split, row, 2)
  float *part_gq, *part_gk, *part_gv;            // splits > 1: (split, row, D), (split, N, L, Hk, D)
  int row_splits;
};

// Rows of a tile: image n (N: none), its regions, and where the tile begins among the rows of one key head.
struct RowTile {
  int n, first, rows;  // first row of the tile within the image, number of rows of the image (per key head)
  const int* order;    // regions of the image, or null: the image's own number
};

// Tile `t` of the rows, `size` rows each; false: there is none.
__device__ __forceinline__ bool row_tile(const AttnParams& p, int t, int size, RowTile& o) {
  const int per = p.T * p.G;
  if (!p.order) {
    const int tiles = (per + size - 1) / size;
    o.n = t / tiles;
    if (o.n >= p.N) return false;
    o.first = (t - o.n * tiles) * size;
    o.rows = per;
    o.order = nullptr;
    return true;
  }
  // tiles[n]: number of tiles of the images before n, n <= N + 1
  int lo = 0, hi = p.N + 1;
  if (t >= p.tiles[hi]) return false;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.tiles[mid] <= t) lo = mid;
    else hi = mid;
  }
  o.n = lo;
  o.first = (t - p.tiles[lo]) * size;
  o.rows = (p.starts[lo + 1] - p.starts[lo]) * per;
  o.order = p.order + p.starts[lo];
  return true;
}
__device__ __forceinline__ RowTile image_rows(const AttnParams& p, int n) {
  RowTile o;
  o.n = n;
  o.first = 0;
  o.rows = (p.order ? p.starts[n + 1] - p.starts[n] : 1) * p.T * p.G;
  o.order = p.order ? p.order + p.starts[n] : nullptr;
  return o;
}

// Region, token and query head of row j of an image's key head.
struct Row {
  int r, t, h;
};
__device__ __forceinline__ Row row_of(const AttnParams& p, const RowTile& o, int j, int hk) {
  const int token = p.by_G.quotient(j);
  Row w;
  w.h = hk * p.G + (j - token * p.G);
  const int slot = p.by_T.quotient(token);
  w.t = token - slot * p.T;
  w.r = o.order ? o.order[slot] : o.n;
  return w;
}
__device__ __forceinline__ long long row_number(const AttnParams& p, const Row& w) {
  return ((long long)w.r * p.T + w.t) * p.Hq + w.h;
}

// States of image n that may be read: [0, n_states); the mask says which of them are.
__device__ __forceinline__ int states_of(const AttnParams& p, int n) {
  if (n >= p.N) return 0;
  if (!p.lengths) return p.L;
  const long long l = p.lengths64 ? ((const long long*)p.lengths)[n] : ((const int*)p.lengths)[n];
  return l < 0 ? 0 : l < p.L ? (int)l : p.L;
}

// ---- grouping of regions by image ---------------------------------------------------------------------
// A stable counting sort by one CTA: each warp counts the images of a consecutive part of the regions, the counts are summed over
// images and warps, and each warp places its part in order.  `tiles`: running number of tiles of `tile` rows per image.
// Index types: 0 float, 1 half, 2 double, 3 bfloat16, 4 int32, 5 int64, 6 int16, 7 uint8; a floating index is cut towards zero, as
// the roi kernels read it.
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int image_index(const void* index, int type, long long stride, int r, int N) {
  const long long at = (long long)r * stride;
  double f;
  switch (type) {
    case 0: f = ((const float*)index)[at]; break;
    case 1: f = __half2float(((const __half*)index)[at]); break;
    case 2: f = ((const double*)index)[at]; break;
    case 3: f = __bfloat162float(((const __nv_bfloat16*)index)[at]); break;
    case 4: f = ((const int*)index)[at]; break;
    case 5: {
      const long long v = ((const long long*)index)[at];
      return v >= 0 && v < N ? (int)v : N;
    }
    case 6: f = ((const short*)index)[at]; break;
    default: f = ((const unsigned char*)index)[at]; break;
  }
  return f > -1.0 && f < (double)N ? (int)f : N;  // NaN: none
}

// counts: shared memory, (warps + 1) * (N + 1) ints
__global__ void __launch_bounds__(kPlanThreads)
attn_plan(const void* index, int type, long long stride, int R, int N, int rows_per_region, int tile, int warps, int* order,
          int* starts, int* tiles, int* status) {
  extern __shared__ int counts[];
  __shared__ int carry[2], part[2][32];
  grid_dependency();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, groups = N + 1;
  for (int i = threadIdx.x; i < warps * groups; i += kPlanThreads) counts[i] = 0;
  if (threadIdx.x == 0) carry[0] = carry[1] = 0;
  __syncthreads();
  const int per = ((R + warps - 1) / warps + 31) & ~31, lo = min(R, w * per), hi = min(R, lo + per);
  if (w < warps) {
    bool bad = false;
    for (int r = lo + lane; r < hi; r += 32) {
      const int n = image_index(index, type, stride, r, N);
      bad |= n == N;
      atomicAdd(&counts[w * groups + n], 1);
    }
    if (bad && status) atomicOr(status, 1);
  }
  __syncthreads();
  // per image: running sum over the warps, then over the images, 1024 images at a time
  for (int base = 0; base < groups; base += kPlanThreads) {
    const int n = base + threadIdx.x;
    int total = 0;
    if (n < groups)
      for (int i = 0; i < warps; ++i) {
        const int c = counts[i * groups + n];
        counts[i * groups + n] = total;
        total += c;
      }
    int sum = total, sumt = n < groups ? (int)(((long long)total * rows_per_region + tile - 1) / tile) : 0;
    const int mine = sum, minet = sumt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int a = __shfl_up_sync(~0u, sum, d), b = __shfl_up_sync(~0u, sumt, d);
      if (lane >= d) sum += a, sumt += b;
    }
    if (lane == 31) part[0][w] = sum, part[1][w] = sumt;
    __syncthreads();
    int before = carry[0], beforet = carry[1];
    for (int i = 0; i < w; ++i) before += part[0][i], beforet += part[1][i];
    before += sum - mine;
    beforet += sumt - minet;
    if (n < groups) {
      starts[n] = before;
      tiles[n] = beforet;
      for (int i = 0; i < warps; ++i) counts[i * groups + n] += before;
      if (n == groups - 1) starts[groups] = before + mine, tiles[groups] = beforet + minet;
    }
    __syncthreads();
    if (threadIdx.x == kPlanThreads - 1) carry[0] = before + mine, carry[1] = beforet + minet;
    __syncthreads();
  }
  if (w < warps) {
    for (int base = lo; base < hi; base += 32) {
      const int r = base + lane;
      const int n = r < hi ? image_index(index, type, stride, r, N) : -1;
      const unsigned same = __match_any_sync(~0u, n);
      const int rank = __popc(same & ((1u << lane) - 1));
      int at = 0;
      if (n >= 0) at = counts[w * groups + n] + rank;
      __syncwarp();
      if (n >= 0) {
        order[at] = r;
        if (rank == 0) counts[w * groups + n] += __popc(same);
      }
      __syncwarp();
    }
  }
}

// ---- joining of parts ---------------------------------------------------------------------------------
// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s of the parts' maxima, sums and unscaled outputs.  A thread takes W columns of
// a row.
template <typename T, int W>
__global__ void __launch_bounds__(256) attn_join(const __grid_constant__ AttnParams p) {
  grid_dependency();
  const long long rows = (long long)p.R * p.T * p.Hq, at = (long long)blockIdx.x * 256 + threadIdx.x, row = at / (p.D / W);
  const int d = (int)(at - row * (p.D / W)) * W;
  if (row >= rows) return;
  const float2* ml = (const float2*)p.part_ml + row;
  float m = -INFINITY, l = 0.0f, o[W] = {};
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[s * rows].x);
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 v = ml[s * rows];
    const float w = exp2f(v.x - ref);
    const Vec<float, W> part = *(const Vec<float, W>*)(p.part_o + (s * rows + row) * p.D + d);
    l += w * v.y;
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] += w * part.v[i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  Vec<T, W> out;
#pragma unroll
  for (int i = 0; i < W; ++i) out.v[i] = from_float<T>(o[i] * inv);
  *(Vec<T, W>*)((T*)p.out + row * p.D + d) = out;
  if (p.lse && d == 0) p.lse[row] = l == 0.0f ? -INFINITY : ref + log2f(l);
}

// dst[i] = factor * sum over the parts, in order.  A thread takes W elements at a time.
template <typename T, int W>
__global__ void __launch_bounds__(256) attn_sum(const float* part, T* dst, long long n, int parts, float factor) {
  grid_dependency();
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * W; i < n; i += (long long)gridDim.x * 256 * W) {
    float v[W] = {};
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
      const Vec<float, W> x = *(const Vec<float, W>*)(part + s * n + i);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += x.v[k];
    }
    Vec<T, W> out;
#pragma unroll
    for (int k = 0; k < W; ++k) out.v[k] = from_float<T>(v[k] * factor);
    *(Vec<T, W>*)(dst + i) = out;
  }
}

// delta = g.o per row.  One warp a row.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta(const __grid_constant__ AttnParams p) {
  grid_dependency();
  const long long rows = (long long)p.R * p.T * p.Hq, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int h = (int)(row % p.Hq);
  const long long rt = row / p.Hq;
  const int t = (int)(rt % p.T);
  const long long r = rt / p.T;
  const T* g = (const T*)p.g + r * p.g_r + t * p.g_t + h * p.g_h;
  const T* o = (const T*)p.o + row * p.D;
  float v = 0.0f;
  for (int d = lane; d < p.D; d += 32) v += to_float(g[d]) * to_float(o[d]);
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  if (lane == 0) p.delta[row] = v;
}

}  // namespace mvr
