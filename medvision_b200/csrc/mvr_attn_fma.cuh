// Attention products in float arithmetic: float inputs, and every shape that the tensor-core kernels do not take (head sizes that
// are no multiple of 8, operands that are not 16-byte aligned).
//
// A CTA of 16 x 16 threads holds a stationary tile of BT rows and streams tiles of BT others through shared memory, padded by four
// floats so that 16-byte reads of neighbouring rows fall on different banks.  Per tile a thread forms an (BT/16)^2 patch of
// products from two 16-byte reads for 16 multiply-adds, stores its weights, and adds them into its rows' sums.  Bound by the
// issue of the multiply-adds and of the reads that feed them: issue slots 58 to 62 % busy in the gradients of 128 x 49 rows of 8 heads
// of 32 over 2 x 4096 states.  (200 regions over three images of 13 635 states, 4 heads of 64, forward 0.12 ms, backward 0.45 to 0.53.)
// What is left to it: small float calls, where it is the faster form, float head sizes above 64, half ones above 128, and
// operands that TMA cannot read.
#pragma once
#include "mvr_attn.cuh"

namespace mvr {

constexpr int kFmaThreads = 256;

template <int DP>
struct FmaTile {
  static constexpr int BT = DP <= 128 ? 64 : 32, MT = BT / 16, CW = DP / 16, VW = CW < 4 ? CW : 4, LD = DP + 4, LP = BT + 4;
  static constexpr size_t bytes(int tiles) { return (size_t)(tiles * BT * LD + BT * LP + 3 * BT) * sizeof(float); }
};

// acc[i][j] += a_(ty MT + i) . b_(tx + 16 j)
template <int DP>
__device__ __forceinline__ void fma_dots(float (&acc)[FmaTile<DP>::MT][FmaTile<DP>::MT], const float* a, const float* b, int tx, int ty) {
  typedef FmaTile<DP> F;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 av[F::MT], bv[F::MT];
#pragma unroll
    for (int i = 0; i < F::MT; ++i) av[i] = *(const float4*)(a + (ty * F::MT + i) * F::LD + d);
#pragma unroll
    for (int j = 0; j < F::MT; ++j) bv[j] = *(const float4*)(b + (tx + 16 * j) * F::LD + d);
#pragma unroll
    for (int i = 0; i < F::MT; ++i)
#pragma unroll
      for (int j = 0; j < F::MT; ++j)
        acc[i][j] += av[i].x * bv[j].x + av[i].y * bv[j].y + av[i].z * bv[j].z + av[i].w * bv[j].w;
  }
}

// Column of a thread's c-th sum.
template <int DP>
__device__ __forceinline__ int fma_col(int c, int tx) {
  typedef FmaTile<DP> F;
  return (c / F::VW) * (16 * F::VW) + tx * F::VW + c % F::VW;
}

// acc[i][.] += sum_b w[b][ty MT + i] x[b][.]
template <int DP>
__device__ __forceinline__ void fma_add(float (&acc)[FmaTile<DP>::MT][FmaTile<DP>::CW], const float* w, const float* x, int tx, int ty) {
  typedef FmaTile<DP> F;
  typedef Vec<float, F::MT> W;
  typedef Vec<float, F::VW> X;
#pragma unroll 4
  for (int b = 0; b < F::BT; ++b) {
    const W wv = *(const W*)(w + b * F::LP + ty * F::MT);
#pragma unroll
    for (int c = 0; c < F::CW / F::VW; ++c) {
      const X xv = *(const X*)(x + b * F::LD + c * 16 * F::VW + tx * F::VW);
#pragma unroll
      for (int i = 0; i < F::MT; ++i)
#pragma unroll
        for (int e = 0; e < F::VW; ++e) acc[i][c * F::VW + e] += wv.v[i] * xv.v[e];
    }
  }
}

// w[tx + 16 j][ty MT + .] = v[.][j]
template <int DP>
__device__ __forceinline__ void fma_put(float* w, const float (&v)[FmaTile<DP>::MT][FmaTile<DP>::MT], int tx, int ty) {
  typedef FmaTile<DP> F;
#pragma unroll
  for (int j = 0; j < F::MT; ++j) {
    Vec<float, F::MT> o;
#pragma unroll
    for (int i = 0; i < F::MT; ++i) o.v[i] = v[i][j];
    *(Vec<float, F::MT>*)(w + (tx + 16 * j) * F::LP + ty * F::MT) = o;
  }
}

// States [first, first + BT) of (n, hk) as floats; those that are not allowed, and the padding, as 0.
template <typename T, int DP>
__device__ __forceinline__ void fma_load_states(float* dst, const T* src, long long stride, int first, const float* allowed, int D) {
  typedef FmaTile<DP> F;
  constexpr int U = 8;  // loads under way together; those of elements left out go to the first one
  for (int e0 = threadIdx.x; e0 < F::BT * DP; e0 += U * kFmaThreads) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kFmaThreads, j = e / DP, d = e % DP;
      const bool in = allowed[j] != 0.0f && d < D;
      const float x = to_float(src[in ? (long long)(first + j) * stride + d : 0]);
      v[u] = in ? x : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kFmaThreads;
      dst[e / DP * F::LD + e % DP] = v[u];
    }
  }
}
// Where the rows of a tile lie: offsets into queries and gradient, and row numbers (-1: no row).
template <int BT>
struct FmaRows {
  long long q[BT], g[BT], number[BT];
  __device__ __forceinline__ void find(const AttnParams& p, const RowTile& o, int first, int hk) {
    if ((int)threadIdx.x < BT) {
      const int j = first + threadIdx.x;
      number[threadIdx.x] = -1;
      if (j < o.rows) {
        const Row w = row_of(p, o, j, hk);
        q[threadIdx.x] = w.r * p.q_r + w.t * p.q_t + w.h * p.q_h;
        g[threadIdx.x] = w.r * p.g_r + w.t * p.g_t + w.h * p.g_h;
        number[threadIdx.x] = row_number(p, w);
      }
    }
  }
};
template <typename T, int DP>
__device__ __forceinline__ void fma_load_rows(float* dst, const T* src, const long long* at, const long long* number, int D) {
  typedef FmaTile<DP> F;
  constexpr int U = 8;
  for (int e0 = threadIdx.x; e0 < F::BT * DP; e0 += U * kFmaThreads) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kFmaThreads, j = e / DP, d = e % DP;
      const bool in = number[j] >= 0 && d < D;
      const float x = to_float(src[in ? at[j] + d : 0]);
      v[u] = in ? x : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kFmaThreads;
      dst[e / DP * F::LD + e % DP] = v[u];
    }
  }
}

// allowed[j] = 1 for the states of the tile that are; whether there are any (the same answer for all threads)
__device__ __forceinline__ bool fma_allowed(float* allowed, const AttnParams& p, int n, int first, int end, int size) {
  bool any = false;
  if ((int)threadIdx.x < size) {
    const int j = first + threadIdx.x;
    any = j < end && (!p.mask || p.mask[(long long)n * p.L + j]);
    allowed[threadIdx.x] = any ? 1.0f : 0.0f;
  }
  return __syncthreads_or(any);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kFmaThreads) attn_fma_fwd(const __grid_constant__ AttnParams p) {
  typedef FmaTile<DP> F;
  extern __shared__ __align__(16) float fma_smem[];
  float *qs = fma_smem, *ks = qs + F::BT * F::LD, *vs = ks + F::BT * F::LD, *ws = vs + F::BT * F::LD, *allowed = ws + F::BT * F::LP;
  grid_dependency();
  RowTile o;
  if (!row_tile(p, blockIdx.x, F::BT, o)) return;
  const int hk = blockIdx.y, split = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int tiles = (p.L + F::BT - 1) / F::BT, per = (tiles + p.splits - 1) / p.splits;
  const int begin = split * per * F::BT, end = min(states_of(p, o.n), (split + 1) * per * F::BT);
  __shared__ FmaRows<F::BT> at;
  at.find(p, o, o.first, hk);
  __syncthreads();
  fma_load_rows<T, DP>(qs, (const T*)p.q, at.q, at.number, p.D);
  const T* k = (const T*)p.k + (long long)o.n * p.k_n + (long long)hk * p.k_h;
  const T* v = (const T*)p.v + (long long)o.n * p.v_n + (long long)hk * p.v_h;
  float acc[F::MT][F::CW] = {}, m[F::MT], l[F::MT] = {};
#pragma unroll
  for (int i = 0; i < F::MT; ++i) m[i] = -INFINITY;
  for (int j0 = begin; j0 < end; j0 += F::BT) {
    // (the barrier inside also ends the last tile's reads)
    if (!fma_allowed(allowed, p, o.n, j0, end, F::BT)) continue;
    fma_load_states<T, DP>(ks, k, p.k_l, j0, allowed, p.D);
    fma_load_states<T, DP>(vs, v, p.v_l, j0, allowed, p.D);
    __syncthreads();
    float s[F::MT][F::MT] = {};
    fma_dots<DP>(s, qs, ks, tx, ty);
#pragma unroll
    for (int i = 0; i < F::MT; ++i) {
      float top = m[i];
#pragma unroll
      for (int j = 0; j < F::MT; ++j) {
        s[i][j] = allowed[tx + 16 * j] != 0.0f ? s[i][j] * p.scale_log2 : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      const float ref = top == -INFINITY ? 0.0f : top, shrink = exp2f(m[i] - ref);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < F::MT; ++j) {
        s[i][j] = exp2f(s[i][j] - ref);
        sum += s[i][j];
      }
      l[i] = l[i] * shrink + sum;
      m[i] = top;
#pragma unroll
      for (int c = 0; c < F::CW; ++c) acc[i][c] *= shrink;
    }
    fma_put<DP>(ws, s, tx, ty);
    __syncthreads();
    fma_add<DP>(acc, ws, vs, tx, ty);
    __syncthreads();
  }
  const long long rows = (long long)p.R * p.T * p.Hq;
#pragma unroll
  for (int i = 0; i < F::MT; ++i) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) l[i] += __shfl_xor_sync(~0u, l[i], d);
    const long long row = at.number[ty * F::MT + i];
    if (row < 0) continue;
    const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
    for (int c = 0; c < F::CW; ++c) {
      const int d = fma_col<DP>(c, tx);
      if (d >= p.D) continue;
      if (p.splits > 1) p.part_o[(split * rows + row) * p.D + d] = acc[i][c];
      else ((T*)p.out)[row * p.D + d] = from_float<T>(acc[i][c] * inv);
    }
    if (tx == 0) {
      if (p.splits > 1) {
        p.part_ml[(split * rows + row) * 2] = m[i];
        p.part_ml[(split * rows + row) * 2 + 1] = l[i];
      } else if (p.lse) {
        p.lse[row] = l[i] == 0.0f ? -INFINITY : (m[i] == -INFINITY ? 0.0f : m[i]) + log2f(l[i]);
      }
    }
  }
}

// Gradient of the queries: a tile of rows against the states of its image.
template <typename T, int DP>
__global__ void __launch_bounds__(kFmaThreads) attn_fma_dq(const __grid_constant__ AttnParams p) {
  typedef FmaTile<DP> F;
  extern __shared__ __align__(16) float fma_smem[];
  float *qs = fma_smem, *gs = qs + F::BT * F::LD, *ks = gs + F::BT * F::LD, *vs = ks + F::BT * F::LD, *ws = vs + F::BT * F::LD,
        *allowed = ws + F::BT * F::LP;
  grid_dependency();
  RowTile o;
  if (!row_tile(p, blockIdx.x, F::BT, o)) return;
  const int hk = blockIdx.y, split = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int tiles = (p.L + F::BT - 1) / F::BT, per = (tiles + p.splits - 1) / p.splits;
  const int begin = split * per * F::BT, end = min(states_of(p, o.n), (split + 1) * per * F::BT);
  __shared__ FmaRows<F::BT> at;
  at.find(p, o, o.first, hk);
  __syncthreads();
  fma_load_rows<T, DP>(qs, (const T*)p.q, at.q, at.number, p.D);
  fma_load_rows<T, DP>(gs, (const T*)p.g, at.g, at.number, p.D);
  const T* k = (const T*)p.k + (long long)o.n * p.k_n + (long long)hk * p.k_h;
  const T* v = (const T*)p.v + (long long)o.n * p.v_n + (long long)hk * p.v_h;
  float acc[F::MT][F::CW] = {}, lse[F::MT], delta[F::MT];
#pragma unroll
  for (int i = 0; i < F::MT; ++i) {
    const long long row = at.number[ty * F::MT + i];
    lse[i] = row < 0 ? -INFINITY : p.lse[row];
    delta[i] = row < 0 ? 0.0f : p.delta[row];
  }
  for (int j0 = begin; j0 < end; j0 += F::BT) {
    if (!fma_allowed(allowed, p, o.n, j0, end, F::BT)) continue;
    fma_load_states<T, DP>(ks, k, p.k_l, j0, allowed, p.D);
    fma_load_states<T, DP>(vs, v, p.v_l, j0, allowed, p.D);
    __syncthreads();
    float s[F::MT][F::MT] = {}, dp[F::MT][F::MT] = {};
    fma_dots<DP>(s, qs, ks, tx, ty);
    fma_dots<DP>(dp, gs, vs, tx, ty);
#pragma unroll
    for (int i = 0; i < F::MT; ++i)
#pragma unroll
      for (int j = 0; j < F::MT; ++j) {
        const bool in = allowed[tx + 16 * j] != 0.0f && lse[i] != -INFINITY;
        s[i][j] = in ? exp2f(s[i][j] * p.scale_log2 - lse[i]) * (dp[i][j] - delta[i]) : 0.0f;
      }
    fma_put<DP>(ws, s, tx, ty);
    __syncthreads();
    fma_add<DP>(acc, ws, ks, tx, ty);
    __syncthreads();
  }
  const long long rows = (long long)p.R * p.T * p.Hq;
#pragma unroll
  for (int i = 0; i < F::MT; ++i) {
    const long long row = at.number[ty * F::MT + i];
    if (row < 0) continue;
#pragma unroll
    for (int c = 0; c < F::CW; ++c) {
      const int d = fma_col<DP>(c, tx);
      if (d >= p.D) continue;
      if (p.splits > 1) p.part_gq[(split * rows + row) * p.D + d] = acc[i][c];
      else ((T*)p.gq)[row * p.D + d] = from_float<T>(acc[i][c] * p.scale);
    }
  }
}

// Gradients of keys and values: a tile of states against the rows that read its image.
template <typename T, int DP>
__global__ void __launch_bounds__(kFmaThreads) attn_fma_dkv(const __grid_constant__ AttnParams p) {
  typedef FmaTile<DP> F;
  extern __shared__ __align__(16) float fma_smem[];
  float *ks = fma_smem, *vs = ks + F::BT * F::LD, *qs = vs + F::BT * F::LD, *gs = qs + F::BT * F::LD, *ws = gs + F::BT * F::LD,
        *allowed = ws + F::BT * F::LP, *lse = allowed + F::BT, *delta = lse + F::BT;
  grid_dependency();
  const int tiles = (p.L + F::BT - 1) / F::BT, n = blockIdx.x / tiles, j0 = (blockIdx.x - n * tiles) * F::BT;
  const int hk = blockIdx.y, split = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  __shared__ FmaRows<F::BT> at;
  const RowTile o = image_rows(p, n);
  const int row_tiles = (o.rows + F::BT - 1) / F::BT, per = (row_tiles + p.row_splits - 1) / p.row_splits;
  const bool any = fma_allowed(allowed, p, n, j0, states_of(p, n), F::BT);
  const int first = any ? split * per * F::BT : 0, last = any ? min(o.rows, (split + 1) * per * F::BT) : 0;
  float dk[F::MT][F::CW] = {}, dv[F::MT][F::CW] = {};
  if (first < last) {
    fma_load_states<T, DP>(ks, (const T*)p.k + (long long)n * p.k_n + (long long)hk * p.k_h, p.k_l, j0, allowed, p.D);
    fma_load_states<T, DP>(vs, (const T*)p.v + (long long)n * p.v_n + (long long)hk * p.v_h, p.v_l, j0, allowed, p.D);
  }
  for (int r0 = first; r0 < last; r0 += F::BT) {
    at.find(p, o, r0, hk);
    __syncthreads();
    fma_load_rows<T, DP>(qs, (const T*)p.q, at.q, at.number, p.D);
    fma_load_rows<T, DP>(gs, (const T*)p.g, at.g, at.number, p.D);
    if ((int)threadIdx.x < F::BT) {
      const long long row = at.number[threadIdx.x];
      lse[threadIdx.x] = row < 0 ? -INFINITY : p.lse[row];
      delta[threadIdx.x] = row < 0 ? 0.0f : p.delta[row];
    }
    __syncthreads();
    float s[F::MT][F::MT] = {}, dp[F::MT][F::MT] = {};
    fma_dots<DP>(s, ks, qs, tx, ty);
    fma_dots<DP>(dp, vs, gs, tx, ty);
#pragma unroll
    for (int i = 0; i < F::MT; ++i)
#pragma unroll
      for (int j = 0; j < F::MT; ++j) {
        const float a = lse[tx + 16 * j];
        const bool in = allowed[ty * F::MT + i] != 0.0f && a != -INFINITY;
        s[i][j] = in ? exp2f(s[i][j] * p.scale_log2 - a) : 0.0f;
        dp[i][j] = in ? s[i][j] * (dp[i][j] - delta[tx + 16 * j]) : 0.0f;
      }
    fma_put<DP>(ws, s, tx, ty);
    __syncthreads();
    fma_add<DP>(dv, ws, gs, tx, ty);
    __syncthreads();
    fma_put<DP>(ws, dp, tx, ty);
    __syncthreads();
    fma_add<DP>(dk, ws, qs, tx, ty);
    __syncthreads();
  }
  const long long all = (long long)p.N * p.L * p.Hk * p.D;
#pragma unroll
  for (int i = 0; i < F::MT; ++i) {
    const int j = j0 + ty * F::MT + i;
    if (j >= p.L) continue;
    const long long to = (((long long)n * p.L + j) * p.Hk + hk) * p.D;
    const bool in = allowed[ty * F::MT + i] != 0.0f;  // others: 0, also where rows hold NaN
#pragma unroll
    for (int c = 0; c < F::CW; ++c) {
      const int d = fma_col<DP>(c, tx);
      if (d >= p.D) continue;
      const float a = in ? dk[i][c] : 0.0f, b = in ? dv[i][c] : 0.0f;
      if (p.row_splits > 1) {
        p.part_gk[split * all + to + d] = a;
        p.part_gv[split * all + to + d] = b;
      } else {
        ((T*)p.gk)[to + d] = from_float<T>(a * p.scale);
        ((T*)p.gv)[to + d] = from_float<T>(b);
      }
    }
  }
}

}  // namespace mvr
