// Log-probabilities of given labels, entropy and best alternatives of class scores x (batch, classes, space), and the gradient of
// the scores:
//
//   lse = log sum_c exp x_c        log_prob = x_y - lse        H = lse - sum_c p_c x_c,   p_c = exp(x_c - lse)
//   top: the largest x_c - lse, ties to the lowest class, NaN before everything
//   dx_c = a (1[c == y] - p_c) - b p_c (log p_c + H)           a, b: gradients of log_prob (0 where no label is given) and of H
//
// One pass keeps, per position, the running maximum m, l = sum exp(x - m) and u = sum (x - m) exp(x - m), all in float: with them
// lse = m + log l and H = log l - u / l, a difference that stays small whatever the scores' offset.  When the maximum moves by d,
// l and u + d l are scaled by exp(d).  A position whose scores are all -inf has log_prob -inf, entropy 0 and gradient 0.
//
// Two layouts: classes apart (NC[D]HW maps; a thread walks the classes of neighbouring positions, so that a warp reads
// consecutive ones) and classes together (rows; a warp or a CTA shares a row).
#pragma once
#include "mvr_types.cuh"

namespace mvr {

struct LogProbParams {
  const void* x;
  const void* labels;
  int label_type;        // 0 uint8, 1 int16, 2 int32, 3 int64
  float *log_prob, *entropy, *lse, *top_value;
  int* top_label;
  long long batch, space, batch_stride, class_stride;  // elements; positions of one batch item are consecutive
  int classes, top;
  // backward
  const float *grad_log_prob, *grad_entropy;           // or null
  void* grad;
  long long grad_batch_stride, grad_class_stride;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The label at a position; -1 where none is given (it is not one of the classes).
__device__ __forceinline__ int label_at(const LogProbParams& p, long long i) {
  long long v;
  switch (p.label_type) {
    case 0: v = ((const uint8_t*)p.labels)[i]; break;
    case 1: v = ((const int16_t*)p.labels)[i]; break;
    case 2: v = ((const int32_t*)p.labels)[i]; break;
    default: v = ((const int64_t*)p.labels)[i]; break;
  }
  return v >= 0 && v < p.classes ? (int)v : -1;
}

// Running (m, l, u) of one position.
struct Online {
  float m = -INFINITY, l = 0.0f, u = 0.0f;

  __device__ __forceinline__ void raise(float to) {  // to >= m, or NaN
    if (to == m) return;
    if (m == -INFINITY) {
      m = to;
      return;
    }
    const float d = m - to, r = exp2f(d * kLog2e);
    u = r == 0.0f ? 0.0f : (u + d * l) * r;
    l *= r;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {  // x <= m
    const float d = x - m, e = exp2f(d * kLog2e);
    l += e;
    u += e == 0.0f ? 0.0f : d * e;
  }
  __device__ __forceinline__ void join(const Online& o) {
    // NaN wins over everything: fmaxf would drop it
    const float to = (m != m || o.m != o.m) ? NAN : fmaxf(m, o.m);
    Online b = o;
    raise(to);
    b.raise(to);
    if (b.m == -INFINITY) return;
    l += b.l;
    u += b.u;
  }
  __device__ __forceinline__ float lse() const { return m == -INFINITY ? m : m + log2f(l) * kLn2; }
  __device__ __forceinline__ float entropy() const { return m == -INFINITY ? 0.0f : log2f(l) * kLn2 - u / l; }
};

__device__ __forceinline__ float log_prob_of(float x, const Online& o) { return x == -INFINITY ? x : (x - o.m) - log2f(o.l) * kLn2; }

// Order of the alternatives: NaN first, then the larger score; equal ones by class.
__device__ __forceinline__ bool above(float a, float b) { return a > b || (a != a && b == b); }
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) {
  return above(a, b) || (!above(b, a) && ia < ib);
}

// Sorted list of the best TOP (value, class) pairs offered so far, classes in rising order.
template <int TOP>
struct Best {
  float v[TOP > 0 ? TOP : 1];
  int c[TOP > 0 ? TOP : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < TOP; ++k) v[k] = -INFINITY, c[k] = 0x7fffffff;
  }
  __device__ __forceinline__ void offer(float x, int cls) {
    if (TOP == 0 || !before(x, cls, v[TOP > 0 ? TOP - 1 : 0], c[TOP > 0 ? TOP - 1 : 0])) return;
#pragma unroll
    for (int k = TOP - 1; k >= 0; --k) {
      const bool here = before(x, cls, v[k], c[k]);
      if (here && k + 1 < TOP) v[k + 1] = v[k], c[k + 1] = c[k];
      const bool next = k > 0 && before(x, cls, v[k > 0 ? k - 1 : 0], c[k > 0 ? k - 1 : 0]);
      if (here && !next) v[k] = x, c[k] = cls;
    }
  }
};

// ---- classes apart: positions consecutive ------------------------------------------------------------
constexpr int kApartThreads = 128;

// A thread takes V consecutive positions of one batch item and walks their classes eight at a time: the maximum of eight moves
// the sums once.
template <typename T, int V, int TOP>
__global__ void __launch_bounds__(kApartThreads) logprob_apart_fwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const long long per_item = (p.space + V - 1) / V, item = (long long)blockIdx.x * kApartThreads + threadIdx.x;
  if (item >= per_item * p.batch) return;
  const long long b = item / per_item, s = (item - b * per_item) * V;
  const T* x = (const T*)p.x + b * p.batch_stride + s;
  const int n = (int)(p.space - s < V ? p.space - s : V);
  const long long at = b * p.space + s;
  Online o[V];
  Best<TOP> best[V];
  float given[V];
  int label[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    best[k].clear();
    given[k] = 0.0f;
    label[k] = k < n ? label_at(p, at + k) : -1;
  }
  constexpr int kStep = V >= 4 ? 4 : 8;
  for (int c0 = 0; c0 < p.classes; c0 += kStep) {
    float f[kStep][V];
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      if (c0 + j < p.classes) {
        const T* q = x + (long long)(c0 + j) * p.class_stride;
        if (n == V) {
          const Vec<T, V> w = *(const Vec<T, V>*)q;
#pragma unroll
          for (int k = 0; k < V; ++k) f[j][k] = to_float(w.v[k]);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) f[j][k] = k < n ? to_float(q[k]) : 0.0f;
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[j][k] = -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float m = o[k].m;
#pragma unroll
      for (int j = 0; j < kStep; ++j) m = m != m || f[j][k] <= m ? m : f[j][k];  // NaN stays
      o[k].raise(m);
      if (m != -INFINITY) {
#pragma unroll
        for (int j = 0; j < kStep; ++j) o[k].add(f[j][k]);
      }
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        if (c0 + j < p.classes) {
          if (TOP > 0) best[k].offer(f[j][k], c0 + j);
          if (label[k] == c0 + j) given[k] = f[j][k];
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if (k >= n) break;
    p.log_prob[at + k] = label[k] < 0 ? 0.0f : log_prob_of(given[k], o[k]);
    p.entropy[at + k] = o[k].entropy();
    if (p.lse) p.lse[at + k] = o[k].lse();
#pragma unroll
    for (int t = 0; t < TOP; ++t) {
      if (t < p.top) {
        p.top_value[(b * p.top + t) * p.space + s + k] = log_prob_of(best[k].v[t], o[k]);
        p.top_label[(b * p.top + t) * p.space + s + k] = best[k].c[t];
      }
    }
  }
}

// What the gradient of one position needs beside its scores.
struct Slope {
  float lse, h, a, b;
  int label;
  __device__ __forceinline__ float at(float x, int c) const {
    const float lp = x - lse, e = exp2f(lp * kLog2e);
    const float w = e == 0.0f ? 0.0f : e * (a + b * (lp + h));  // probability 0: lp may be -inf
    const float g = (c == label ? a : 0.0f) - w;
    return lse == -INFINITY ? 0.0f : g;
  }
};
__device__ __forceinline__ Slope slope_at(const LogProbParams& p, long long i) {
  Slope s;
  s.label = label_at(p, i);
  s.lse = p.lse[i];
  s.h = p.entropy[i];
  s.a = s.label >= 0 && p.grad_log_prob ? p.grad_log_prob[i] : 0.0f;
  s.b = p.grad_entropy ? p.grad_entropy[i] : 0.0f;
  return s;
}

template <typename T, int V>
__global__ void __launch_bounds__(kApartThreads) logprob_apart_bwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const long long per_item = (p.space + V - 1) / V, item = (long long)blockIdx.x * kApartThreads + threadIdx.x;
  if (item >= per_item * p.batch) return;
  const long long b = item / per_item, s = (item - b * per_item) * V;
  const T* x = (const T*)p.x + b * p.batch_stride + s;
  T* g = (T*)p.grad + b * p.grad_batch_stride + s;
  const int n = (int)(p.space - s < V ? p.space - s : V);
  Slope q[V];
#pragma unroll
  for (int k = 0; k < V; ++k) q[k] = slope_at(p, b * p.space + s + (k < n ? k : 0));
#pragma unroll 4
  for (int c = 0; c < p.classes; ++c) {
    const T* xc = x + (long long)c * p.class_stride;
    T* gc = g + (long long)c * p.grad_class_stride;
    if (n == V) {
      const Vec<T, V> w = *(const Vec<T, V>*)xc;
      Vec<T, V> r;
#pragma unroll
      for (int k = 0; k < V; ++k) r.v[k] = from_float<T>(q[k].at(to_float(w.v[k]), c));
      *(Vec<T, V>*)gc = r;
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k < n) gc[k] = from_float<T>(q[k].at(to_float(xc[k]), c));
    }
  }
}

// ---- classes together: rows -------------------------------------------------------------------------
// LANES threads (a warp, or a CTA of 512) share a row.  The alternatives need a second look at the row: split into 32 parts, the
// top-th largest of the parts' maxima is a bound that at least `top` classes reach, and few more do (some 20 of a random row for
// top = 8); what reaches it is collected and ranked.  Where more reach it than there is room for (many equal scores), the
// alternatives are picked one by one instead.
constexpr int kWide = 512, kRoom = 256;

template <int LANES>
struct RowShared {
  static constexpr int kWarps = LANES / 32;
  float m[kWarps], l[kWarps], u[kWarps];
  float peak[32];
  float cand[kRoom];
  int cand_class[kRoom];
  int count;
  float pick_v;
  float wv[kWarps];
  int wc[kWarps];
};

template <int LANES>
__device__ __forceinline__ void row_sync() {
  if (LANES == 32) __syncwarp();
  else __syncthreads();
}

// Visits a row: f(value, class) on this thread's classes, 16-byte vectors in between for the wide form.
template <typename T, int LANES, typename F>
__device__ __forceinline__ void walk_row(const T* x, int n, int lane, F&& f) {
  if (LANES == 32) {
    for (int c = lane; c < n; c += 32) f(to_float(x[c]), c);
  } else {
    constexpr int V = 16 / (int)sizeof(T);
    const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T)), vecs = (n - head) / V;
    if (lane < head) f(to_float(x[lane]), lane);
    const Vec<T, V>* v = (const Vec<T, V>*)(x + head);
#pragma unroll 4
    for (int i = lane; i < vecs; i += LANES) {
      const Vec<T, V> w = v[i];
#pragma unroll
      for (int k = 0; k < V; ++k) f(to_float(w.v[k]), head + i * V + k);
    }
    for (int c = head + vecs * V + lane; c < n; c += LANES) f(to_float(x[c]), c);
  }
}

template <int LANES>
__device__ __forceinline__ void best_of_row(float& v, int& c, RowShared<LANES>& sh, int lane) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float ov = __shfl_xor_sync(~0u, v, d);
    const int oc = __shfl_xor_sync(~0u, c, d);
    if (before(ov, oc, v, c)) v = ov, c = oc;
  }
  if (LANES > 32) {
    if ((lane & 31) == 0) sh.wv[lane >> 5] = v, sh.wc[lane >> 5] = c;
    __syncthreads();
    v = sh.wv[0], c = sh.wc[0];
    for (int w = 1; w < LANES / 32; ++w)
      if (before(sh.wv[w], sh.wc[w], v, c)) v = sh.wv[w], c = sh.wc[w];
    __syncthreads();
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(LANES == 32 ? 128 : LANES) logprob_rows_fwd(const __grid_constant__ LogProbParams p) {
  constexpr int kRows = LANES == 32 ? 4 : 1;
  __shared__ RowShared<LANES> shared[kRows];
  grid_dependency();
  const int lane = LANES == 32 ? threadIdx.x & 31 : threadIdx.x, mine = LANES == 32 ? threadIdx.x >> 5 : 0;
  RowShared<LANES>& sh = shared[mine];
  const long long row = (long long)blockIdx.x * kRows + mine;
  if (row >= p.batch) return;
  const T* x = (const T*)p.x + row * p.batch_stride;
  const int n = p.classes;
  Online o;
  float peak = -INFINITY;  // this thread's maximum, NaN above all
  walk_row<T, LANES>(x, n, lane, [&](float v, int) {
    if (!(v <= o.m)) o.raise(v != v || o.m == o.m ? v : o.m);
    if (o.m != -INFINITY) o.add(v);
    peak = above(v, peak) ? v : peak;
  });
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    Online b;
    b.m = __shfl_xor_sync(~0u, o.m, d);
    b.l = __shfl_xor_sync(~0u, o.l, d);
    b.u = __shfl_xor_sync(~0u, o.u, d);
    // the same two operands in the same order on both lanes, so that all lanes hold the same sums
    if (lane & d) {
      b.join(o);
      o = b;
    } else {
      o.join(b);
    }
  }
  if (LANES > 32) {
    if ((lane & 31) == 0) sh.m[lane >> 5] = o.m, sh.l[lane >> 5] = o.l, sh.u[lane >> 5] = o.u;
    __syncthreads();
    o.m = sh.m[0], o.l = sh.l[0], o.u = sh.u[0];
    for (int w = 1; w < LANES / 32; ++w) {
      Online b;
      b.m = sh.m[w], b.l = sh.l[w], b.u = sh.u[w];
      o.join(b);
    }
  }
  if (lane == 0) {
    const int y = label_at(p, row);
    p.log_prob[row] = y < 0 ? 0.0f : log_prob_of(to_float(x[y]), o);
    p.entropy[row] = o.entropy();
    if (p.lse) p.lse[row] = o.lse();
    sh.count = 0;
  }
  if (p.top == 0) return;
  // the parts' maxima, and of them the one of rank top - 1 (equal ones by part); a part without classes counts as -inf
#pragma unroll
  for (int d = LANES / 64; d; d >>= 1) {
    const float other = __shfl_xor_sync(~0u, peak, d);
    peak = above(other, peak) ? other : peak;
  }
  if (lane % (LANES / 32) == 0) sh.peak[lane / (LANES / 32)] = peak;
  row_sync<LANES>();
  if (lane < 32) {
    peak = sh.peak[lane];
    int rank = 0;
    for (int i = 0; i < 32; ++i) rank += before(sh.peak[i], i, peak, lane);
    if (rank == p.top - 1) sh.pick_v = peak;
  }
  row_sync<LANES>();
  const float bound = sh.pick_v;
  walk_row<T, LANES>(x, n, lane, [&](float v, int c) {
    if (!above(bound, v)) {
      const int k = atomicAdd(&sh.count, 1);
      if (k < kRoom) sh.cand[k] = v, sh.cand_class[k] = c;
    }
  });
  row_sync<LANES>();
  const int count = sh.count;
  if (count <= kRoom) {
    for (int i = lane; i < count; i += LANES) {
      const float v = sh.cand[i];
      const int c = sh.cand_class[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += before(sh.cand[j], sh.cand_class[j], v, c);
      if (rank < p.top) {
        p.top_value[row * p.top + rank] = log_prob_of(v, o);
        p.top_label[row * p.top + rank] = c;
      }
    }
  } else {
    float last_v = 0.0f;
    int last_c = -1;
    for (int t = 0; t < p.top; ++t) {
      float v = -INFINITY;
      int c = 0x7fffffff;
      walk_row<T, LANES>(x, n, lane, [&](float w, int k) {
        if ((t == 0 || before(last_v, last_c, w, k)) && before(w, k, v, c)) v = w, c = k;
      });
      best_of_row<LANES>(v, c, sh, lane);
      if (lane == 0) {
        p.top_value[row * p.top + t] = log_prob_of(v, o);
        p.top_label[row * p.top + t] = c;
      }
      last_v = v, last_c = c;
    }
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(LANES == 32 ? 128 : LANES) logprob_rows_bwd(const __grid_constant__ LogProbParams p) {
  constexpr int kRows = LANES == 32 ? 4 : 1;
  grid_dependency();
  const int lane = LANES == 32 ? threadIdx.x & 31 : threadIdx.x, mine = LANES == 32 ? threadIdx.x >> 5 : 0;
  const long long row = (long long)blockIdx.x * kRows + mine;
  if (row >= p.batch) return;
  const T* x = (const T*)p.x + row * p.batch_stride;
  T* g = (T*)p.grad + row * p.grad_batch_stride;
  const int n = p.classes;
  const Slope q = slope_at(p, row);
  constexpr int V = 16 / (int)sizeof(T);
  // vectors where scores and gradient have the same alignment
  if (LANES > 32 && (((uintptr_t)x ^ (uintptr_t)g) & 15) == 0) {
    const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T)), vecs = (n - head) / V;
    if (lane < head) g[lane] = from_float<T>(q.at(to_float(x[lane]), lane));
#pragma unroll 4
    for (int i = lane; i < vecs; i += LANES) {
      const Vec<T, V> w = ((const Vec<T, V>*)(x + head))[i];
      Vec<T, V> r;
#pragma unroll
      for (int k = 0; k < V; ++k) r.v[k] = from_float<T>(q.at(to_float(w.v[k]), head + i * V + k));
      ((Vec<T, V>*)(g + head))[i] = r;
    }
    for (int c = head + vecs * V + lane; c < n; c += LANES) g[c] = from_float<T>(q.at(to_float(x[c]), c));
    return;
  }
  for (int c = lane; c < n; c += LANES) g[c] = from_float<T>(q.at(to_float(x[c]), c));
}

// ---- launches ----------------------------------------------------------------------------------------
// 0, or 1: more CTAs than a grid has.
template <typename T, int V>
int launch_logprob_apart(const LogProbParams& p, bool fwd, cudaStream_t st) {
  const long long items = (p.space + V - 1) / V * p.batch, ctas = (items + kApartThreads - 1) / kApartThreads;
  if (ctas > 0x7fffffffLL) return 1;
  const dim3 grid((unsigned)ctas);
  if (!fwd) launch_dependent(logprob_apart_bwd<T, V>, grid, kApartThreads, 0, st, p);
  else if (p.top == 0) launch_dependent(logprob_apart_fwd<T, V, 0>, grid, kApartThreads, 0, st, p);
  else if (p.top <= 2) launch_dependent(logprob_apart_fwd<T, V, 2>, grid, kApartThreads, 0, st, p);
  else if (p.top <= 5) launch_dependent(logprob_apart_fwd<T, 1, 5>, dim3((unsigned)((p.space * p.batch + kApartThreads - 1) / kApartThreads)), kApartThreads, 0, st, p);
  else launch_dependent(logprob_apart_fwd<T, 1, 16>, dim3((unsigned)((p.space * p.batch + kApartThreads - 1) / kApartThreads)), kApartThreads, 0, st, p);
  return 0;
}

template <typename T>
int launch_logprob(const LogProbParams& p, bool fwd, cudaStream_t st) {
  if (p.class_stride == 1 && p.space == 1) {
    if (p.classes <= 1024) {
      const long long ctas = (p.batch + 3) / 4;
      if (ctas > 0x7fffffffLL) return 1;
      if (fwd) launch_dependent(logprob_rows_fwd<T, 32>, dim3((unsigned)ctas), 128, 0, st, p);
      else launch_dependent(logprob_rows_bwd<T, 32>, dim3((unsigned)ctas), 128, 0, st, p);
    } else {
      if (p.batch > 0x7fffffffLL) return 1;
      if (fwd) launch_dependent(logprob_rows_fwd<T, kWide>, dim3((unsigned)p.batch), kWide, 0, st, p);
      else launch_dependent(logprob_rows_bwd<T, kWide>, dim3((unsigned)p.batch), kWide, 0, st, p);
    }
    return 0;
  }
  if (p.space * p.batch > 0x7fffffffLL * kApartThreads) return 1;
  constexpr int V = 8 / (int)sizeof(T);
  const long long strides = p.batch_stride | p.class_stride | (fwd ? 0 : p.grad_batch_stride | p.grad_class_stride);
  const uintptr_t at = (uintptr_t)p.x | (fwd ? 0 : (uintptr_t)p.grad);
  if (strides % V == 0 && at % 8 == 0) return launch_logprob_apart<T, V>(p, fwd, st);
  return launch_logprob_apart<T, 1>(p, fwd, st);
}

}  // namespace mvr
