// Log-probabilities of given labels, entropy and best alternatives of class scores x (batch, classes, space), and the gradient of
// the scores:
//
//   lse = log sum_c exp x_c        log_prob = x_y - lse        H = lse - sum_c p_c x_c,   p_c = exp(x_c - lse)
//   top: the largest x_c - lse, ties to the lowest class, NaN before everything
//   dx_c = a (1[c == y] - p_c) - b p_c (log p_c + H)           a, b: gradients of log_prob (0 where no label is given) and of H
//
// With the maximum m, l = sum exp(x - m) and u = sum (x - m) exp(x - m), all in float: lse = m + log l, and H = log l - u / l, a
// difference that stays small whatever the scores' offset.  The logarithm is the accurate one, once a position: near certainty l = 1 + r,
// and a loss of r is off by half a step of 1 (2^-24) and no more, where the fast one would add 1.7e-7.  Where the scores do not fit the
// registers they are walked once with a running maximum: when it moves by d, l and u + d l are scaled by exp(d).  A position whose
// scores are all -inf has log_prob -inf, entropy 0 and gradient 0.
//
// The gradient forms log p_c = x_c - lse - rest, where rest is what the rounding of lse to a float left: half a step of lse, which far
// from 0 is no small change of a probability (0.02 % at 8192, 3 % at 10^6).  The forward writes both; where the caller has kept lse alone,
// the rest is log sum exp(x - lse), one more walk over the scores.
//
// Two layouts: classes apart (NC[D]HW maps; a thread walks the classes of neighbouring positions, so that a warp reads
// consecutive ones) and classes together (rows; a warp or a CTA shares a row).  Up to 16 classes apart, 1024 classes of a warp's row
// and 65536 half (32768 float) classes of a CTA's row are read once, all loads under way together, and kept: in registers, but
// that half scores apart have 64 of them a thread, so that eight CTAs fit an SM, and 9 to 16 classes up to 17 words more.  The scores are
// read once by each direction, the gradient written once.
//
// Measured: 2 x 14 x 96^3 half scores with two alternatives 41 us, gradient 36 us (issue slots 61 and 53 % busy: the alternatives, the
// exponentials and the conversions of 24.8 M scores beside the memory's 16 us); 2000 rows of 32 001 bfloat16 scores with eight
// alternatives 58 us (issue 43 %, waits between the row's phases), gradient 50 us (5.1 TB/s); 16 rows of 81 float scores 6 us.
#pragma once
#include "mvr_types.cuh"

namespace mvr {

struct LogProbParams {
  const void* x;
  const void* labels;
  int label_type;        // 0 uint8, 1 int16, 2 int32, 3 int64
  float *log_prob, *entropy, *lse, *lse_rest, *top_value;  // lse + lse_rest: log sum exp; either may be null
  int* top_label;
  long long batch, space, batch_stride, class_stride;  // elements; positions of one batch item are consecutive
  int classes, top;
  // backward
  const float *grad_log_prob, *grad_entropy;           // or null
  void* grad;
  long long first;                                     // classes apart: first position of the launch, and how many
  int positions;
  long long grad_batch_stride, grad_class_stride;
};

constexpr float kLog2e = 1.4426950408889634f;

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

// 2^x to some 2^-22, relatively; 0 below 2^-126.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
    // (a score of -inf adds 0 to both: its distance is kept finite)
    const float d = x - m, e = exp2_approx(d * kLog2e);
    l += e;
    u = fmaf(fmaxf(d, -1e30f), e, u);
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
};

// What the sums of one position come to: its maximum and log l.
struct Position {
  float m, g;
  __device__ __forceinline__ explicit Position(const Online& o) : m(o.m), g(logf(o.l)) {}
  __device__ __forceinline__ float log_prob(float x) const { return m == -INFINITY ? m : (x - m) - g; }
  // log_prob of the label's score, entropy, and lse = m + g as its float and what that leaves of it
  __device__ __forceinline__ void put(const LogProbParams& p, long long i, const Online& o, int label, float given) const {
    p.log_prob[i] = label < 0 ? 0.0f : log_prob(given);
    p.entropy[i] = m == -INFINITY ? 0.0f : g - o.u / o.l;
    const float sum = m + g, of_g = sum - m;
    if (p.lse) p.lse[i] = m == -INFINITY ? m : sum;
    if (p.lse_rest) p.lse_rest[i] = m == -INFINITY ? 0.0f : (m - (sum - of_g)) + (g - of_g);
  }
};

// (l, u) of pairs of scores about fixed maxima.
struct Sums2 {
  float2 l = make_float2(0.0f, 0.0f), u = make_float2(0.0f, 0.0f);
  __device__ __forceinline__ void add(float2 x, float2 minus_m) {
    // (a score of -inf adds 0 to both: its distance is kept finite)
    const float2 d = add2(x, minus_m), t = mul2(d, make_float2(kLog2e, kLog2e));
    const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
    l = add2(l, e);
    u = fma2(make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), e, u);
  }
};

// Order of the alternatives: NaN first, then the larger score; equal ones by class.
__device__ __forceinline__ bool above(float a, float b) { return a > b || (a != a && b == b); }
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) {
  return above(a, b) || (!above(b, a) && ia < ib);
}

// The alternatives of a position whose scores are NaN, infinite or too few for the fast way, one by one.
template <typename T>
__device__ __forceinline__ void pick_apart(const T* x, long long stride, int classes, int top, long long space, float* value, int* label,
                                        Position q) {
  float last_v = 0.0f;
  int last_c = -1;
  for (int t = 0; t < top; ++t) {
    float v = -INFINITY;
    int c = 0x7fffffff;
    for (int k = 0; k < classes; ++k) {
      const float f = to_float(x[k * stride]);
      if ((t == 0 || before(last_v, last_c, f, k)) && before(f, k, v, c)) v = f, c = k;
    }
    value[t * space] = q.log_prob(v);
    label[t * space] = c;
    last_v = v, last_c = c;
  }
}

// ---- classes apart: positions consecutive ------------------------------------------------------------
constexpr int kApartThreads = 128, kApartItems = 32768;  // batch items of a grid's second dimension

// Sorted list of the best TOP scores, offered by rising class: an equal score comes behind.  (NaN is left to pick_apart.)
template <int TOP>
struct Best {
  float v[TOP];
  int c[TOP];
  __device__ __forceinline__ Best() {
#pragma unroll
    for (int k = 0; k < TOP; ++k) v[k] = -INFINITY, c[k] = -1;
  }
  __device__ __forceinline__ void offer(float x, int cls) {
    if (TOP > 2 && !(x > v[TOP - 1])) return;
#pragma unroll
    for (int k = TOP - 1; k > 0; --k) {
      const bool above_k = x > v[k], above_next = x > v[k - 1];
      v[k] = above_next ? v[k - 1] : above_k ? x : v[k];
      c[k] = above_next ? c[k - 1] : above_k ? cls : c[k];
    }
    c[0] = x > v[0] ? cls : c[0];
    v[0] = fmaxf(v[0], x);
  }
};
template <>
struct Best<0> {
  __device__ __forceinline__ void offer(float, int) {}
};

// A thread takes two consecutive positions of one batch item (PAIR: they are loaded and stored together).  Batch item and class are
// the CTA's, the position is the thread's and has 32 bits, so that an access costs no arithmetic on addresses: with 64 bits of each
// they were two thirds of the instructions.  CACHE: number of classes that stay in registers (0: eight at a time, the maximum of eight
// moves the sums once).
template <typename T, bool PAIR, int TOP, int CACHE>
__global__ void __launch_bounds__(kApartThreads, TOP <= 2 && sizeof(T) == 2 ? 8 : 4) logprob_apart_fwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const unsigned s = (blockIdx.x * kApartThreads + threadIdx.x) * 2;
  const long long b = blockIdx.y + (long long)blockIdx.z * kApartItems;
  if (s >= (unsigned)p.positions || b >= p.batch) return;
  const T* items = (const T*)p.x + b * p.batch_stride + p.first;
  const bool second = s + 1 < (unsigned)p.positions;
  const long long at = b * p.space + p.first;
  constexpr int kStep = CACHE > 0 ? CACHE : 8;
  const int label[2] = {label_at(p, at + s), second ? label_at(p, at + s + 1) : -1};
  float given[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) given[k] = label[k] >= 0 ? to_float(items[(long long)label[k] * p.class_stride + s + k]) : 0.0f;
  Online o[2];
  Best<TOP> best[2];
  for (int c0 = 0; c0 < p.classes; c0 += kStep) {
    Two<T> w[kStep];
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      w[j] = both<T>(-INFINITY);  // classes that are not there
      if (c0 + j < p.classes) {
        const T* q = items + (long long)(c0 + j) * p.class_stride;
        if (PAIR) w[j] = *(const Two<T>*)(q + s);
        else w[j] = rounded<T>(make_float2(to_float(q[s]), second ? to_float(q[s + 1]) : 0.0f));
      }
    }
    Two<T> most = w[0];
#pragma unroll
    for (int j = 1; j < kStep; ++j) most = larger(most, w[j]);
    const float2 m2 = floats(most);
    float m[2] = {fmaxf(m2.x, o[0].m), fmaxf(m2.y, o[1].m)};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (CACHE == 0 && m[k] != o[k].m) o[k].raise(m[k]);
      o[k].m = m[k];
    }
    // (nothing but -inf so far: about 0, which leaves the sums 0, or makes them NaN where there is one)
    const float2 minus = make_float2(m[0] == -INFINITY ? 0.0f : -m[0], m[1] == -INFINITY ? 0.0f : -m[1]);
    Sums2 sum;
#pragma unroll
    for (int j = 0; j < kStep; ++j) sum.add(floats(w[j]), minus);
    o[0].l += sum.l.x, o[1].l += sum.l.y;
    o[0].u += sum.u.x, o[1].u += sum.u.y;
    if constexpr (TOP > 0) {
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        const float2 f = floats(w[j]);
        best[0].offer(f.x, c0 + j);
        best[1].offer(f.y, c0 + j);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (o[k].l != o[k].l) o[k].m = NAN;
  const Position q[2] = {Position(o[0]), Position(o[1])};
  float* value = TOP > 0 ? p.top_value + b * p.top * p.space + p.first + s : nullptr;
  int* best_label = TOP > 0 ? p.top_label + b * p.top * p.space + p.first + s : nullptr;
  unsigned apart = 0;  // a bit for each position whose alternatives are left to pick_apart
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 1 && !second) break;
    if constexpr (TOP > 0) {
      bool all = o[k].l == o[k].l;
#pragma unroll
      for (int t = 0; t < TOP; ++t) all = all && (t >= p.top || best[k].c[t] >= 0);
      if (all) {
#pragma unroll
        for (int t = 0; t < TOP; ++t)
          if (t < p.top) (value + t * p.space)[k] = q[k].log_prob(best[k].v[t]), (best_label + t * p.space)[k] = best[k].c[t];
      } else {
        apart |= 1u << k;
      }
    }
    q[k].put(p, at + s + k, o[k], label[k], given[k]);
  }
  if constexpr (TOP > 0) {
    // (At the end and in place, once for both.  As a function that was called between the two, it cost the kernels spills, and those
    // of more than two alternatives ended in accesses outside of memory that no line of it makes.)
#pragma unroll 1
    for (int k = 0; k < 2; ++k)
      if ((apart >> k) & 1) pick_apart(items + s + k, p.class_stride, p.classes, p.top, p.space, value + k, best_label + k, k ? q[1] : q[0]);
  }
}

// What the gradient of one position needs beside its scores: g_c = -e (a + b (lp + H)), lp = x - lse - rest, e = exp lp; a more at the
// label.  With d = x - lse the rest goes into two constants: e = 2^(d log2 e + shift), and k + b d with k = a + b (H - rest).
struct Slope {
  float lse, shift, a, b, k;
  int label;
  __device__ __forceinline__ float at(float x) const {
    // (a class of probability 0 has d = -inf: kept where e is 0 and b d finite, whatever b; NaN is in lse and k as well)
    const float d = fmaxf(x - lse, -1e4f);
    return -exp2_approx(fmaf(d, kLog2e, shift)) * fmaf(b, d, k);
  }
  __device__ __forceinline__ bool empty() const { return lse == -INFINITY; }
  __device__ __forceinline__ void less(float rest) { shift = -rest * kLog2e, k = fmaf(-b, rest, k); }
};
template <bool REST>
__device__ __forceinline__ Slope slope_at(const LogProbParams& p, long long i) {
  Slope s;
  s.label = label_at(p, i);
  s.lse = p.lse[i];
  s.a = s.label >= 0 && p.grad_log_prob ? p.grad_log_prob[i] : 0.0f;
  s.b = p.grad_entropy ? p.grad_entropy[i] : 0.0f;
  s.k = fmaf(s.b, p.entropy[i], s.a);
  if (REST) s.less(p.lse_rest[i]);
  if (s.lse != s.lse) s.k = NAN;
  return s;
}

// A thread's part of the sum of exp(x - lse): classes first, first + step, ... (0 where lse is -inf).
template <typename T>
__device__ __forceinline__ float rest_part(const T* x, long long stride, int first, int step, int classes, float lse) {
  float l = 0.0f;
  if (lse != -INFINITY)
    for (int c = first; c < classes; c += step) l += exp2_approx((to_float(x[c * stride]) - lse) * kLog2e);
  return l;
}
__device__ __forceinline__ float rest_of(float l, float lse) { return lse == -INFINITY ? 0.0f : logf(l); }

// REST: the forward's lse_rest is there.
template <typename T, bool PAIR, bool REST>
__global__ void __launch_bounds__(kApartThreads, 8) logprob_apart_bwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const unsigned s = (blockIdx.x * kApartThreads + threadIdx.x) * 2;
  const long long b = blockIdx.y + (long long)blockIdx.z * kApartItems;
  if (s >= (unsigned)p.positions || b >= p.batch) return;
  const T* x = (const T*)p.x + b * p.batch_stride + p.first;
  T* g = (T*)p.grad + b * p.grad_batch_stride + p.first;
  const bool second = s + 1 < (unsigned)p.positions;
  const long long at = b * p.space + p.first;
  Slope q[2] = {slope_at<REST>(p, at + s), slope_at<REST>(p, at + s + (second ? 1 : 0))};
  if (!REST) {
    for (int k = 0; k < 2; ++k)
      q[k].less(rest_of(rest_part(x + s + (second ? k : 0), p.class_stride, 0, 1, p.classes, q[k].lse), q[k].lse));
  }
  constexpr int kStep = 8;
  for (int c0 = 0; c0 < p.classes; c0 += kStep) {
    Two<T> w[kStep];
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      if (c0 + j < p.classes) {
        const T* xc = x + (long long)(c0 + j) * p.class_stride;
        if (PAIR) w[j] = *(const Two<T>*)(xc + s);
        else w[j] = rounded<T>(make_float2(to_float(xc[s]), to_float(xc[s + (second ? 1 : 0)])));
      }
    }
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      if (c0 + j < p.classes) {
        T* gc = g + (long long)(c0 + j) * p.grad_class_stride;
        const float2 f = floats(w[j]);
        float r[2] = {q[0].at(f.x), q[1].at(f.y)};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (c0 + j == q[k].label) r[k] += q[k].a;
          if (q[k].empty()) r[k] = 0.0f;
        }
        if (PAIR) {
          *(Two<T>*)(gc + s) = rounded<T>(make_float2(r[0], r[1]));
        } else {
          gc[s] = from_float<T>(r[0]);
          if (second) gc[s + 1] = from_float<T>(r[1]);
        }
      }
    }
  }
}

// ---- classes together: rows -------------------------------------------------------------------------
// A warp's row: lane i holds the classes i, i + 32, ...; the alternatives are picked one by one, each a round of the lanes' best.
__device__ __forceinline__ void best_of_warp(float& v, int& c) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float ov = __shfl_xor_sync(~0u, v, d);
    const int oc = __shfl_xor_sync(~0u, c, d);
    if (before(ov, oc, v, c)) v = ov, c = oc;
  }
}

template <typename T, int CAP>
__global__ void __launch_bounds__(128) logprob_warp_fwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.batch) return;
  const T* x = (const T*)p.x + row * p.batch_stride;
  const int n = p.classes, y = label_at(p, row);
  float f[CAP];
#pragma unroll
  for (int j = 0; j < CAP; ++j) f[j] = lane + 32 * j < n ? to_float(x[lane + 32 * j]) : -INFINITY;
  const float given = y < 0 ? 0.0f : to_float(x[y]);
  Online o;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < CAP; ++j) {
    o.m = fmaxf(o.m, f[j]);
    nan |= f[j] != f[j];
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) o.m = fmaxf(o.m, __shfl_xor_sync(~0u, o.m, d));
  if (__any_sync(~0u, nan)) o.m = NAN;
  if (o.m != -INFINITY) {
#pragma unroll
    for (int j = 0; j < CAP; ++j)
      if (32 * j < n) o.add(f[j]);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    o.l += __shfl_xor_sync(~0u, o.l, d);
    o.u += __shfl_xor_sync(~0u, o.u, d);
  }
  const Position q(o);
  if (lane == 0) q.put(p, row, o, y, given);
  float last_v = 0.0f;
  int last_c = -1;
  for (int t = 0; t < p.top; ++t) {
    float v = -INFINITY;
    int c = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < CAP; ++j) {
      const int k = lane + 32 * j;
      if (k < n && (t == 0 || before(last_v, last_c, f[j], k)) && before(f[j], k, v, c)) v = f[j], c = k;
    }
    best_of_warp(v, c);
    if (lane == t) {
      p.top_value[row * p.top + t] = q.log_prob(v);
      p.top_label[row * p.top + t] = c;
    }
    last_v = v, last_c = c;
  }
}

template <typename T, bool REST>
__global__ void __launch_bounds__(128) logprob_warp_bwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.batch) return;
  const T* x = (const T*)p.x + row * p.batch_stride;
  T* g = (T*)p.grad + row * p.grad_batch_stride;
  Slope q = slope_at<REST>(p, row);
  if (!REST) {
    float l = rest_part(x, 1, lane, 32, p.classes, q.lse);
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
    q.less(rest_of(l, q.lse));
  }
#pragma unroll 4
  for (int c = lane; c < p.classes; c += 32) {
    const float v = q.at(to_float(x[c])) + (c == q.label ? q.a : 0.0f);
    g[c] = from_float<T>(q.empty() ? 0.0f : v);
  }
}

// A CTA's row.  The alternatives need a second look at the scores: split into 32 parts, the top-th largest of the parts' maxima is a
// bound that at least `top` classes reach, and of long rows few more do (some 20 of a random row for top = 8); what reaches it is collected
// and ranked.  Where more reach it than there is room for, or there is a NaN, they are picked one by one: many equal scores, and rows so
// short that fewer than `top` parts hold a class (half types with up to 128 (top - 1) of them), whose bound is -inf.
constexpr int kWide = 512, kRoom = 256;

struct RowShared {
  float m[kWide / 32], l[kWide / 32], u[kWide / 32];
  float peak[32], cand[kRoom];
  int cand_class[kRoom];
  int count, wc[kWide / 32];
  float bound, wv[kWide / 32];
};

template <typename T>
__device__ __forceinline__ void pick_row(const T* x, int classes, int top, float* value, int* label, Position q, RowShared& sh) {
  const int lane = threadIdx.x, w = lane >> 5;
  float last_v = 0.0f;
  int last_c = -1;
  for (int t = 0; t < top; ++t) {
    float v = -INFINITY;
    int c = 0x7fffffff;
    for (int k = lane; k < classes; k += kWide) {
      const float f = to_float(x[k]);
      if ((t == 0 || before(last_v, last_c, f, k)) && before(f, k, v, c)) v = f, c = k;
    }
    best_of_warp(v, c);
    if ((lane & 31) == 0) sh.wv[w] = v, sh.wc[w] = c;
    __syncthreads();
    v = sh.wv[0], c = sh.wc[0];
    for (int i = 1; i < kWide / 32; ++i)
      if (before(sh.wv[i], sh.wc[i], v, c)) v = sh.wv[i], c = sh.wc[i];
    __syncthreads();
    if (lane == 0) value[t] = q.log_prob(v), label[t] = c;
    last_v = v, last_c = c;
  }
}

// A row as a few classes in front, vectors of 16 bytes, a few classes behind.
template <typename T>
struct RowShape {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* x;
  int n, head, vecs, behind;  // behind: first class after the vectors
  __device__ __forceinline__ RowShape(const T* row, int classes) : x(row), n(classes) {
    head = min(n, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
    vecs = (n - head) / V;
    behind = head + vecs * V;
  }
  __device__ __forceinline__ const Vec<T, V>* vectors() const { return (const Vec<T, V>*)(x + head); }
};

// The vectors' elements as pairs.
template <typename T>
struct alignas(16) Pairs {
  static constexpr int N = 8 / (int)sizeof(T);
  Two<T> v[N];
  __device__ __forceinline__ Two<T> most() const {
    Two<T> m = v[0];
#pragma unroll
    for (int k = 1; k < N; ++k) m = larger(m, v[k]);
    return m;
  }
};

// NV > 0: that many vectors a thread stay in registers; 0: the row is read again.
template <typename T, int NV>
__global__ void __launch_bounds__(kWide, NV >= 16 ? 1 : 2) logprob_row_fwd(const __grid_constant__ LogProbParams p) {
  __shared__ RowShared sh;
  grid_dependency();
  const int lane = threadIdx.x, w = lane >> 5;
  const long long row = blockIdx.x;
  const RowShape<T> r((const T*)p.x + row * p.batch_stride, p.classes);
  constexpr int V = RowShape<T>::V;
  typedef Pairs<T> P;
  const P* vectors = (const P*)r.vectors();
  const int y = label_at(p, row);
  if (lane == 0) sh.count = 0;
  // the odd ones: in front of the vectors (threads 0..) and behind them (threads 32..)
  const int odd_class = lane < r.head ? lane : lane >= 32 && r.behind + lane - 32 < r.n ? r.behind + lane - 32 : -1;
  const float odd = odd_class >= 0 ? to_float(r.x[odd_class]) : -INFINITY;
  const float given = y < 0 || lane ? 0.0f : to_float(r.x[y]);
  Online o;
  P f[NV > 0 ? NV : 1];
  if (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (lane + j * kWide < r.vecs) {
        f[j] = vectors[lane + j * kWide];
      } else {
#pragma unroll
        for (int k = 0; k < P::N; ++k) f[j].v[k] = both<T>(-INFINITY);
      }
    }
    Two<T> most = f[0].most();
#pragma unroll
    for (int j = 1; j < NV; ++j) most = larger(most, f[j].most());
    const float2 m = floats(most);
    o.m = fmaxf(odd, fmaxf(m.x, m.y));  // (NaN is not seen by the maximum, but by the sum)
  } else {
    o.m = odd;
    if (odd != -INFINITY) o.add(odd);
#pragma unroll 4
    for (int i = lane; i < r.vecs; i += kWide) {
      const P v = vectors[i];
      const float2 m2 = floats(v.most());
      const float m = fmaxf(m2.x, m2.y);
      if (m > o.m) o.raise(m);
      const float minus = o.m == -INFINITY ? 0.0f : -o.m;
      Sums2 sum;
#pragma unroll
      for (int k = 0; k < P::N; ++k) sum.add(floats(v.v[k]), make_float2(minus, minus));
      o.l += sum.l.x + sum.l.y;
      o.u += sum.u.x + sum.u.y;
    }
    if (o.l != o.l) o.m = NAN;
  }
  float peak = o.m;
  if (NV > 0) {
    // maximum of the row, then the sums about it
    float m = o.m;
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    if ((lane & 31) == 0) sh.m[w] = m;
    __syncthreads();
    m = sh.m[lane & 15];
#pragma unroll
    for (int d = 8; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    const float minus = m == -INFINITY ? 0.0f : -m;  // all -inf: the sums are 0, or NaN where there is one
    Sums2 sum;
    if (odd_class >= 0) sum.add(make_float2(odd, -INFINITY), make_float2(minus, minus));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * kWide < r.vecs) {
#pragma unroll
        for (int k = 0; k < P::N; ++k) sum.add(floats(f[j].v[k]), make_float2(minus, minus));
      }
    }
    o.m = m;
    o.l = sum.l.x + sum.l.y;
    o.u = sum.u.x + sum.u.y;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      o.l += __shfl_xor_sync(~0u, o.l, d);
      o.u += __shfl_xor_sync(~0u, o.u, d);
    }
  } else {
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
  }
  // the parts' maxima: 16 neighbouring threads each
#pragma unroll
  for (int d = 8; d; d >>= 1) peak = fmaxf(peak, __shfl_xor_sync(~0u, peak, d));
  if ((lane & 15) == 0) sh.peak[lane >> 4] = peak;
  if ((lane & 31) == 0) {
    if (NV == 0) sh.m[w] = o.m;
    sh.l[w] = o.l, sh.u[w] = o.u;
  }
  __syncthreads();
  if (NV > 0) {
    o.l = o.u = 0.0f;
    for (int i = 0; i < kWide / 32; ++i) o.l += sh.l[i], o.u += sh.u[i];
    if (o.l != o.l) o.m = NAN;
  } else {
    o.m = sh.m[0], o.l = sh.l[0], o.u = sh.u[0];
    for (int i = 1; i < kWide / 32; ++i) {
      Online b;
      b.m = sh.m[i], b.l = sh.l[i], b.u = sh.u[i];
      o.join(b);
    }
  }
  const Position q(o);
  if (lane == 0) q.put(p, row, o, y, given);
  if (p.top == 0) return;
  const auto put = [&](int t, float v, int c) {
    p.top_value[row * p.top + t] = q.log_prob(v);
    p.top_label[row * p.top + t] = c;
  };
  if (o.l == o.l) {
    // of the parts' maxima the one of rank top - 1 (equal ones by part); a part without classes counts as -inf
    peak = sh.peak[lane & 31];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int part = w * 2 + k;
      const float mine = sh.peak[part];
      const int rank = __popc(__ballot_sync(~0u, peak > mine || (peak == mine && (lane & 31) < part)));
      if (rank == p.top - 1) sh.bound = mine;
    }
    __syncthreads();
    const float bound = sh.bound;
    const auto offer = [&](float v, int c) {
      if (v >= bound) {
        const int k = atomicAdd(&sh.count, 1);
        if (k < kRoom) sh.cand[k] = v, sh.cand_class[k] = c;
      }
    };
    const auto offer_vector = [&](const P& v, int first) {
      const float2 m = floats(v.most());
      if (fmaxf(m.x, m.y) >= bound) {
#pragma unroll
        for (int k = 0; k < P::N; ++k) {
          const float2 e = floats(v.v[k]);
          offer(e.x, first + 2 * k);
          offer(e.y, first + 2 * k + 1);
        }
      }
    };
    if (odd_class >= 0) offer(odd, odd_class);
    if (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (lane + j * kWide < r.vecs) offer_vector(f[j], r.head + (lane + j * kWide) * V);
    } else {
#pragma unroll 4
      for (int i = lane; i < r.vecs; i += kWide) offer_vector(vectors[i], r.head + i * V);
    }
    __syncthreads();
    const int count = sh.count;
    if (count <= kRoom) {
      for (int i = lane; i < count; i += kWide) {
        const float v = sh.cand[i];
        const int c = sh.cand_class[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += sh.cand[j] > v || (sh.cand[j] == v && sh.cand_class[j] < c);
        if (rank < p.top) put(rank, v, c);
      }
      return;
    }
  }
  pick_row(r.x, r.n, p.top, p.top_value + row * p.top, p.top_label + row * p.top, q, sh);
}

template <typename T, bool REST>
__global__ void __launch_bounds__(kWide, 3) logprob_row_bwd(const __grid_constant__ LogProbParams p) {
  grid_dependency();
  const int lane = threadIdx.x;
  const long long row = gridDim.x - 1 - blockIdx.x;  // backwards: the rows that the forward read last are still in L2
  const RowShape<T> r((const T*)p.x + row * p.batch_stride, p.classes);
  T* g = (T*)p.grad + row * p.grad_batch_stride;
  Slope q = slope_at<REST>(p, row);
  if (!REST) {
    __shared__ float parts[kWide / 32];
    float l = rest_part(r.x, 1, lane, kWide, r.n, q.lse);
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
    if ((lane & 31) == 0) parts[lane >> 5] = l;
    __syncthreads();
    l = 0.0f;
    for (int i = 0; i < kWide / 32; ++i) l += parts[i];
    q.less(rest_of(l, q.lse));
  }
  constexpr int V = RowShape<T>::V;
  const auto one = [&](int c) {
    const float v = q.at(to_float(r.x[c])) + (c == q.label ? q.a : 0.0f);
    g[c] = from_float<T>(q.empty() ? 0.0f : v);
  };
  // vectors where scores and gradient have the same alignment
  if ((((uintptr_t)r.x ^ (uintptr_t)g) & 15) != 0) {
#pragma unroll 4
    for (int c = lane; c < r.n; c += kWide) one(c);
    return;
  }
  if (lane < r.head) one(lane);
  if (r.behind + lane < r.n) one(r.behind + lane);
  const int vector_of_label = q.label < r.head || q.label >= r.behind ? -1 : (q.label - r.head) / V;
  for (int i0 = lane; i0 < r.vecs; i0 += 4 * kWide) {
    Vec<T, V> v[4];  // all under way together
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * kWide < r.vecs) v[j] = r.vectors()[i0 + j * kWide];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * kWide;
      if (i >= r.vecs) break;
      Vec<T, V> to;
      float f[V];
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = q.at(to_float(v[j].v[k]));
      if (i == vector_of_label) {
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] += r.head + i * V + k == q.label ? q.a : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) to.v[k] = from_float<T>(q.empty() ? 0.0f : f[k]);
      ((Vec<T, V>*)(g + r.head))[i] = to;
    }
  }
}

// ---- launches ----------------------------------------------------------------------------------------
// 0, or 1: more CTAs than a grid has.
template <typename T, bool PAIR, int TOP>
void launch_apart_fwd(const LogProbParams& p, dim3 grid, cudaStream_t st) {
  // (with more than two alternatives the registers hold those)
  if (TOP <= 2 && p.classes <= 8) launch_dependent(logprob_apart_fwd<T, PAIR, TOP, TOP <= 2 ? 8 : 0>, grid, kApartThreads, 0, st, p);
  else if (TOP <= 2 && p.classes <= 16) launch_dependent(logprob_apart_fwd<T, PAIR, TOP, TOP <= 2 ? 16 : 0>, grid, kApartThreads, 0, st, p);
  else launch_dependent(logprob_apart_fwd<T, PAIR, TOP, 0>, grid, kApartThreads, 0, st, p);
}
template <typename T, bool PAIR>
void launch_logprob_apart(const LogProbParams& p, bool fwd, dim3 grid, cudaStream_t st) {
  if (!fwd) launch_dependent(p.lse_rest ? logprob_apart_bwd<T, PAIR, true> : logprob_apart_bwd<T, PAIR, false>, grid, kApartThreads, 0, st, p);
  else if (p.top == 0) launch_apart_fwd<T, PAIR, 0>(p, grid, st);
  else if (p.top <= 2) launch_apart_fwd<T, PAIR, 2>(p, grid, st);
  else if (p.top <= 5) launch_apart_fwd<T, PAIR, 5>(p, grid, st);
  else launch_apart_fwd<T, PAIR, 16>(p, grid, st);
}

template <typename T>
int launch_logprob(const LogProbParams& p, bool fwd, cudaStream_t st) {
  if (p.class_stride == 1 && p.space == 1) {
    const long long ctas = p.classes <= 1024 ? (p.batch + 3) / 4 : p.batch;
    if (ctas > 0x7fffffffLL) return 1;
    const dim3 grid((unsigned)ctas);
    // vectors of a thread, if the row is to stay in registers
    const long long vecs = (p.classes / RowShape<T>::V + kWide - 1) / kWide;
    if (p.classes <= 1024) {
      if (!fwd) launch_dependent(p.lse_rest ? logprob_warp_bwd<T, true> : logprob_warp_bwd<T, false>, grid, 128, 0, st, p);
      else if (p.classes <= 128) launch_dependent(logprob_warp_fwd<T, 4>, grid, 128, 0, st, p);
      else launch_dependent(logprob_warp_fwd<T, 32>, grid, 128, 0, st, p);
    } else if (!fwd) {
      launch_dependent(p.lse_rest ? logprob_row_bwd<T, true> : logprob_row_bwd<T, false>, grid, kWide, 0, st, p);
    } else if (vecs <= 2) {
      launch_dependent(logprob_row_fwd<T, 2>, grid, kWide, 0, st, p);
    } else if (vecs <= 8) {
      launch_dependent(logprob_row_fwd<T, 8>, grid, kWide, 0, st, p);
    } else if (vecs <= 16) {
      launch_dependent(logprob_row_fwd<T, 16>, grid, kWide, 0, st, p);
    } else {
      launch_dependent(logprob_row_fwd<T, 0>, grid, kWide, 0, st, p);
    }
    return 0;
  }
  if (p.batch > 60000LL * kApartItems) return 1;
  const long long strides = p.space | p.batch_stride | p.class_stride | (fwd ? 0 : p.grad_batch_stride | p.grad_class_stride);
  const uintptr_t at = (uintptr_t)p.x | (fwd ? 0 : (uintptr_t)p.grad);
  const bool pair = strides % 2 == 0 && at % (2 * sizeof(T)) == 0;
  LogProbParams q = p;
  constexpr long long kMost = 1LL << 30;  // positions of a launch
  for (q.first = 0; q.first < p.space; q.first += kMost) {
    q.positions = (int)(p.space - q.first < kMost ? p.space - q.first : kMost);
    const dim3 grid((unsigned)(((q.positions + 1) / 2 + kApartThreads - 1) / kApartThreads), (unsigned)(p.batch < kApartItems ? p.batch : kApartItems),
                    (unsigned)((p.batch + kApartItems - 1) / kApartItems));
    if (pair) launch_logprob_apart<T, true>(q, fwd, grid, st);
    else launch_logprob_apart<T, false>(q, fwd, grid, st);
  }
  return 0;
}

}  // namespace mvr
