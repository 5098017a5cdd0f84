// Rotary positions of several axes: pair i of an axis with n pairs turns by angle = position * base^(-i / n),
//   (a, b) -> (a cos - b sin, a sin + b cos),
// pairs are neighbouring columns (2i, 2i + 1) or half of the turned columns apart (i, i + pairs); further columns are copied.  The
// gradient is the same turn backwards.
//
// Angles.  A far position times a frequency has more turns than 24 bits leave room for, so the product is formed in 64 bits, in turns
// (the frequencies come divided by 2 pi), and its whole turns are taken off before it becomes a float; what that rounding leaves goes
// into sine and cosine by their derivatives.  Both are within a few 2^-24 for every position below 2^31.
//
// Bound by memory: every element is read and written once.  A thread takes one vector of columns (both of a pair) of one token and
// walks the heads, so that sines and cosines, some 60 instructions a pair, are formed once for all of them, of queries and keys alike.
// Where tokens are few the heads are spread over more threads, which form them again.
#pragma once
#include <algorithm>

#include "mvr_types.cuh"

namespace mvr {

constexpr int kRotaryThreads = 256, kRotaryPairs = 256, kRotaryAxes = 4;

struct RotaryParams {
  const void* x[2];       // queries, keys (or null)
  void* out[2];           // contiguous (N, L, heads, D)
  long long s_n[2], s_l[2], s_h[2];
  const void* positions;  // (N, L, axes)
  int position_type;      // 0 float, 1 int32, 2 int64
  long long p_n, p_l, p_a;
  long long tokens;       // N * L
  int L, D, heads[2];
  int pairs, ends[kRotaryAxes];  // pairs of all axes, and where each axis ends among them
  int units, lanes;       // threads of a row: vectors of pairs and of copied columns; threads that share a token's heads
  float sign;
  double turns[kRotaryPairs];  // per position, of every pair
};

__device__ __forceinline__ double position_at(const RotaryParams& p, long long at) {
  return p.position_type == 0 ? (double)((const float*)p.positions)[at] : p.position_type == 1 ? (double)((const int*)p.positions)[at]
                                                                                              : (double)((const long long*)p.positions)[at];
}

__device__ __forceinline__ void turn_of(double turns, float& c, float& s) {
  const double half = 2.0 * (turns - rint(turns));  // in half turns, within 1
  const float h = (float)half, rest = (float)(half - (double)h) * 3.14159265358979f;
  sincospif(h, &s, &c);
  const float c0 = c;
  c = fmaf(-s, rest, c);
  s = fmaf(c0, rest, s);
}

// V: elements of a vector; a thread holds V pairs (INTERLEAVED: V / 2, or one with V 1) or V copied columns.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kPairs = INTERLEAVED ? (V + 1) / 2 : V, kAtOnce = V * sizeof(T) >= 16 ? 4 : 8;
  constexpr bool kTwo = !INTERLEAVED || V == 1;  // a pair's columns lie in two vectors
  typedef Vec<T, V> Vector;
  grid_dependency();
  const long long id = (long long)blockIdx.x * kRotaryThreads + threadIdx.x, group = id / p.units;
  const int unit = (int)(id - group * p.units);
  const long long token = group / p.lanes;
  const int lane = (int)(group - token * p.lanes);
  if (token >= p.tokens) return;
  const long long n = token / p.L;
  const int l = (int)(token - n * p.L);
  const int turned = p.pairs / kPairs;  // units that turn
  const bool turns = unit < turned;
  // first column of the vector, and of the one with the pairs' other columns
  const int pair = unit * kPairs;
  const int col = !turns ? 2 * p.pairs + (unit - turned) * V : INTERLEAVED ? 2 * pair : pair, other = INTERLEAVED ? col + 1 : col + p.pairs;
  float c[kPairs], s[kPairs];
  if (turns) {
    const long long at = n * p.p_n + l * p.p_l;
    int axis = 0;
    double place = 0.0;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      if (k == 0 || pair + k >= p.ends[axis]) {
        while (pair + k >= p.ends[axis]) ++axis;
        place = position_at(p, at + axis * p.p_a);
      }
      turn_of(place * p.turns[pair + k], c[k], s[k]);
      s[k] *= p.sign;
    }
  }
  const int heads = p.heads[0] + p.heads[1];
  for (int h0 = lane; h0 < heads; h0 += kAtOnce * p.lanes) {
    Vector a[kAtOnce], b[kAtOnce];
    T* to[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + i * p.lanes;
      if (h >= heads) break;
      const int which = h >= p.heads[0], head = which ? h - p.heads[0] : h;
      const T* from = (const T*)p.x[which] + n * p.s_n[which] + l * p.s_l[which] + head * p.s_h[which];
      to[i] = (T*)p.out[which] + (token * p.heads[which] + head) * p.D;
      a[i] = *(const Vector*)(from + col);
      if (kTwo && turns) b[i] = *(const Vector*)(from + other);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (h0 + i * p.lanes >= heads) break;
      if (turns) {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          T& first = a[i].v[kTwo ? k : 2 * k];
          T& second = kTwo ? b[i].v[k] : a[i].v[2 * k + 1 < V ? 2 * k + 1 : 0];
          const float u = to_float(first), v = to_float(second);
          first = from_float<T>(u * c[k] - v * s[k]);
          second = from_float<T>(u * s[k] + v * c[k]);
        }
      }
      *(Vector*)(to[i] + col) = a[i];
      if (kTwo && turns) *(Vector*)(to[i] + other) = b[i];
    }
  }
}

// 0, or 1: more CTAs than a grid has.
template <typename T, int V>
int launch_rotary(RotaryParams& p, bool interleaved, cudaStream_t st) {
  const int per = interleaved ? (V + 1) / 2 : V, heads = p.heads[0] + p.heads[1];
  p.units = p.pairs / per + (p.D - 2 * p.pairs) / V;
  // threads that share a token's heads: until a row's vectors lie together in 128 bytes, and until there are two CTAs' worth an SM
  const long long want = 148LL * 2 * 1024;
  long long lanes = std::max<long long>(128 / (int)sizeof(T) / V / p.units, (want + p.tokens * p.units - 1) / (p.tokens * p.units));
  p.lanes = (int)std::max<long long>(1, std::min<long long>(lanes, heads));
  const long long ctas = (p.tokens * p.lanes * p.units + kRotaryThreads - 1) / kRotaryThreads;
  if (ctas > 0x7fffffffLL) return 1;
  launch_dependent(interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>, dim3((unsigned)ctas), dim3(kRotaryThreads), 0, st, p);
  return 0;
}

}  // namespace mvr
