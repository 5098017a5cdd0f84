// Rotary positions of several axes: pair i of an axis with n pairs turns by angle = position * base^(-i / n),
//   (a, b) -> (a cos - b sin, a sin + b cos),
// pairs are neighbouring columns (2i, 2i + 1) or half of the turned columns apart (i, i + pairs); further columns are copied.  The
// gradient is the same turn backwards.
//
// Angles.  A far position times a frequency has more turns than 24 bits leave room for, so the product is formed in whole numbers:
// frequencies come as 64-bit fractions of a turn, their product with a position wraps at whole turns by itself, and its upper 32 bits,
// rounded, are the angle: off by 2^-33 of a turn, and by the frequency's own error, up to 2^-64 (of pair i of slow bases about i 2^-66) times the
// position, which is 2^-33 at 2^31.  A floating position is a number of 24 bits, whose product is shifted.  (In
// 64-bit floating arithmetic the conversions and products took longer than memory: 80 000 tokens of 128 columns 37 us.)  Half types: sine
// and cosine by the function units (2^-21); float: the library's, and what the angle's rounding to a float left by their derivatives.
//
// Bound by memory: every element is read and written once.  A CTA takes some tokens of an image and forms their sines and cosines once, in
// shared memory; a thread takes one vector of columns (both of a pair) of one token and a few heads at a time, of queries and keys alike, and
// asks for the next ones before it turns those.  Measured: 8 x 13 635 tokens of 20 heads of 64, bfloat16, 97 us (5.7 TB/s, 88 % of a copy's
// rate); 20 000 tokens of 32 heads of 128: float 111 us (a copy 107), bfloat16 61 (57); with pairs apart by no multiple of a vector 166 to 175 (1.9
// TB/s: the partners' words are loaded one by one, and every column twice).
#pragma once
#include <algorithm>

#include "mvr_types.cuh"

namespace mvr {

constexpr int kRotaryThreads = 256, kRotaryPairs = 256, kRotaryAxes = 4;

struct RotaryParams {
  const void* x[2];       // queries, keys (or null)
  void* out[2];           // contiguous (N, L, heads, D)
  long long s_n[2];
  int s_l[2], s_h[2];
  const void* positions;  // (N, L, axes)
  int position_type;      // 0 float, 1 int32, 2 int64
  long long p_n, p_l, p_a;
  int L, D, heads[2];
  int pairs, ends[kRotaryAxes];  // pairs of all axes, and where each axis ends among them
  int units, lanes;       // threads of a row, each with a vector of columns (or two of a pair's); threads that share a token's heads
  int stride;             // a token's sines and cosines in shared memory
  int together, ctas;     // tokens of a CTA, CTAs of an image
  int n0;                 // the launch's first image
  Divisor by_units, by_lanes, by_pairs;
  float sign;
  unsigned long long turns[kRotaryPairs];  // per position, of every pair, in 2^-64
};

// A position as a whole number times 2^shift.
struct Place {
  unsigned long long number;  // of a floating one: 24 bits
  int shift;
  bool floating, negative, finite;
};
__device__ __forceinline__ Place place_at(const RotaryParams& p, long long at) {
  Place v = {0, 0, false, false, true};
  if (p.position_type == 0) {
    const unsigned bits = ((const unsigned*)p.positions)[at], exponent = (bits >> 23) & 255;
    v.number = (bits & 0x7fffff) | (exponent ? 0x800000 : 0);
    v.shift = (int)(exponent ? exponent : 1) - 150;
    v.floating = true;
    v.negative = bits >> 31;
    v.finite = exponent != 255;
  } else {
    v.number = p.position_type == 1 ? (unsigned long long)(long long)((const int*)p.positions)[at] : ((const unsigned long long*)p.positions)[at];
  }
  return v;
}
// The angle in 2^-32 turns, rounded.
__device__ __forceinline__ int angle_of(const Place& v, unsigned long long turns) {
  const unsigned long long low = v.number * turns, half = 1ull << 31;
  if (!v.floating) return (int)((low + half) >> 32);
  const unsigned long long high = __umul64hi(v.number, turns);
  const int s = v.shift;
  unsigned long long a = s >= 0 ? (s < 64 ? low << s : 0) : s > -64 ? (low >> -s) | (high << (64 + s)) : s > -128 ? high >> (-64 - s) : 0;
  if (v.negative) a = 0 - a;
  return (int)((a + half) >> 32);
}
template <typename T>
__device__ __forceinline__ void turn_of(int angle, float& c, float& s) {
  const float f = (float)angle;  // in 2^-31 half turns
  if constexpr (sizeof(T) == 2) {
    __sincosf(f * 1.4629180792671596e-9f, &s, &c);  // pi 2^-31
  } else {
    sincospif(f * 4.656612873077393e-10f, &s, &c);  // 2^-31
    const float rest = (float)(angle - __float2int_rn(f)) * 1.4629180792671596e-9f, c0 = c;
    c = fmaf(-s, rest, c);
    s = fmaf(c0, rest, s);
  }
}

// What a thread holds.
//   kApart     V columns, and those half of the turned columns apart: V pairs (or V copied columns)
//   kNeighbour V columns: V / 2 pairs
//   kOwn       V columns, with the others of their pairs wherever these lie: for pairs apart by no multiple of V (columns and rows are); it reads
//              words of the others' columns, which other threads load as well, and stores vectors
//   kScalar    a pair, or a copied column: rows of any size and place
enum { kApart = 0, kNeighbour = 1, kOwn = 2, kScalar = 3 };

// Heads that a thread asks for at once.
template <typename T, int V, int KIND>
constexpr int kRotaryHeads = KIND == kScalar ? 8 : KIND == kOwn ? 2 : 4;

// V neighbouring elements of a row from any place on: words of 4 bytes, shifted where the place is odd.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_anywhere(const T* from) {
  Vec<T, V> to;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) to.v[e] = from[e];
  } else {
    uint32_t* const words = (uint32_t*)&to;
    if (((uintptr_t)from & 2) == 0) {
#pragma unroll
      for (int e = 0; e < V / 2; ++e) words[e] = ((const uint32_t*)from)[e];
    } else {  // (a row begins at a multiple of 16 bytes: the element before, and the one behind, are the row's)
      const uint32_t* at = (const uint32_t*)(from - 1);
      uint32_t w[V / 2 + 1];
#pragma unroll
      for (int e = 0; e <= V / 2; ++e) w[e] = at[e];
#pragma unroll
      for (int e = 0; e < V / 2; ++e) words[e] = __byte_perm(w[e], w[e + 1], 0x5432);
    }
  }
  return to;
}

// INTERLEAVED: pairs are neighbours (kNeighbour; kScalar).
template <typename T, int V, int KIND, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, KIND == kApart && V == 8 ? 2 : 3) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kColumns = KIND == kApart ? V : KIND == kNeighbour ? V / 2 : V;  // sines (and cosines) of a thread: of its pairs, or its columns
  constexpr int kAtOnce = kRotaryHeads<T, V, KIND>;
  constexpr bool kTwo = KIND != kNeighbour;
  typedef Vec<T, V> Vector;
  typedef Vec<float, kColumns> Floats;
  extern __shared__ __align__(16) float cosines[];
  float* const sines = cosines + p.together * p.stride;
  // (neighbouring threads want different frequencies: from the launch's constants they would come one after another every time)
  __shared__ unsigned long long frequencies[kRotaryPairs];
  for (int i = threadIdx.x; i < p.pairs; i += kRotaryThreads) frequencies[i] = p.turns[i];
  __syncthreads();
  grid_dependency();
  const int image = blockIdx.x / p.ctas, n = p.n0 + image, first = (blockIdx.x - image * p.ctas) * p.together, count = min(p.together, p.L - first);
  const int items = count * p.units * p.lanes, heads = p.heads[0] + p.heads[1], turned = p.stride / kColumns;  // turned: units that turn
  // of the CTA's first token
  const T* const x0 = (const T*)p.x[0] + n * p.s_n[0] + (long long)first * p.s_l[0];
  const T* const x1 = (const T*)p.x[1] + n * p.s_n[1] + (long long)first * p.s_l[1];
  T* const y0 = (T*)p.out[0] + ((long long)n * p.L + first) * p.heads[0] * p.D;
  T* const y1 = (T*)p.out[1] + ((long long)n * p.L + first) * p.heads[1] * p.D;
  struct Item {  // a vector of columns of kAtOnce heads
    Vector a[kAtOnce], b[kAtOnce];
    int unit, mine, lane, col, other;
  };
  const auto head_at = [&](const Item& t, int i) { return t.lane + i * p.lanes; };
  const auto load = [&](int item) {
    Item t;
    const int group = p.by_units.quotient(item);
    t.unit = item - group * p.units;
    t.mine = p.by_lanes.quotient(group);
    t.lane = group - t.mine * p.lanes;
    const bool turns = t.unit < turned;
    // first column of the vector, and how far the pairs' other columns are from there
    t.other = 0;
    if (KIND == kNeighbour || KIND == kOwn) {
      t.col = t.unit * V;
      if (KIND == kOwn) t.other = t.col + V <= p.pairs ? p.pairs : t.col >= p.pairs ? -p.pairs : 0;  // (0: some lie ahead, some behind)
    } else {
      t.col = !turns ? 2 * p.pairs + (t.unit - turned) * V : INTERLEAVED ? 2 * t.unit : t.unit * V;
      t.other = INTERLEAVED ? 1 : p.pairs;
    }
    const T* const q = x0 + (long long)t.mine * p.s_l[0] + t.col;
    const T* const k = x1 + (long long)t.mine * p.s_l[1] + t.col;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = head_at(t, i);
      if (h < heads) {
        const T* from = h < p.heads[0] ? q + (long long)h * p.s_h[0] : k + (long long)(h - p.heads[0]) * p.s_h[1];
        t.a[i] = *(const Vector*)from;
        if (KIND == kOwn && turns) {
          if (t.other != 0 && t.col + V <= 2 * p.pairs) {
            t.b[i] = load_anywhere<T, V>(from + t.other);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) t.b[i].v[e] = from[t.col + e < p.pairs ? e + p.pairs : t.col + e < 2 * p.pairs ? e - p.pairs : e];
          }
        } else if (kTwo && turns) {
          t.b[i] = *(const Vector*)(from + t.other);
        }
      }
    }
    return t;
  };
  const auto turn = [&](const Item& t) {
    T* const to_q = y0 + (long long)t.mine * p.heads[0] * p.D + t.col;
    T* const to_k = y1 + (long long)t.mine * p.heads[1] * p.D + t.col;
    const bool turns = t.unit < turned;
    Floats c, s;
    if (turns) {
      c = *(const Floats*)(cosines + t.mine * p.stride + t.unit * kColumns);
      s = *(const Floats*)(sines + t.mine * p.stride + t.unit * kColumns);
    }
    // (of a vector that turns, columns that do not)
    const int whole = KIND == kNeighbour ? p.pairs - t.unit * kColumns : KIND == kOwn ? 2 * p.pairs - t.col : V;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = head_at(t, i);
      if (h < heads) {
        T* to = h < p.heads[0] ? to_q + h * p.D : to_k + (h - p.heads[0]) * p.D;
        if (!turns) {
          *(Vector*)to = t.a[i];
        } else if constexpr (KIND == kNeighbour) {
          FloatPairs<T, V> u(t.a[i]);
#pragma unroll
          for (int e = 0; e < kColumns; ++e) {
            const float x = u.v[e].x, y = u.v[e].y;
            if (e < whole) u.v[e] = make_float2(x * c.v[e] - y * s.v[e], x * s.v[e] + y * c.v[e]);
          }
          *(Vector*)to = u.vector();
        } else {
          FloatPairs<T, V> u(t.a[i]), v(t.b[i]);
#pragma unroll
          for (int e = 0; e < FloatPairs<T, V>::kPairs; ++e) {
            const float2 cos2 = make_float2(c.v[2 * e], c.v[V == 1 ? 0 : 2 * e + 1]), sin2 = make_float2(s.v[2 * e], s.v[V == 1 ? 0 : 2 * e + 1]);
            const float2 x = u.v[e], y = v.v[e];
            if constexpr (KIND == kOwn) {
              const float2 r = fma2(x, cos2, mul2(y, sin2));
              u.v[e] = make_float2(2 * e < whole ? r.x : x.x, 2 * e + 1 < whole ? r.y : x.y);
            } else {
              u.v[e] = fma2(x, cos2, mul2(y, make_float2(-sin2.x, -sin2.y)));
              v.v[e] = fma2(x, sin2, mul2(y, cos2));
            }
          }
          *(Vector*)to = u.vector();
          if (KIND != kOwn) *(Vector*)(to + t.other) = v.vector();
        }
      }
    }
  };
  int item = threadIdx.x;
  Item now;
  if (item < items) now = load(item);
  for (int i = threadIdx.x; i < count * p.pairs; i += kRotaryThreads) {
    const int t = p.by_pairs.quotient(i), at = i - t * p.pairs;
    const int axis = (at >= p.ends[0]) + (at >= p.ends[1]) + (at >= p.ends[2]);
    const Place place = place_at(p, n * p.p_n + (first + t) * p.p_l + axis * p.p_a);
    float c, s;
    turn_of<T>(angle_of(place, frequencies[at]), c, s);
    c = place.finite ? c : NAN;
    s = place.finite ? s * p.sign : NAN;
    cosines[t * p.stride + at] = c;
    sines[t * p.stride + at] = KIND == kOwn ? -s : s;
    if (KIND == kOwn) {
      cosines[t * p.stride + p.pairs + at] = c;
      sines[t * p.stride + p.pairs + at] = s;
    }
  }
  __syncthreads();
  for (; item < items; item += kRotaryThreads) {
    Item next;
    if (item + kRotaryThreads < items) next = load(item + kRotaryThreads);
    turn(now);
    now = next;
  }
}

// Nothing, or a launch that failed.
template <typename T, int V, int KIND>
bool launch_rotary(RotaryParams& p, int images, bool interleaved, cudaStream_t st) {
  const int heads = p.heads[0] + p.heads[1], columns = 2 * p.pairs;
  if (KIND == kApart || KIND == kScalar) p.units = p.pairs / V + (p.D - columns) / V, p.stride = p.pairs;
  if (KIND == kNeighbour) p.units = p.D / V, p.stride = (columns + V - 1) / V * (V / 2);
  if (KIND == kOwn) p.units = p.D / V, p.stride = (columns + V - 1) / V * V;
  p.lanes = (heads + kRotaryHeads<T, V, KIND> - 1) / kRotaryHeads<T, V, KIND>;
  // Tokens of a CTA: so many that all CTAs run at once (three an SM), in as many waves as leave a thread four turns at most (one turn a CTA
  // took twice as long), and a CTA 32 KB of sines and cosines.
  const long long all = ((long long)images * p.L * p.units * p.lanes + kRotaryThreads - 1) / kRotaryThreads, at_once = 148 * 3;
  const long long waves = (all + 4 * at_once - 1) / (4 * at_once), of_image = std::max<long long>(1, waves * at_once / images);
  const long long least = std::max(1, kRotaryThreads / (p.units * p.lanes));  // tokens of one turn
  p.together = (int)std::max<long long>(1, std::min<long long>({std::max((p.L + of_image - 1) / of_image, least), 4096 / std::max(1, p.stride), p.L}));
  p.ctas = (p.L + p.together - 1) / p.together;
  p.by_units.set(p.units);
  p.by_lanes.set(p.lanes);
  p.by_pairs.set(std::max(1, p.pairs));
  const int most = std::max(1, (1 << 30) / p.ctas);  // images of a launch
  const size_t shared = (size_t)p.together * p.stride * 2 * sizeof(float);
  for (int first = 0; first < images; first += most) {
    p.n0 = first;
    const long long ctas = (long long)std::min(most, images - first) * p.ctas;
    const dim3 grid((unsigned)ctas), threads(kRotaryThreads);
    if constexpr (KIND == kScalar) launch_dependent(interleaved ? rotary_kernel<T, V, KIND, true> : rotary_kernel<T, V, KIND, false>, grid, threads, shared, st, p);
    else launch_dependent(rotary_kernel<T, V, KIND, KIND == kNeighbour>, grid, threads, shared, st, p);
    if (cudaGetLastError() != cudaSuccess) return false;
  }
  return true;
}

}  // namespace mvr
