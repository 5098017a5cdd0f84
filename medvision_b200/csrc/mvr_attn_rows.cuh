// Attention forward of a few rows over a window of states: a new token at the end of a cache, with the heads that share a key head.
//
// Bound by memory: each state is read once for all rows of its key head.  A lane holds eight columns, so that a warp reads 32 / (D / 8) states
// in one access of 16 bytes a lane; each lane copies its own pieces to shared memory three steps of four accesses ahead and reads them back,
// so that no thread waits for another.  Products with the rows' columns are summed over a state's lanes by shuffles that leave each lane a
// part of the scores, for which it keeps maximum and sum; joined at the end over groups, warps (shared memory) and parts of the states
// (attn_join).  Weights stay in float.
//
// 32 caches' windows of 2051 states, 8 heads of 128, bfloat16: 55 us (floor 41; without the copies ahead 86).  Beyond two rows (float: eight)
// the shuffles and products of this kernel take longer than what the tensor cores' (the tiles') fixed steps cost.
#pragma once
#include "mvr_attn.cuh"

namespace mvr {

constexpr int kRowsThreads = 128, kRowsAhead = 4, kRowsStages = 4;
template <typename T>
constexpr size_t kRowsShared = (size_t)kRowsStages * kRowsAhead * 2 * kRowsThreads * 8 * sizeof(T);

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float larger_or_nan(float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }

// DP: head size, rounded up to a power of two of at least 32.  R: rows, likewise.
template <typename T, int DP, int R>
__global__ void __launch_bounds__(kRowsThreads) attn_rows_fwd(const __grid_constant__ AttnParams p) {
  constexpr int kLanes = DP / 8, kStates = 32 / kLanes, kWarps = kRowsThreads / 32, kPairs = 4;  // lanes of a state, states of a warp's access
  constexpr int kValues = kRowsAhead * R, kOwn = kValues > kLanes ? kValues / kLanes : 1;         // scores of a group, and of a lane of it
  static_assert(kRowsAhead == 4, "");
  // the lane of a group that keeps value i (among others)
  const auto lane_of = [](int i) { return kValues > kLanes ? i / kOwn : i * (kLanes / kValues); };
  typedef Vec<T, 8> Vector;
  typedef FloatPairs<T, 8> P;
  __shared__ Span spans[R];
  __shared__ float tops[kWarps][R], totals[kWarps][R];
  __shared__ __align__(16) float sums[kWarps][R][DP];  // (written in pairs)
  grid_dependency();
  const int n = blockIdx.x, hk = blockIdx.y, split = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % kLanes;
  const int rows = p.T * p.G, end = states_of(p, n);
  const Places places = places_of(p, n);
  if (threadIdx.x < R) {
    const int token = p.by_G.quotient(min((int)threadIdx.x, rows - 1));
    spans[threadIdx.x] = span_of(p, places, token, token, end);
  }
  const Span all = span_of(p, places, 0, p.T - 1, end);
  // the states that any row reads, in a row: the first ones, then the window
  const int leading = min(all.sink, all.lo), count = leading + all.hi - all.lo;
  const int per = (count + p.splits - 1) / p.splits, begin = min(count, split * per), stop = min(count, begin + per);
  const bool in = part * 8 < p.D;  // (of a head size that is no power of two: lanes without columns)
  float2 q[R][kPairs], acc[R][kPairs];
  float top[kOwn], total[kOwn];
  const int row0 = (kValues > kLanes ? part * kOwn : part / (kLanes / kValues)) % R;  // this lane's first row
#pragma unroll
  for (int i = 0; i < kOwn; ++i) top[i] = -INFINITY, total[i] = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) q[r][k] = acc[r][k] = make_float2(0.0f, 0.0f);
    if (r < rows && in) {
      const int token = p.by_G.quotient(r);
      const P x(*(const Vector*)((const T*)p.q + n * p.q_r + token * p.q_t + (hk * p.G + r - token * p.G) * p.q_h + part * 8));
#pragma unroll
      for (int k = 0; k < kPairs; ++k) q[r][k] = mul2(x.v[k], make_float2(p.scale_log2, p.scale_log2));
    }
  }
  __syncthreads();
  const T* const keys = (const T*)p.k + (long long)n * p.k_n + (long long)hk * p.k_h + part * 8;
  const T* const values = (const T*)p.v + (long long)n * p.v_n + (long long)hk * p.v_h + part * 8;
  const bool alike = p.T == 1;  // one token: all rows read the same states
  // Each lane copies its own pieces of keys and values to shared memory, some steps ahead, and reads them back: nobody waits for another.
  constexpr int kBytes = 8 * sizeof(T), kStep = kStates * kRowsAhead;
  extern __shared__ __align__(16) char rows_ring[];
  char* const ring = rows_ring + (warp * 32 + lane) * 16;
  constexpr int kPiece = kRowsThreads * 16, kParts = kBytes / 16, kStage = kRowsAhead * 2 * kParts * kPiece;  // of all threads
  const auto ask = [&](int base, int stage) {
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      const int at = base + u * kStates + lane / kLanes, state = at < leading ? at : all.lo + (at - leading);
      const bool there = at < stop && in;
      const T* const k = keys + (there ? (long long)state * p.k_l : 0);
      const T* const v = values + (there ? (long long)state * p.v_l : 0);
#pragma unroll
      for (int e = 0; e < kParts; ++e) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + stage * kStage + (u * 2 * kParts + e) * kPiece);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"((const char*)k + e * 16), "r"(there ? 16 : 0) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + kParts * kPiece), "l"((const char*)v + e * 16), "r"(there ? 16 : 0) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto take = [&](int stage, int u, int which) {
    Vector x;
#pragma unroll
    for (int e = 0; e < kParts; ++e) ((uint4*)&x)[e] = *(const uint4*)(ring + stage * kStage + ((u * 2 + which) * kParts + e) * kPiece);
    return x;
  };
  const int first = begin + warp * kStep, stride = kWarps * kStep;
  if (first < stop) {
#pragma unroll
    for (int i = 0; i < kRowsStages - 1; ++i) ask(first + i * stride, i);
  }
  for (int base = first, stage = 0; base < stop; base += stride, stage = stage + 1 == kRowsStages ? 0 : stage + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRowsStages - 2) : "memory");
    // products of this lane's columns: value u R + r
    float s[kValues];
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      const P x(take(stage, u, 0));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 d = mul2(q[r][0], x.v[0]);
#pragma unroll
        for (int e = 1; e < kPairs; ++e) d = fma2(q[r][e], x.v[e], d);
        s[u * R + r] = d.x + d.y;
      }
    }
    // Summed over a state's lanes, halving what each lane keeps: the upper bits of a lane's number within its group are the upper bits of the
    // number of its value (the first two: u), and with more values than lanes it keeps some neighbouring ones.
    int left = kValues;
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) {
      if (left > 1) {
        left /= 2;
        const bool upper = (lane & d) != 0;
#pragma unroll
        for (int i = 0; i < kValues / 2; ++i) {
          if (i >= left) continue;
          const float mine = upper ? s[i + left] : s[i], other = upper ? s[i] : s[i + left];
          s[i] = mine + __shfl_xor_sync(~0u, other, d);
        }
      } else {
        s[0] += __shfl_xor_sync(~0u, s[0], d);
      }
    }
    // this lane's rows: maximum, weights
    const int at = base + (part / (kLanes / 4)) * kStates + lane / kLanes, mine = at >= stop ? -1 : at < leading ? at : all.lo + (at - leading);
    bool moved = false;
    float shrink[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      bool read = mine >= 0;
      if (!alike && read) {
        const Span own = spans[row0 + i];
        read = mine < own.sink || (mine >= own.lo && mine < own.hi);
      }
      if (!read) s[i] = -INFINITY;
      float most = larger_or_nan(s[i], __shfl_xor_sync(~0u, s[i], kLanes / 2));
      most = larger_or_nan(most, __shfl_xor_sync(~0u, most, kLanes / 4));
      most = larger_or_nan(top[i], most);
      if (most == INFINITY) most = NAN;  // (as inf - inf is)
      const bool same = most == top[i];
      moved |= !same;
      shrink[i] = same ? 1.0f : exp2_of(top[i] - most);
      s[i] = s[i] == -INFINITY ? 0.0f : exp2_of(s[i] - most);
      total[i] = fmaf(total[i], shrink[i], s[i]);
      top[i] = most;
    }
    const int group = lane & ~(kLanes - 1);
    if (__any_sync(~0u, moved)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float f = __shfl_sync(~0u, shrink[r % kOwn], group + lane_of(r));
#pragma unroll
        for (int e = 0; e < kPairs; ++e) acc[r][e] = mul2(acc[r][e], make_float2(f, f));
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      const P x(take(stage, u, 1));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = __shfl_sync(~0u, s[r % kOwn], group + lane_of(u * R + r));
#pragma unroll
        for (int e = 0; e < kPairs; ++e) acc[r][e] = fma2(make_float2(w, w), x.v[e], acc[r][e]);
      }
    }
    ask(base + (kRowsStages - 1) * stride, stage == 0 ? kRowsStages - 1 : stage - 1);  // (the place of the step before)
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // what this lane's rows have, to all lanes of the group
  float tops_of[R], totals_of[R];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    total[i] += __shfl_xor_sync(~0u, total[i], kLanes / 2);
    total[i] += __shfl_xor_sync(~0u, total[i], kLanes / 4);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    tops_of[r] = __shfl_sync(~0u, top[r % kOwn], (lane & ~(kLanes - 1)) + lane_of(r));
    totals_of[r] = __shfl_sync(~0u, total[r % kOwn], (lane & ~(kLanes - 1)) + lane_of(r));
  }
  // groups of a warp, then the warps
  const auto weight = [](float mine, float of_all) { return mine == -INFINITY ? 0.0f : exp2f(mine - of_all); };
#pragma unroll
  for (int d = kLanes; d < 32; d <<= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float other = __shfl_xor_sync(~0u, tops_of[r], d), most = larger_or_nan(tops_of[r], other);
      const float a = weight(tops_of[r], most), b = weight(other, most);
      tops_of[r] = most;
      totals_of[r] = totals_of[r] * a + __shfl_xor_sync(~0u, totals_of[r], d) * b;
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const float2 far = make_float2(__shfl_xor_sync(~0u, acc[r][e].x, d), __shfl_xor_sync(~0u, acc[r][e].y, d));
        acc[r][e] = fma2(far, make_float2(b, b), mul2(acc[r][e], make_float2(a, a)));
      }
    }
  if (lane < kLanes) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (lane == 0) tops[warp][r] = tops_of[r], totals[warp][r] = totals_of[r];
#pragma unroll
      for (int e = 0; e < kPairs; ++e) *(float2*)&sums[warp][r][part * 8 + 2 * e] = acc[r][e];
    }
  }
  __syncthreads();
  const long long number = (long long)p.R * p.T * p.Hq;
  for (int i = threadIdx.x; i < rows * DP; i += kRowsThreads) {
    const int r = i / DP, d = i % DP;
    float most = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = larger_or_nan(most, tops[w][r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = weight(tops[w][r], most);
      l += f * totals[w][r];
      o += f * sums[w][r][d];
    }
    const int token = p.by_G.quotient(r);
    const long long row = ((long long)n * p.T + token) * p.Hq + hk * p.G + (r - token * p.G);
    if (d < p.D) {
      if (p.splits > 1) p.part_o[(split * number + row) * p.D + d] = o;
      const float result = l == 0.0f ? 0.0f : o / l;
      if (p.splits == 1) ((T*)p.out)[row * p.D + d] = from_float<T>(result);
      if (p.splits == 1 && p.rest) p.rest[row * p.D + d] = from_float<__nv_bfloat16>(result - to_float(from_float<T>(result)));
    }
    if (d == 0) {
      if (p.splits > 1) {
        p.part_ml[(split * number + row) * 2] = most;
        p.part_ml[(split * number + row) * 2 + 1] = l;
      } else if (p.lse) {
        p.lse[row] = l == 0.0f ? -INFINITY : most + log2f(l);
      }
    }
  }
}

}  // namespace mvr
