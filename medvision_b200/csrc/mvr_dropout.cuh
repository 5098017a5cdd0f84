// Dropout from a counter-based generator: out[e] = residual[e] + (kept(e) ? x[e] * scale : 0).
//
// kept(e) is a function of (seed, offset, e) alone, so no mask is stored: the gradient calls the same kernel on the output's
// gradient.  The generator is Philox 4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) with
// key = seed and counter = (e / 8, offset).  An element takes 16 of the 128 bits, so one evaluation serves the eight elements that a
// thread loads as one 16-byte vector: 10 rounds of two 32x32->64 products for 8 elements keep the arithmetic below the memory's
// time; at 32 bits an element it would be above it for 2-byte types.  The probability is therefore a multiple of 2^-16 (off by at
// most 2^-17), and the scale is the inverse of the probability that results, so that the expectation is exact.
//
// Measured: 27.9 M bfloat16 elements with a residual 30 us (5.5 TB/s), their gradient 23 us (4.8 TB/s); 33.6 M float16 elements 26 us
// (5.1 TB/s): 85, 73 and 78 % of a plain copy's rate.  Half of the issue slots are busy with the generator's products beside the loads.
#pragma once
#include "mvr_types.cuh"

namespace mvr {

struct PhiloxKeys {
  unsigned x[10], y[10];  // of the rounds

  __host__ __device__ __forceinline__ void from(unsigned long long seed) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      x[r] = (unsigned)seed + r * 0x9E3779B9u;
      y[r] = (unsigned)(seed >> 32) + r * 0xBB67AE85u;
    }
  }
};

struct DropoutParams {
  const void* x;
  const void* residual;  // or null
  void* out;
  long long n;
  unsigned floor;        // an element stays when its 16 bits, as the upper half of a word, are >= this
  float scale;
  PhiloxKeys keys;       // constants of the launch, so that a round is two products and two three-way exclusive ors
  unsigned long long offset;
  const unsigned long long* seed_at;  // or null; else the seed lies there, on the device
};

// `low`, `high`: the counter's first two words; `offset` (and `high`, which is the CTA's) are the same in all threads, and with them
// the second product of the first round and the first of the second.
__device__ __forceinline__ uint4 philox(const PhiloxKeys& k, unsigned low, unsigned high, unsigned long long offset) {
  uint4 c = make_uint4(low, high, (unsigned)offset, (unsigned)(offset >> 32));
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c.x * 0xD2511F53u, b = (unsigned long long)c.z * 0xCD9E8D57u;
    c = make_uint4((unsigned)(b >> 32) ^ c.y ^ k.x[r], (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ k.y[r], (unsigned)a);
  }
  return c;
}

constexpr int kDropThreads = 256, kDropGroups = 4;

// A thread takes kDropGroups groups of eight consecutive elements, a CTA's width apart, all their loads under way together.
// VECTOR: x, residual and out are 16-byte aligned.  DEVICE: the seed lies on the device.
template <typename T, bool VECTOR, bool RESIDUAL, bool DEVICE>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  grid_dependency();
  PhiloxKeys own;
  if (DEVICE) own.from(*p.seed_at);
  // A CTA's elements: a place of 64 bits that is the CTA's, and one of 32 that is the thread's.
  constexpr int kGroups = kDropGroups * kDropThreads;
  const long long group0 = (long long)blockIdx.x * kGroups, e0 = group0 * 8;
  const int left = (int)(p.n - e0 < 8 * kGroups ? p.n - e0 : 8 * kGroups);  // elements from there on
  const T* x = (const T*)p.x + e0;
  const T* res = (const T*)p.residual + e0;
  T* out = (T*)p.out + e0;
  constexpr int kParts = sizeof(T) == 2 ? 1 : 2, kPart = 8 / kParts;
  typedef Vec<T, kPart> V;
  V xv[kDropGroups][kParts], rv[kDropGroups][kParts];
  const bool full = VECTOR && left == 8 * kGroups;  // (the same in all threads)
  if (full) {
#pragma unroll
    for (int i = 0; i < kDropGroups; ++i) {
      const int e = (threadIdx.x + i * kDropThreads) * 8;
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        xv[i][k] = *(const V*)(x + e + k * kPart);
        if (RESIDUAL) rv[i][k] = *(const V*)(res + e + k * kPart);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kDropGroups; ++i) {
      const int e = (threadIdx.x + i * kDropThreads) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = e + k < left;
        xv[i][k / kPart].v[k % kPart] = in ? x[e + k] : from_float<T>(0.0f);
        if (RESIDUAL) rv[i][k / kPart].v[k % kPart] = in ? res[e + k] : from_float<T>(0.0f);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kDropGroups; ++i) {
    const int e = (threadIdx.x + i * kDropThreads) * 8;
    // (a CTA's groups begin at a multiple of their number: no carry)
    const uint4 r = philox(DEVICE ? own : p.keys, (unsigned)group0 + threadIdx.x + i * kDropThreads, (unsigned)(group0 >> 32), p.offset);
    const unsigned word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool stays = ((k & 1) ? word[k >> 1] : word[k >> 1] << 16) >= p.floor;
      // a dropped element gives 0 whatever it held, NaN and infinities included
      float v = stays ? to_float(xv[i][k / kPart].v[k % kPart]) * p.scale : 0.0f;
      if (RESIDUAL) v += to_float(rv[i][k / kPart].v[k % kPart]);
      xv[i][k / kPart].v[k % kPart] = from_float<T>(v);
    }
    if (full) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) *(V*)(out + e + k * kPart) = xv[i][k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < left) out[e + k] = xv[i][k / kPart].v[k % kPart];
    }
  }
}

// 0, or 1: more CTAs than a grid has.
template <typename T>
int launch_dropout(const DropoutParams& p, cudaStream_t st) {
  const long long per = 8LL * kDropGroups * kDropThreads, ctas = (p.n + per - 1) / per;
  if (ctas > 0x7fffffffLL) return 1;
  const dim3 grid((unsigned)ctas);
  const bool vec = (((uintptr_t)p.x | (uintptr_t)p.out | (uintptr_t)p.residual) & 15) == 0;
  const auto go = [&](auto kernel) { launch_dependent(kernel, grid, kDropThreads, 0, st, p); };
  if (p.seed_at) {
    if (vec) p.residual ? go(dropout_kernel<T, true, true, true>) : go(dropout_kernel<T, true, false, true>);
    else p.residual ? go(dropout_kernel<T, false, true, true>) : go(dropout_kernel<T, false, false, true>);
  } else {
    if (vec) p.residual ? go(dropout_kernel<T, true, true, false>) : go(dropout_kernel<T, true, false, false>);
    else p.residual ? go(dropout_kernel<T, false, true, false>) : go(dropout_kernel<T, false, false, false>);
  }
  return 0;
}

}  // namespace mvr
