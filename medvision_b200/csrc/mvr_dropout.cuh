// Dropout from a counter-based generator: out[e] = residual[e] + (kept(e) ? x[e] * scale : 0).
//
// kept(e) is a function of (seed, offset, e) alone, so no mask is stored: the gradient calls the same kernel on the output's
// gradient.  The generator is Philox 4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) with
// key = seed and counter = (e / 8, offset).  An element takes 16 of the 128 bits, so one evaluation serves the eight elements that a
// thread loads as one 16-byte vector: 10 rounds of two 32x32->64 products for 8 elements keep the arithmetic below the memory's
// time; at 32 bits an element it would be above it for 2-byte types.  The probability is therefore a multiple of 2^-16 (off by at
// most 2^-17), and the scale is the inverse of the probability that results, so that the expectation is exact.
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

__device__ __forceinline__ uint4 philox(const PhiloxKeys& k, uint4 c) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c.x * 0xD2511F53u, b = (unsigned long long)c.z * 0xCD9E8D57u;
    c = make_uint4((unsigned)(b >> 32) ^ c.y ^ k.x[r], (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ k.y[r], (unsigned)a);
  }
  return c;
}

constexpr int kDropThreads = 256, kDropGroups = 2;

// A thread takes kDropGroups groups of eight consecutive elements, a CTA's width apart, all their loads under way together.
// VECTOR: x, residual and out are 16-byte aligned.  DEVICE: the seed lies on the device.
template <typename T, bool VECTOR, bool RESIDUAL, bool DEVICE>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  grid_dependency();
  PhiloxKeys own;
  if (DEVICE) own.from(*p.seed_at);
  const T* x = (const T*)p.x;
  const T* res = (const T*)p.residual;
  T* out = (T*)p.out;
  constexpr int kParts = sizeof(T) == 2 ? 1 : 2, kPart = 8 / kParts;
  typedef Vec<T, kPart> V;
  const long long first = ((long long)blockIdx.x * kDropGroups * kDropThreads + threadIdx.x) << 3;
  V xv[kDropGroups][kParts], rv[kDropGroups][kParts];
  bool whole[kDropGroups];
#pragma unroll
  for (int i = 0; i < kDropGroups; ++i) {
    const long long e = first + i * kDropThreads * 8;
    whole[i] = VECTOR && e + 8 <= p.n;
    if (whole[i]) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        xv[i][k] = *(const V*)(x + e + k * kPart);
        if (RESIDUAL) rv[i][k] = *(const V*)(res + e + k * kPart);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = e + k < p.n;
        xv[i][k / kPart].v[k % kPart] = in ? x[e + k] : from_float<T>(0.0f);
        if (RESIDUAL) rv[i][k / kPart].v[k % kPart] = in ? res[e + k] : from_float<T>(0.0f);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kDropGroups; ++i) {
    const long long e = first + i * kDropThreads * 8, g = e >> 3;
    const uint4 r = philox(DEVICE ? own : p.keys, make_uint4((unsigned)g, (unsigned)(g >> 32), (unsigned)p.offset, (unsigned)(p.offset >> 32)));
    const unsigned word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool stays = ((k & 1) ? word[k >> 1] : word[k >> 1] << 16) >= p.floor;
      // a dropped element gives 0 whatever it held, NaN and infinities included
      float v = stays ? to_float(xv[i][k / kPart].v[k % kPart]) * p.scale : 0.0f;
      if (RESIDUAL) v += to_float(rv[i][k / kPart].v[k % kPart]);
      xv[i][k / kPart].v[k % kPart] = from_float<T>(v);
    }
    if (whole[i]) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) *(V*)(out + e + k * kPart) = xv[i][k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < p.n) out[e + k] = xv[i][k / kPart].v[k % kPart];
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
