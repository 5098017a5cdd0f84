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

struct DropoutParams {
  const void* x;
  const void* residual;  // or null
  void* out;
  long long n;
  unsigned cut;          // an element stays when its 16 bits are >= cut; 65536: none stays
  float scale;
  unsigned long long seed, offset;
  const unsigned long long* seed_at;  // or null; else the seed lies there, on the device
};

__device__ __forceinline__ uint4 philox(uint2 key, uint4 c) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c.x * 0xD2511F53u, b = (unsigned long long)c.z * 0xCD9E8D57u;
    c = make_uint4((unsigned)(b >> 32) ^ c.y ^ key.x, (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ key.y, (unsigned)a);
    key.x += 0x9E3779B9u;
    key.y += 0xBB67AE85u;
  }
  return c;
}

constexpr int kDropThreads = 256;

// A thread takes groups of eight consecutive elements.  VECTOR: x, residual and out are 16-byte aligned.
template <typename T, bool VECTOR, bool RESIDUAL>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  grid_dependency();
  const unsigned long long seed = p.seed_at ? *p.seed_at : p.seed;
  const uint2 key = make_uint2((unsigned)seed, (unsigned)(seed >> 32));
  const T* x = (const T*)p.x;
  const T* res = (const T*)p.residual;
  T* out = (T*)p.out;
  constexpr int kParts = sizeof(T) == 2 ? 1 : 2, kPart = 8 / kParts;
  typedef Vec<T, kPart> V;
  const long long groups = (p.n + 7) >> 3;
  for (long long g = (long long)blockIdx.x * kDropThreads + threadIdx.x; g < groups; g += (long long)gridDim.x * kDropThreads) {
    const long long e = g << 3;
    const bool whole = VECTOR && e + 8 <= p.n;
    alignas(16) T xv[8];
    alignas(16) T rv[8];
    if (whole) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        *(V*)(xv + k * kPart) = *(const V*)(x + e + k * kPart);
        if (RESIDUAL) *(V*)(rv + k * kPart) = *(const V*)(res + e + k * kPart);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = e + k < p.n;
        xv[k] = in ? x[e + k] : from_float<T>(0.0f);
        if (RESIDUAL) rv[k] = in ? res[e + k] : from_float<T>(0.0f);
      }
    }
    const uint4 r = philox(key, make_uint4((unsigned)g, (unsigned)(g >> 32), (unsigned)p.offset, (unsigned)(p.offset >> 32)));
    const unsigned word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned bits = (k & 1) ? word[k >> 1] >> 16 : word[k >> 1] & 0xffffu;
      // a dropped element gives 0 whatever it held, NaN and infinities included
      float v = bits >= p.cut ? to_float(xv[k]) * p.scale : 0.0f;
      if (RESIDUAL) v += to_float(rv[k]);
      xv[k] = from_float<T>(v);
    }
    if (whole) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) *(V*)(out + e + k * kPart) = *(const V*)(xv + k * kPart);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < p.n) out[e + k] = xv[k];
    }
  }
}

template <typename T>
cudaError_t launch_dropout(const DropoutParams& p, cudaStream_t st) {
  const long long groups = (p.n + 7) >> 3, want = (groups + kDropThreads - 1) / kDropThreads;
  const dim3 grid((unsigned)(want < (1LL << 30) ? want : (1LL << 30)));
  const bool vec = (((uintptr_t)p.x | (uintptr_t)p.out | (uintptr_t)p.residual) & 15) == 0;
  if (vec) return p.residual ? launch_dependent(dropout_kernel<T, true, true>, grid, kDropThreads, 0, st, p)
                             : launch_dependent(dropout_kernel<T, true, false>, grid, kDropThreads, 0, st, p);
  return p.residual ? launch_dependent(dropout_kernel<T, false, true>, grid, kDropThreads, 0, st, p)
                    : launch_dependent(dropout_kernel<T, false, false>, grid, kDropThreads, 0, st, p);
}

}  // namespace mvr
