// Element types of the head operators (float, half, bfloat16): conversions, 16-byte vectors, launches as programmatic dependents.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mvr {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Pairs of floats in one instruction each.
__device__ __forceinline__ unsigned long long bits_of(float2 a) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 pair_of(unsigned long long b) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(b));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return pair_of(r);
}

// Two neighbouring elements: as floats, rounded from floats, and the larger of each (NaN is not seen).
template <typename T>
struct Two {
  T v[2];
};
template <> struct alignas(4) Two<__half> { __half2 v; };
template <> struct alignas(4) Two<__nv_bfloat16> { __nv_bfloat162 v; };
template <> struct alignas(8) Two<float> { float2 v; };
__device__ __forceinline__ float2 floats(Two<float> a) { return a.v; }
__device__ __forceinline__ float2 floats(Two<__half> a) { return __half22float2(a.v); }
__device__ __forceinline__ float2 floats(Two<__nv_bfloat16> a) { return __bfloat1622float2(a.v); }
template <typename T> __device__ __forceinline__ Two<T> rounded(float2 f);
template <> __device__ __forceinline__ Two<float> rounded<float>(float2 f) { return {f}; }
template <> __device__ __forceinline__ Two<__half> rounded<__half>(float2 f) { return {__float22half2_rn(f)}; }
template <> __device__ __forceinline__ Two<__nv_bfloat16> rounded<__nv_bfloat16>(float2 f) { return {__float22bfloat162_rn(f)}; }
__device__ __forceinline__ Two<float> larger(Two<float> a, Two<float> b) { return {make_float2(fmaxf(a.v.x, b.v.x), fmaxf(a.v.y, b.v.y))}; }
__device__ __forceinline__ Two<__half> larger(Two<__half> a, Two<__half> b) { return {__hmax2(a.v, b.v)}; }
__device__ __forceinline__ Two<__nv_bfloat16> larger(Two<__nv_bfloat16> a, Two<__nv_bfloat16> b) { return {__hmax2(a.v, b.v)}; }
template <typename T> __device__ __forceinline__ Two<T> both(float f) { return rounded<T>(make_float2(f, f)); }

// N consecutive elements, loaded and stored as one access of their size (at most 16 bytes each).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
  T v[N];
};

// What precedes the kernel in its stream has ended completely, and its writes are visible; the next kernel may become resident.
__device__ __forceinline__ void grid_dependency() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launch as a programmatic dependent: the kernel may become resident while its predecessor ends.  Every kernel launched like this
// calls grid_dependency() before its first access to memory.
template <typename... A, typename... B>
cudaError_t launch_dependent(void (*kernel)(A...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, B&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<A>(args)...);
}

}  // namespace mvr
