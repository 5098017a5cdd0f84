// Fifth-generation tensor cores, tensor memory and TMA of sm_100a as the attention kernels use them: thin wrappers of the PTX
// instructions, shared-memory and instruction descriptors, bounded waits.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mvr_types.cuh"

namespace mvr {

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers ----------------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One arrival of a warp, behind what all its lanes did before (an arrival of every lane is 32 accesses, one after another).
__device__ __forceinline__ void bar_arrive_warp(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "  selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long nanoseconds() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

constexpr unsigned long long kWaitLimit = 2000000000ull;  // 2 s: far above any wait of a call that makes progress

// Waits until the phase of the given parity has completed; false when it has not within the limit, or another thread of the CTA
// has given up (`lost`, in shared memory).
static __device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* lost) {
  const unsigned long long begin = nanoseconds();
  for (;;) {
    if (*lost) return false;
    for (int i = 0; i < 32; ++i)
      if (bar_try(bar, parity)) return true;
    if (nanoseconds() - begin > kWaitLimit) *lost = 1;
  }
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* lost) {
  return bar_try(bar, parity) || bar_wait_slow(bar, parity, lost);
}

// The same by a whole warp, with one answer.
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* lost) {
  return __all_sync(~0u, bar_wait(bar, parity, lost));
}
// A wait whose outcome is not looked at: once given up, every later wait ends at once, and the kernel runs to its end on whatever lies
// in its buffers, always within them, and stores nothing.  (A vote about each outcome took a tenth of the kernels' time.)
__device__ __forceinline__ void bar_pass(uint32_t bar, uint32_t parity, volatile int* lost) {
  if (!bar_try(bar, parity)) bar_wait_slow(bar, parity, lost);
  __syncwarp();
}

// One lane of a converged warp.  (The products and copies below take their operands from registers that a warp shares: in a branch
// that elect.sync guards the compiler knows that one thread runs; behind a comparison of the lane it would issue them in a loop over
// the lanes.)
__device__ __forceinline__ bool elect_one() {
  uint32_t lane = 0, is = 0;
  asm volatile(
      "{\n"
      "  .reg .b32 r;\n"
      "  .reg .pred p;\n"
      "  elect.sync r|p, %2;\n"
      "  @p mov.s32 %1, 1;\n"
      "  mov.s32 %0, r;\n"
      "}\n"
      : "+r"(lane), "+r"(is)
      : "r"(0xffffffffu));
  return is != 0;
}

// Writes of this thread to shared memory become visible to TMA and the tensor cores.
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- TMA ----------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// ---- tensor memory ------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t to_smem, int columns) {  // one whole warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_smem), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, int columns) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: column i in v[i].  Valid after tmem_wait_load().
__device__ __forceinline__ void tmem_load32(uint32_t (&v)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// ---- products -----------------------------------------------------------------------------------------
// Shared-memory operands are tiles of rows of 128 bytes (64 elements) in TMA's 128-byte swizzle; the tile starts at a multiple of
// 1024 bytes.  K along the row (K-major): 8-row groups are 1024 bytes apart, and 16 elements further is 32 bytes further.  K down
// the rows (MN-major): 8-row groups 1024 bytes apart again, the next 64 elements of M or N are `block` bytes away, and 16 rows
// further is 2048 bytes further.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t at) {
  return (uint64_t)((at & 0x3ffff) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t at, uint32_t block) {
  return (uint64_t)((at & 0x3ffff) >> 4) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <typename T> struct TcType;
template <> struct TcType<__half> {
  static constexpr uint32_t code = 0;
  static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
};
template <> struct TcType<__nv_bfloat16> {
  static constexpr uint32_t code = 1;
  static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
};

// Instruction descriptor: float sums of products of two operands of type T, 128 x n.
template <typename T>
__device__ __forceinline__ uint32_t tc_shape(int n, bool b_mn_major, bool negate_a = false) {
  return (1u << 4) | (TcType<T>::code << 7) | (TcType<T>::code << 10) | ((negate_a ? 1u : 0u) << 13) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

template <int N> struct Number { static constexpr int value = N; };

// d (+)= a b, 16 deep; a in shared memory (SS) or tensor memory (TS).  One thread.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.u32 p, %4, 0;\n"
      "  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.u32 p, %4, 0;\n"
      "  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"(add ? 1u : 0u)
      : "memory");
}
// d (+)= a b over `depth` sixteens of K-major tiles in blocks of 64 elements a row, `block_a` and `block_b` bytes each.
template <int MOST>
__device__ __forceinline__ void mma_rows(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, int depth, uint32_t block_a, uint32_t block_b,
                                         bool add = false) {
  const auto step = [&](int k) {
    mma_ss(d, a + (((k >> 2) * block_a + (k & 3) * 32) >> 4), b + (((k >> 2) * block_b + (k & 3) * 32) >> 4), shape, add || k > 0);
  };
  const auto steps = [&](auto n) {  // (a number the compiler knows: a loop issues at half the rate)
#pragma unroll
    for (int k = 0; k < decltype(n)::value; ++k) step(k);
  };
  if (depth == MOST) {
    steps(Number<MOST>());
  } else if (depth == MOST / 2) {
    steps(Number<MOST / 2>());
  } else {
    for (int k = 0; k < depth; ++k) step(k);
  }
}
// Arrives at the barrier once when all products issued before by this thread are complete.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x of two numbers up to 64 on the arithmetic pipes, where the units for functions are the limit: x = n + f with f within a half,
// a polynomial of degree 4 for 2^f (its relative error is nearly the same at all its extremes, 2.55e-6 to 2.65e-6: a hundredth of a
// half step of float16), times 2^n.  -inf, and whatever lies below, gives about 2^-126; NaN stays.
__device__ __forceinline__ float2 exp2_polynomial(float2 x) {
  const float2 magic = make_float2(12582912.0f, 12582912.0f);  // 1.5 2^23: its sum with x ends in n
  x = make_float2(max_nan(x.x, -126.0f), max_nan(x.y, -126.0f));
  const float2 n = add2(x, magic), f = fma2(add2(n, make_float2(-12582912.0f, -12582912.0f)), make_float2(-1.0f, -1.0f), x);
  float2 p = fma2(f, make_float2(0.009570100344717503f, 0.009570100344717503f), make_float2(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  return mul2(p, make_float2(__int_as_float((__float_as_int(n.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(n.y) << 23) + 0x3f800000)));
}

// The largest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---- float operands in pieces --------------------------------------------------------------------------
// A float is the exact sum of three bfloat16 numbers, its 24 bits eight at a time (cut off, so that no piece overflows).  A product of
// two floats is that of their pieces; of the nine, the three whose size is 2^-24 of the product or less are left out: six products of
// bfloat16 operands, summed in float, for one of float operands.  (200 regions' queries, 4 heads of 64, over three images of 13 635
// states, forward and backward: 0.30 ms, of which the cutting into pieces, bound by memory, is a quarter; in float arithmetic 0.51 ms.
// Errors against float64 2.9e-7 to 5.3e-7; the plain float form has 2.5e-7 to 7.7e-7.)
template <int PIECES, typename F>
__device__ __forceinline__ void for_pairs(F&& f) {  // f(piece of a, piece of b, is it the first): small products first
  if constexpr (PIECES == 1) {
    f(0, 0, true);
  } else {
    f(1, 1, true);
    f(0, 2, false);
    f(2, 0, false);
    f(0, 1, false);
    f(1, 0, false);
    f(0, 0, false);
  }
}
// Two floats as the three words of their pieces.
__device__ __forceinline__ void pieces_of(float2 f, uint32_t& a, uint32_t& b, uint32_t& c) {
  const float2 neg = make_float2(-1.0f, -1.0f);
  a = __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
  f = fma2(make_float2(__uint_as_float(__float_as_uint(f.x) & 0xffff0000u), __uint_as_float(__float_as_uint(f.y) & 0xffff0000u)), neg, f);
  b = __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
  f = fma2(make_float2(__uint_as_float(__float_as_uint(f.x) & 0xffff0000u), __uint_as_float(__float_as_uint(f.y) & 0xffff0000u)), neg, f);
  c = pack2<__nv_bfloat16>(f.x, f.y);
}

// Rows of D floats (three outer dimensions with strides) as pieces: to[piece][row][W], W: D rounded up to 8, zeros behind D.  A thread
// takes eight columns.  An infinity is the largest bfloat16 of its sign, 0 and the infinity: the third piece meets nothing but the other
// operand's first, so that no 0 among that one's smaller pieces makes a NaN of an infinite product, and the first piece gives infinity
// times infinity.  NaN is the third piece alone.
struct SplitFloats {
  const float* from;
  long long s0, s1, s2;
  int n1, n2;
  long long rows;
  __nv_bfloat16* to;
};
struct SplitCall {
  SplitFloats of[4];  // blockIdx.y: a call's operands in one launch
  int D, W;
};
static __global__ void __launch_bounds__(256) split_floats(const __grid_constant__ SplitCall call) {
  grid_dependency();
  const SplitFloats& t = call.of[blockIdx.y];
  const int W = call.W, D = call.D;
  const long long rows = t.rows, id = (long long)blockIdx.x * 256 + threadIdx.x, row = id / (W / 8);
  if (row >= rows) return;
  const int col = (int)(id - row * (W / 8)) * 8;
  const long long i01 = row / t.n2, i0 = i01 / t.n1;
  const float* src = t.from + i0 * t.s0 + (i01 - i0 * t.n1) * t.s1 + (row - i01 * t.n2) * t.s2 + col;
  __nv_bfloat16* to = t.to;
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = col + k < D ? src[k] : 0.0f;
  uint32_t w[3][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    pieces_of(make_float2(f[2 * k], f[2 * k + 1]), w[0][k], w[1][k], w[2][k]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (!(fabsf(f[2 * k + h]) < INFINITY)) {  // (infinity less itself is no number)
        const uint32_t sign = (__float_as_uint(f[2 * k + h]) >> 16) & 0x8000, keep = h ? 0xffffu : 0xffff0000u;
        const bool nan = f[2 * k + h] != f[2 * k + h];
        w[0][k] = (w[0][k] & keep) | ((nan ? 0u : sign | 0x7f7f) << (16 * h));
        w[1][k] &= keep;
        w[2][k] = (w[2][k] & keep) | ((nan ? 0x7fffu : sign | 0x7f80) << (16 * h));
      }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) *(uint4*)(to + (k * rows + row) * W + col) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}

// ---- host ---------------------------------------------------------------------------------------------
typedef CUresult (*TcEncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline void* tc_driver_function(const char* name) {
  void* ptr = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint(name, &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  return ptr;
}
inline TcEncodeTiled tc_encoder() {
  static TcEncodeTiled fn = (TcEncodeTiled)tc_driver_function("cuTensorMapEncodeTiled");
  return fn;
}
// Makes the runtime's context current in a thread that has not called CUDA yet (autograd's threads, a data loader's): a tensor map
// cannot be made without one.
inline void tc_need_context() {
  static CUresult (*const current)(CUcontext*) = (CUresult(*)(CUcontext*))tc_driver_function("cuCtxGetCurrent");
  CUcontext context = nullptr;
  int device = 0;
  if (current && current(&context) == CUDA_SUCCESS && context) return;
  if (cudaGetDevice(&device) == cudaSuccess) cudaSetDevice(device);
  cudaGetLastError();
}

// Map over (D, heads, rows, images), D contiguous elements of 2 bytes, boxes of 64 elements x `box_heads` x `box_rows`; false where
// TMA cannot describe the tensor.
template <typename T>
bool tc_map(CUtensorMap* map, const void* base, int D, int heads, int rows, int images, long long s_head, long long s_row,
            long long s_image, int box_heads, int box_rows) {
  TcEncodeTiled encode = tc_encoder();
  if (!encode || (uintptr_t)base % 16 != 0) return false;
  // a dimension of one element may have any stride
  if (heads == 1) s_head = D;
  if (rows == 1) s_row = D;
  if (images == 1) s_image = D;
  for (long long s : {s_head, s_row, s_image})
    if (s <= 0 || s % 8 != 0 || s * 2 >= (1LL << 40)) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)images};
  const cuuint64_t strides[3] = {(cuuint64_t)s_head * 2, (cuuint64_t)s_row * 2, (cuuint64_t)s_image * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows, 1}, step[4] = {1, 1, 1, 1};
  return encode(map, TcType<T>::tma, 4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mvr
