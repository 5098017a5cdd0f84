// What the C ABI's attention calls (mvr_heads.cu, mvr_window.cu) share on the host: how work is cut into parts, kernels' shared memory,
// tensor maps, float operands in pieces.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "../../include/mvr.h"
#include "mvr_attn_fma.cuh"
#include "mvr_attn_tc.cuh"
#include "mvr_attn_tc_bwd.cuh"

namespace {

using namespace mvr;

bool head_dtype(int t) { return t == MVR_F32 || t == MVR_F16 || t == MVR_BF16; }

int launched() { return cudaGetLastError() == cudaSuccess ? MVR_OK : MVR_ERR_LAUNCH; }

constexpr int kMultiprocessors = 148;

long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

// What a kernel takes for one of its steps (a tile of rows against a tile of states), in us, measured: `full` of an SM with all the
// CTAs that it holds (`resident`), `alone` of a CTA by itself.
struct StepTime {
  int resident;
  double full, alone;
};

// A tile of rows against 128 states (forward, dq), and 128 states against a tile of rows (dk, dv); float arithmetic: tiles of its own.
inline StepTime states_step(bool tc, bool pieces, bool backward, bool wide, bool two_tiles) {
  if (pieces) return backward ? StepTime{1, 4.5, 4.5} : StepTime{2, 2.6, 4.0};
  if (!tc) return {2, 3.0, 4.0};
  if (backward) return wide ? StepTime{1, 2.0, 2.0} : StepTime{2, 1.25, 1.8};
  return two_tiles ? StepTime{1, 2.1, 2.1} : wide ? StepTime{2, 1.5, 1.8} : StepTime{4, 0.85, 1.5};
}
inline StepTime rows_step(bool tc, bool pieces, bool wide) {
  return pieces ? StepTime{1, 5.0, 5.0} : !tc ? StepTime{2, 5.0, 7.0} : wide ? StepTime{1, 2.6, 2.6} : StepTime{2, 1.7, 2.3};
}

// Parts into which to cut the `steps` steps of `ctas` CTAs so that they end soonest: the SMs' CTAs one after another at the full rate,
// or, where an SM has few, one CTA's own chain; 1 us a CTA for its beginning and end.  Where CTAs differ in length (`uneven`: lengths
// or a mask), half a part is lost at the end.  Joining takes 3 us and `join` us a part.
int best_parts(long long ctas, long long steps, const StepTime& t, double join, bool uneven) {
  int best = 1;
  double least = 0;
  for (long long s = 1; s <= std::min<long long>(64, std::max<long long>(1, steps)); ++s) {
    const long long per = cdiv(steps, s), on_sm = cdiv(ctas * s, kMultiprocessors), rounds = cdiv(on_sm, t.resident);
    if (s > 1 && cdiv(steps, per) < s) continue;  // a part would have nothing
    const double time = std::max(on_sm * (per * t.full + 1.0 / t.resident), rounds * (per * t.alone + 1.0)) + (uneven ? per * t.alone / 2 : 0) +
                        (s > 1 ? 3 + join * s : 0);
    if (s == 1 || time < 0.92 * least) best = (int)s, least = time;
  }
  return best;
}

// Scores (rows times states) from which float operands in pieces are worth the launches that make them.  (Forward and backward, 4 x 16
// rows over 1024 states, 4 heads of 32: 139 us, in float arithmetic 95; over 2048 states, 8 heads of 64: 146 and 239.)
constexpr double kPieceScores = 1 << 19;

bool rows_aligned(const void* base, const int64_t (&strides)[3], const mvr_attention* a) {
  const int64_t sizes[3] = {a->R, a->T, a->Hq};
  if ((uintptr_t)base % 16 != 0) return false;
  int64_t last = 0;
  for (int i = 0; i < 3; ++i) {
    if (sizes[i] <= 1) continue;
    if (strides[i] % 8 != 0 || strides[i] < 0 || strides[i] > INT64_MAX / 4 / sizes[i]) return false;
    last += (sizes[i] - 1) * strides[i];
  }
  return last / 8 < 0xffffffffLL;  // (rows are found by 32-bit numbers of 16 bytes)
}

// Lets a kernel have `smem` bytes of dynamic shared memory, once per device.  (The same limit in every call of a kernel: calls of
// several threads do not undo one another's.)
template <auto KERNEL>
bool shared_memory(size_t smem) {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (device < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

template <auto KERNEL, typename... A>
int launch_shared(dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  if (grid.x == 0 || grid.y == 0) return MVR_OK;
  if (!shared_memory<KERNEL>(smem)) return MVR_ERR_LAUNCH;
  launch_dependent(KERNEL, grid, dim3(threads), smem, st, args...);
  return launched();
}

unsigned blocks_of(long long n, int per) { return (unsigned)std::min<long long>(cdiv(n, per), 1 << 20); }

template <typename T>
int sum_parts(const float* part, void* dst, long long n, int parts, float factor, cudaStream_t st) {
  if (n == 0) return MVR_OK;
  if (n % 4 == 0 && (uintptr_t)dst % (4 * sizeof(T)) == 0)
    launch_dependent(attn_sum<T, 4>, dim3(blocks_of(n, 1024)), dim3(256), 0, st, part, (T*)dst, n, parts, factor);
  else
    launch_dependent(attn_sum<T, 1>, dim3(blocks_of(n, 256)), dim3(256), 0, st, part, (T*)dst, n, parts, factor);
  return launched();
}

template <typename T>
bool tensor_maps(const mvr_attention* a, bool backward, int pieces, TcMaps& maps, bool& boxes) {
  tc_need_context();
  const int D = (int)a->D, G = (int)(a->Hq / a->Hk);
  const auto states = [&](CUtensorMap* m, const void* base, const int64_t (&s)[3]) {
    return tc_map<T>(m, base, D, (int)a->Hk, (int)a->L, (int)a->N * pieces, s[2], s[1], s[0], 1, kTcBox);
  };
  if (!states(&maps.k, a->k, a->k_strides) || !states(&maps.v, a->v, a->v_strides)) return false;
  const int step = D <= 64 ? kGradStep<64> : kGradStep<128>;
  if (backward && !a->has_index && a->R > 0 && a->T > 0 && step % G == 0) {
    const auto rows = [&](CUtensorMap* m, const void* base, const int64_t (&s)[3]) {
      return tc_map<T>(m, base, D, (int)a->Hq, (int)a->T, (int)a->R * pieces, s[2], s[1], s[0], G, step / G);
    };
    boxes = rows(&maps.q, a->q, a->q_strides) && rows(&maps.g, a->grad_out, a->g_strides);
  }
  return true;
}

// Columns of the operands in memory, and where their pieces lie in the workspace.
struct OperandPieces {
  int W;
  long long q, k, v, g;
};

// Float operands of a call in pieces, in its workspace; `b` is the call on them.
int split_operands(const mvr_attention* a, bool backward, const OperandPieces& c, char* ws, mvr_attention& b, AttnParams& p, cudaStream_t st) {
  SplitCall call = {};
  int operands = 0;
  long long most = 0;
  const auto split = [&](const void* from, const int64_t (&s)[3], long long n0, long long n1, long long n2, long long to) {
    if (n0 * n1 * n2 == 0) return;
    call.of[operands++] = {(const float*)from, (long long)s[0], (long long)s[1], (long long)s[2], (int)n1, (int)n2, n0 * n1 * n2, (__nv_bfloat16*)(ws + to)};
    most = std::max(most, n0 * n1 * n2);
  };
  split(a->q, a->q_strides, a->R, a->T, a->Hq, c.q);
  split(a->k, a->k_strides, a->N, a->L, a->Hk, c.k);
  split(a->v, a->v_strides, a->N, a->L, a->Hk, c.v);
  if (backward) split(a->grad_out, a->g_strides, a->R, a->T, a->Hq, c.g);
  call.D = (int)a->D;
  call.W = c.W;
  if (operands > 0) launch_dependent(split_floats, dim3((unsigned)cdiv(most * (c.W / 8), 256), operands), dim3(256), 0, st, call);
  const int rc = launched();
  if (rc != MVR_OK) return rc;
  b = *a;
  b.D = c.W;
  b.q = ws + c.q; b.k = ws + c.k; b.v = ws + c.v; b.grad_out = ws + c.g;
  const int64_t W = c.W;
  for (int64_t(*s)[3] : {&b.q_strides, &b.g_strides}) (*s)[0] = a->T * a->Hq * W, (*s)[1] = a->Hq * W, (*s)[2] = W;
  for (int64_t(*s)[3] : {&b.k_strides, &b.v_strides}) (*s)[0] = a->L * a->Hk * W, (*s)[1] = a->Hk * W, (*s)[2] = W;
  p.q = b.q; p.k = b.k; p.v = b.v; p.g = b.grad_out;
  p.q_r = p.g_r = b.q_strides[0]; p.q_t = p.g_t = b.q_strides[1]; p.q_h = p.g_h = W;
  p.k_n = p.v_n = b.k_strides[0]; p.k_l = p.v_l = b.k_strides[1]; p.k_h = p.v_h = W;
  p.q_piece = p.g_piece = a->R * a->T * a->Hq * W;
  return MVR_OK;
}

}  // namespace
