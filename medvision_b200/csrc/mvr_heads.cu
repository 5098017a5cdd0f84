// C ABI of the operators behind the roi modules (declared in include/mvr.h): attention to an encoder's states, dropout,
// log-probabilities of labels.  Argument checks, kernel selection and launches; no torch types, device pointers and sizes only.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "../../include/mvr.h"
#include "mvr_attn_fma.cuh"
#include "mvr_attn_tc.cuh"
#include "mvr_attn_tc_bwd.cuh"
#include "mvr_dropout.cuh"
#include "mvr_logprob.cuh"

namespace {

using namespace mvr;

bool head_dtype(int t) { return t == MVR_F32 || t == MVR_F16 || t == MVR_BF16; }

int launched() { return cudaGetLastError() == cudaSuccess ? MVR_OK : MVR_ERR_LAUNCH; }

// ---- attention ----------------------------------------------------------------------------------------

constexpr int kMultiprocessors = 148;
constexpr size_t kPlanShared = 200 * 1024;

// How a call is cut into CTAs, and what lies where in its workspace.
struct AttnCut {
  bool tc;                      // tensor cores (mvr_attn_tc.cuh); float operands in pieces
  bool direct;                  // few regions: the kernel finds those of an image itself
  int W;                        // columns of the operands in memory
  int tile, kv_tile;            // rows and states of a CTA's tile
  long long row_tiles;          // tiles of rows per key head: exact without an index, else no call has more
  int splits, row_splits;
  long long order, starts, tiles, delta, norm, peaks, row_peaks, q, k, v, g, part_o, part_ml, part_gq, part_gk, part_gv, bytes;
};

long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

// What a kernel takes for one of its steps (a tile of rows against a tile of states), in us, measured: `full` of an SM with all the
// CTAs that it holds (`resident`), `alone` of a CTA by itself.
struct StepTime {
  int resident;
  double full, alone;
};

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

AttnCut cut_attention(const mvr_attention* a, bool backward, bool tc) {
  AttnCut c = {};
  c.tc = tc;
  const bool pieces = tc && a->dtype == MVR_F32;
  c.W = (int)(pieces ? cdiv(a->D, 8) * 8 : a->D);
  const long long per = a->T * (a->Hq / a->Hk), rows = a->R * a->T * a->Hq;
  const long long rows_of_image = a->has_index ? cdiv(a->R * per, std::max<int64_t>(1, a->N)) : per;
  c.tile = tc ? (rows_of_image > kTcRows && !backward && a->D > 64 ? 2 * kTcRows : kTcRows) : a->D <= 128 ? 64 : 32;
  c.kv_tile = tc ? 128 : c.tile;  // (some kernels walk half of that at a time)
  c.row_tiles = a->has_index ? cdiv(a->R * per, c.tile) + std::min(a->N + 1, a->R) : a->R * cdiv(per, c.tile);
  c.direct = tc && !backward && a->has_index && a->R * per <= kTcRows && a->N <= 256;
  if (c.direct) c.row_tiles = a->N + 1;
  const long long kv_tiles = std::max<long long>(1, cdiv(a->L, c.kv_tile));
  const long long expected = std::max<long long>(1, a->has_index ? cdiv(rows_of_image, c.tile) * a->N : c.row_tiles) * a->Hk;
  const bool wide = a->D > 64, uneven = a->lengths || a->mask;
  const StepTime walk = pieces ? (backward ? StepTime{1, 4.5, 4.5} : StepTime{2, 2.6, 4.0}) : !tc ? StepTime{2, 3.0, 4.0} : backward ? (wide ? StepTime{1, 2.0, 2.0} : StepTime{2, 1.25, 1.8})
                        : c.tile > kTcRows ? StepTime{1, 2.1, 2.1} : wide ? StepTime{2, 1.5, 1.8} : StepTime{4, 0.85, 1.5};
  // (a part's sums are written and read at 4 MB/us)
  c.splits = best_parts(expected, kv_tiles, walk, rows * a->D * 8 / 4e6, uneven);
  if (tc) c.splits = (int)std::max<long long>(c.splits, cdiv(a->L, kTcMaxStates));
  const StepTime walk_rows = pieces ? StepTime{1, 5.0, 5.0} : !tc ? StepTime{2, 5.0, 7.0} : wide ? StepTime{1, 2.6, 2.6} : StepTime{2, 1.7, 2.3};
  c.row_splits = backward ? best_parts(a->N * a->Hk * kv_tiles, cdiv(rows_of_image, c.tile), walk_rows, (double)a->N * a->L * a->Hk * a->D * 16 / 4e6, false)
                          : 1;
  long long at = 0;
  const auto take = [&at](long long bytes) {
    const long long here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (a->has_index && !c.direct) {
    c.order = take(a->R * 4);
    c.starts = take((a->N + 2) * 4);
    c.tiles = take((a->N + 2) * 4);
  }
  if (pieces) {
    c.q = take(rows * c.W * 6);
    c.k = take(a->N * a->L * a->Hk * c.W * 6);
    c.v = take(a->N * a->L * a->Hk * c.W * 6);
    if (backward) c.g = take(rows * c.W * 6);
  }
  if (backward) {
    c.delta = take(rows * 4);
    if (tc && a->dtype == MVR_F16) {
      c.norm = take(rows * 4);
      c.peaks = take(a->N * a->Hk * 4);
      c.row_peaks = take(c.row_tiles * a->Hk * 8);
    }
    if (c.splits > 1) c.part_gq = take(c.splits * rows * a->D * 4);
    if (c.row_splits > 1) {
      c.part_gk = take(c.row_splits * a->N * a->L * a->Hk * a->D * 4);
      c.part_gv = take(c.row_splits * a->N * a->L * a->Hk * a->D * 4);
    }
  } else if (c.splits > 1) {
    c.part_o = take(c.splits * rows * a->D * 4);
    c.part_ml = take(c.splits * rows * 8);
  }
  c.bytes = at;
  return c;
}

// Scores (rows times states) from which float operands in pieces are worth the launches that make them.  (Forward and backward, 4 x 16
// rows over 1024 states, 4 heads of 32: 139 us, in float arithmetic 95; over 2048 states, 8 heads of 64: 146 and 239.)
constexpr double kPieceScores = 1 << 19;

// Whether type and sizes are the tensor cores'; the operands' alignment is a matter of the call.
bool tc_sizes(const mvr_attention* a) {
  const double rows = (double)a->R * a->T * a->Hq;
  if (a->L == 0 || a->N == 0 || a->L > 64LL * kTcMaxStates || a->N > INT32_MAX / 4 || rows > 2e9) return false;
  return a->dtype == MVR_F32 ? a->D <= 64 && rows * a->L >= kPieceScores : a->D % 8 == 0 && a->D <= 128;
}
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

int check_attention(const mvr_attention* a, bool backward, bool sizes_only) {
  if (!a) return MVR_ERR_NULL;
  if (!head_dtype(a->dtype)) return MVR_ERR_DTYPE;
  if (a->R < 0 || a->T < 0 || a->Hq < 1 || a->Hk < 1 || a->N < 0 || a->L < 0 || a->D < 1) return MVR_ERR_SHAPE;
  if (a->Hq % a->Hk != 0) return MVR_ERR_HEADS;
  if (a->D > 256) return MVR_ERR_HEAD_SIZE;
  if (!a->has_index && a->R != a->N) return MVR_ERR_SHAPE;
  const long long most = INT32_MAX / 4;
  if (a->R > most || a->T > most || a->Hq > 65535 || a->Hk > 65535 || a->N > most || a->L > most) return MVR_ERR_TOO_LARGE;
  if (a->T > 0 && a->R > 0 && a->R * a->T > most / (a->Hq / a->Hk)) return MVR_ERR_TOO_LARGE;  // rows of a key head: 32 bits
  if (a->R * a->T * a->Hq * a->D / 256 > INT32_MAX - 1) return MVR_ERR_TOO_LARGE;  // CTAs of the small kernels
  if (a->has_index && (size_t)(a->N + 1) * 8 > kPlanShared) return MVR_ERR_TOO_LARGE;
  if (cdiv(a->L, 32) * a->N > INT32_MAX) return MVR_ERR_TOO_LARGE;
  if (sizes_only) return MVR_OK;
  const bool any_rows = a->R > 0 && a->T > 0, any_states = a->N > 0 && a->L > 0;
  if (a->has_index && (a->index_type < MVR_INDEX_F32 || a->index_type > MVR_INDEX_U8)) return MVR_ERR_DTYPE;
  if (any_rows && (!a->q || (a->has_index && !a->index))) return MVR_ERR_NULL;
  if (any_states && (!a->k || !a->v)) return MVR_ERR_NULL;
  if (any_rows && (!a->out || (backward && (!a->grad_out || !a->grad_q || !a->lse)))) return MVR_ERR_NULL;
  if (any_states && backward && (!a->grad_k || !a->grad_v)) return MVR_ERR_NULL;
  return MVR_OK;
}

AttnParams attention_params(const mvr_attention* a, const AttnCut& c, char* ws) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.g = a->grad_out; p.out = a->out; p.o = a->out;
  p.gq = a->grad_q; p.gk = a->grad_k; p.gv = a->grad_v; p.lse = a->lse;
  p.q_r = a->q_strides[0]; p.q_t = a->q_strides[1]; p.q_h = a->q_strides[2];
  p.k_n = a->k_strides[0]; p.k_l = a->k_strides[1]; p.k_h = a->k_strides[2];
  p.v_n = a->v_strides[0]; p.v_l = a->v_strides[1]; p.v_h = a->v_strides[2];
  p.g_r = a->g_strides[0]; p.g_t = a->g_strides[1]; p.g_h = a->g_strides[2];
  if (c.direct) {
    p.index = a->index; p.index_type = a->index_type; p.index_stride = a->index_stride;
  } else if (a->has_index) {
    p.order = (const int*)(ws + c.order); p.starts = (const int*)(ws + c.starts); p.tiles = (const int*)(ws + c.tiles);
  }
  p.lengths = a->lengths; p.lengths64 = a->lengths_64; p.mask = a->mask;
  p.R = (int)a->R; p.T = (int)a->T; p.Hq = (int)a->Hq; p.Hk = (int)a->Hk; p.G = (int)(a->Hq / a->Hk);
  p.N = (int)a->N; p.L = (int)a->L; p.D = (int)a->D;
  p.W = c.W;
  p.by_T.set((unsigned)std::max(1, p.T));
  p.by_G.set((unsigned)p.G);
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.splits = c.splits; p.row_splits = c.row_splits;
  p.delta = (float*)(ws + c.delta); p.norm = (float*)(ws + c.norm); p.peaks = (int*)(ws + c.peaks); p.row_peaks = (float2*)(ws + c.row_peaks);
  p.part_o = (float*)(ws + c.part_o); p.part_ml = (float*)(ws + c.part_ml);
  p.part_gq = (float*)(ws + c.part_gq); p.part_gk = (float*)(ws + c.part_gk); p.part_gv = (float*)(ws + c.part_gv);
  return p;
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

int plan_attention(const mvr_attention* a, const AttnCut& c, char* ws, int* status, cudaStream_t st) {
  if (!a->has_index || c.direct) return MVR_OK;
  const int groups = (int)a->N + 1;
  const int warps = (int)std::max<long long>(1, std::min<long long>({32, cdiv(a->R, 32), (long long)(kPlanShared / 4 / groups)}));
  const size_t smem = (size_t)warps * groups * 4;
  if (!shared_memory<attn_plan>(kPlanShared)) return MVR_ERR_LAUNCH;
  launch_dependent(attn_plan, dim3(1), dim3(kPlanThreads), smem, st, a->index, a->index_type, (long long)a->index_stride, (int)a->R,
                   (int)a->N, (int)(a->T * (a->Hq / a->Hk)), c.tile, warps, (int*)(ws + c.order), (int*)(ws + c.starts),
                   (int*)(ws + c.tiles), status);
  return launched();
}

template <typename T, int DP>
int fma_forward(const AttnParams& p, const AttnCut& c, cudaStream_t st) {
  return launch_shared<attn_fma_fwd<T, DP>>(dim3((unsigned)c.row_tiles, p.Hk, c.splits), kFmaThreads, FmaTile<DP>::bytes(3), st, p);
}
template <typename T, int DP>
int fma_backward(const AttnParams& p, const AttnCut& c, cudaStream_t st) {
  if (p.R > 0 && p.T > 0) {
    const int rc = launch_shared<attn_fma_dq<T, DP>>(dim3((unsigned)c.row_tiles, p.Hk, c.splits), kFmaThreads, FmaTile<DP>::bytes(4), st, p);
    if (rc != MVR_OK) return rc;
  }
  return launch_shared<attn_fma_dkv<T, DP>>(dim3((unsigned)(cdiv(p.L, c.kv_tile) * p.N), p.Hk, c.row_splits), kFmaThreads, FmaTile<DP>::bytes(4), st, p);
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

template <typename T, int DP, int TILES, bool MASK, int PIECES>
int tc_forward_as(const AttnParams& p, const AttnCut& c, const TcMaps& maps, int* status, cudaStream_t st) {
  typedef TcForward<DP, TILES, MASK, PIECES> F;
  return launch_shared<attn_tc_fwd<T, DP, TILES, MASK, PIECES>>(dim3((unsigned)c.row_tiles, p.Hk, c.splits), F::kThreads, F::kShared, st, p, maps, status);
}
template <typename T, int DP, int PIECES>
int tc_forward(const AttnParams& p, const AttnCut& c, const TcMaps& maps, int* status, cudaStream_t st) {
  const bool mask = p.mask || p.lengths;
  if constexpr (DP == 128) {
    if (c.tile > kTcRows)
      return mask ? tc_forward_as<T, DP, 2, true, 1>(p, c, maps, status, st) : tc_forward_as<T, DP, 2, false, 1>(p, c, maps, status, st);
  }
  return mask ? tc_forward_as<T, DP, 1, true, PIECES>(p, c, maps, status, st) : tc_forward_as<T, DP, 1, false, PIECES>(p, c, maps, status, st);
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

template <typename T>
int attention_forward(const AttnParams& p, const AttnCut& c, const TcMaps& maps, int* status, cudaStream_t st) {
  int rc;
  if (c.tc) {
    if constexpr (sizeof(T) == 2) rc = p.D <= 64 ? tc_forward<T, 64, 1>(p, c, maps, status, st) : tc_forward<T, 128, 1>(p, c, maps, status, st);
    else rc = tc_forward<__nv_bfloat16, 64, 3>(p, c, maps, status, st);
  } else {
    rc = p.D <= 32 ? fma_forward<T, 32>(p, c, st) : p.D <= 64 ? fma_forward<T, 64>(p, c, st)
         : p.D <= 128 ? fma_forward<T, 128>(p, c, st) : fma_forward<T, 256>(p, c, st);
  }
  if (rc != MVR_OK || c.splits == 1) return rc;
  const long long outputs = (long long)p.R * p.T * p.Hq * p.D;
  if (p.D % 4 == 0 && (uintptr_t)p.out % (4 * sizeof(T)) == 0)
    launch_dependent(attn_join<T, 4>, dim3((unsigned)cdiv(outputs, 1024)), dim3(256), 0, st, p);
  else
    launch_dependent(attn_join<T, 1>, dim3((unsigned)cdiv(outputs, 256)), dim3(256), 0, st, p);
  return launched();
}

template <typename T, int DP, int PIECES>
int tc_backward(const AttnParams& p, const AttnCut& c, const TcMaps& maps, bool boxes, int* status, cudaStream_t st) {
  const dim3 states((unsigned)(cdiv(p.L, 128) * p.N), p.Hk, c.row_splits);
  typedef TcStates<DP, PIECES> S;
  const int rc = boxes ? launch_shared<attn_tc_dkv<T, DP, true, PIECES>>(states, S::kThreads, S::kShared, st, p, maps, status)
                       : launch_shared<attn_tc_dkv<T, DP, false, PIECES>>(states, S::kThreads, S::kShared, st, p, maps, status);
  if (rc != MVR_OK || p.R == 0 || p.T == 0) return rc;
  const dim3 grid((unsigned)c.row_tiles, p.Hk, c.splits);
  if (p.mask || p.lengths) {
    typedef TcRows<DP, true, PIECES> F;
    return launch_shared<attn_tc_dq<T, DP, true, PIECES>>(grid, F::kThreads, F::kShared, st, p, maps, status);
  }
  typedef TcRows<DP, false, PIECES> F;
  return launch_shared<attn_tc_dq<T, DP, false, PIECES>>(grid, F::kThreads, F::kShared, st, p, maps, status);
}

// plain: the call's own tensors, where the operands are in pieces.
template <typename T>
int attention_backward(const AttnParams& p, const AttnParams& plain, const AttnCut& c, const TcMaps& maps, bool boxes, int* status, cudaStream_t st) {
  const long long rows = (long long)p.R * p.T * p.Hq, states = (long long)p.N * p.L * p.Hk * p.D;
  int rc = MVR_OK;
  if (c.tc && std::is_same<T, __half>::value && cudaMemsetAsync(p.peaks, 0, (size_t)p.N * p.Hk * 4, st) != cudaSuccess) {
    cudaGetLastError();
    return MVR_ERR_LAUNCH;
  }
  if (rows > 0) {
    bool done = false;
    if constexpr (sizeof(T) == 2) {
      done = c.tc;
      if (c.tc) launch_dependent(attn_tc_delta<T>, dim3((unsigned)c.row_tiles, p.Hk), dim3(kDeltaThreads), 0, st, p);
    }
    if (!done) launch_dependent(attn_delta<T>, dim3((unsigned)cdiv(rows, 8)), dim3(256), 0, st, plain);
    if ((rc = launched()) != MVR_OK) return rc;
  }
  if (c.tc) {
    if constexpr (sizeof(T) == 2)
      rc = p.D <= 64 ? tc_backward<T, 64, 1>(p, c, maps, boxes, status, st) : tc_backward<T, 128, 1>(p, c, maps, boxes, status, st);
    else
      rc = tc_backward<__nv_bfloat16, 64, 3>(p, c, maps, boxes, status, st);
  }
  if (!c.tc)
    rc = p.D <= 32 ? fma_backward<T, 32>(p, c, st) : p.D <= 64 ? fma_backward<T, 64>(p, c, st)
         : p.D <= 128 ? fma_backward<T, 128>(p, c, st) : fma_backward<T, 256>(p, c, st);
  if (rc == MVR_OK && c.splits > 1) rc = sum_parts<T>(p.part_gq, p.gq, rows * p.D, c.splits, p.scale, st);
  if (rc == MVR_OK && c.row_splits > 1) rc = sum_parts<T>(p.part_gk, p.gk, states, c.row_splits, p.scale, st);
  if (rc == MVR_OK && c.row_splits > 1) rc = sum_parts<T>(p.part_gv, p.gv, states, c.row_splits, 1.0f, st);
  return rc;
}

// Float operands of a call in pieces, in its workspace; `b` is the call on them.
int split_operands(const mvr_attention* a, bool backward, const AttnCut& c, char* ws, mvr_attention& b, AttnParams& p, cudaStream_t st) {
  const auto split = [&](const void* from, const int64_t (&s)[3], long long n0, long long n1, long long n2, long long to) {
    const long long rows = n0 * n1 * n2;
    if (rows > 0)
      launch_dependent(split_floats, dim3((unsigned)cdiv(rows * (c.W / 8), 256)), dim3(256), 0, st, (const float*)from, (long long)s[0], (long long)s[1],
                       (long long)s[2], (int)n1, (int)n2, rows, (int)a->D, c.W, (__nv_bfloat16*)(ws + to));
    return launched();
  };
  int rc = split(a->q, a->q_strides, a->R, a->T, a->Hq, c.q);
  if (rc == MVR_OK) rc = split(a->k, a->k_strides, a->N, a->L, a->Hk, c.k);
  if (rc == MVR_OK) rc = split(a->v, a->v_strides, a->N, a->L, a->Hk, c.v);
  if (rc == MVR_OK && backward) rc = split(a->grad_out, a->g_strides, a->R, a->T, a->Hq, c.g);
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

template <typename T>
int attention_as(const mvr_attention* a, bool backward, char* workspace, int* status, cudaStream_t st) {
  TcMaps maps = {};
  bool boxes = false;
  bool tc = tc_sizes(a);
  if constexpr (sizeof(T) == 2) {
    tc = tc && (uintptr_t)a->out % 16 == 0 && rows_aligned(a->q, a->q_strides, a);
    if (backward)
      tc = tc && rows_aligned(a->grad_out, a->g_strides, a) && (((uintptr_t)a->grad_q | (uintptr_t)a->grad_k | (uintptr_t)a->grad_v) & 15) == 0;
    tc = tc && tensor_maps<T>(a, backward, 1, maps, boxes);
  }
  const AttnCut c = cut_attention(a, backward, tc);
  if (c.row_tiles > INT32_MAX) return MVR_ERR_TOO_LARGE;
  int rc = plan_attention(a, c, workspace, status, st);
  if (rc != MVR_OK) return rc;
  AttnParams p = attention_params(a, c, workspace);
  if constexpr (sizeof(T) == 4) {
    if (tc) {
      const AttnParams plain = p;
      mvr_attention b;
      if ((rc = split_operands(a, backward, c, workspace, b, p, st)) != MVR_OK) return rc;
      if (!tensor_maps<__nv_bfloat16>(&b, backward, 3, maps, boxes)) return MVR_ERR_LAUNCH;
      return backward ? attention_backward<T>(p, plain, c, maps, boxes, status, st)
                      : attention_forward<T>(p, c, maps, status, st);
    }
  }
  return backward ? attention_backward<T>(p, p, c, maps, boxes, status, st)
                  : attention_forward<T>(p, c, maps, status, st);
}

long long attention_bytes(const mvr_attention* a, bool backward) {
  const long long fma = cut_attention(a, backward, false).bytes;
  return tc_sizes(a) ? std::max(fma, cut_attention(a, backward, true).bytes) : fma;
}

int attention(const mvr_attention* a, bool backward, void* workspace, int64_t bytes, int* status, void* stream) {
  const int rc = check_attention(a, backward, false);
  if (rc != MVR_OK) return rc;
  const long long need = attention_bytes(a, backward);
  if (bytes < need || (need > 0 && !workspace)) return MVR_ERR_WORKSPACE;
  const bool any_rows = a->R > 0 && a->T > 0, any_states = a->N > 0 && a->L > 0;
  if (!any_rows && (!backward || !any_states)) return MVR_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case MVR_F32: return attention_as<float>(a, backward, (char*)workspace, status, st);
    case MVR_F16: return attention_as<__half>(a, backward, (char*)workspace, status, st);
    default: return attention_as<__nv_bfloat16>(a, backward, (char*)workspace, status, st);
  }
}

}  // namespace

extern "C" {

int mvr_attention_workspace(const mvr_attention* a, int backward, int64_t* bytes) {
  if (!bytes) return MVR_ERR_NULL;
  const int rc = check_attention(a, backward != 0, true);
  if (rc != MVR_OK) return rc;
  *bytes = attention_bytes(a, backward != 0);
  return MVR_OK;
}

int mvr_attention_forward(const mvr_attention* a, void* workspace, int64_t bytes, int* status, void* stream) {
  return attention(a, false, workspace, bytes, status, stream);
}

int mvr_attention_backward(const mvr_attention* a, void* workspace, int64_t bytes, int* status, void* stream) {
  return attention(a, true, workspace, bytes, status, stream);
}

int mvr_dropout(const void* x, const void* residual, void* out, int dtype, int64_t n, double probability, uint64_t seed,
                const uint64_t* seed_at, uint64_t offset, void* stream) {
  if (!head_dtype(dtype)) return MVR_ERR_DTYPE;
  if (n < 0) return MVR_ERR_SHAPE;
  if (!(probability >= 0.0 && probability <= 1.0)) return MVR_ERR_PROBABILITY;
  if (n == 0) return MVR_OK;
  if (!x || !out) return MVR_ERR_NULL;
  DropoutParams p = {};
  p.x = x; p.residual = residual; p.out = out; p.n = n;
  const int cut = (int)std::floor(probability * 65536.0 + 0.5);  // an element stays when its 16 bits are >= cut
  const cudaStream_t st = (cudaStream_t)stream;
  if (cut == 65536) {  // none does
    if (residual == out) return MVR_OK;
    const size_t bytes = (size_t)n * (dtype == MVR_F32 ? 4 : 2);
    const cudaError_t e = residual ? cudaMemcpyAsync(out, residual, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(out, 0, bytes, st);
    if (e != cudaSuccess) cudaGetLastError();
    return e == cudaSuccess ? MVR_OK : MVR_ERR_LAUNCH;
  }
  p.floor = (unsigned)cut << 16;
  p.scale = (float)(65536.0 / (65536.0 - cut));
  p.keys.from(seed);
  p.seed_at = (const unsigned long long*)seed_at;
  p.offset = offset;
  const int rc = dtype == MVR_F32 ? launch_dropout<float>(p, st) : dtype == MVR_F16 ? launch_dropout<__half>(p, st)
                                                                                    : launch_dropout<__nv_bfloat16>(p, st);
  return rc ? MVR_ERR_TOO_LARGE : launched();
}

static int label_log_probs(const LogProbParams& p, int dtype, bool fwd, void* stream) {
  const cudaStream_t st = (cudaStream_t)stream;
  const int rc = dtype == MVR_F32 ? launch_logprob<float>(p, fwd, st) : dtype == MVR_F16 ? launch_logprob<__half>(p, fwd, st)
                                                                                         : launch_logprob<__nv_bfloat16>(p, fwd, st);
  return rc ? MVR_ERR_TOO_LARGE : launched();
}

static int check_label_log_probs(int dtype, int label_dtype, int64_t batch, int64_t classes, int64_t space) {
  if (!head_dtype(dtype)) return MVR_ERR_DTYPE;
  if (label_dtype < MVR_LABEL_U8 || label_dtype > MVR_LABEL_I64) return MVR_ERR_DTYPE;
  if (batch < 0 || classes < 1 || space < 0) return MVR_ERR_SHAPE;
  if (classes > INT32_MAX - 64) return MVR_ERR_TOO_LARGE;
  if (space > 0 && batch > INT64_MAX / 32 / space) return MVR_ERR_TOO_LARGE;
  return MVR_OK;
}

// rest: the entries that keep what the rounding of lse left; both are wanted then.
static int label_log_probs_forward(const void* logits, int dtype, const void* labels, int label_dtype, float* log_prob, float* entropy,
                                   float* lse, bool rest, float* lse_rest, float* top_log_prob, int32_t* top_label, int64_t batch,
                                   int64_t classes, int64_t space, int64_t batch_stride, int64_t class_stride, int top, void* stream) {
  const int rc = check_label_log_probs(dtype, label_dtype, batch, classes, space);
  if (rc != MVR_OK) return rc;
  if (top < 0 || top > MVR_MAX_TOP || top > classes) return MVR_ERR_TOP;
  if (batch == 0 || space == 0) return MVR_OK;
  if (!logits || !labels || !log_prob || !entropy || (top > 0 && (!top_log_prob || !top_label))) return MVR_ERR_NULL;
  if (rest && (!lse || !lse_rest)) return MVR_ERR_NULL;
  LogProbParams p = {};
  p.x = logits; p.labels = labels; p.label_type = label_dtype;
  p.log_prob = log_prob; p.entropy = entropy; p.lse = lse; p.lse_rest = lse_rest; p.top_value = top_log_prob; p.top_label = top_label;
  p.batch = batch; p.space = space; p.batch_stride = batch_stride; p.class_stride = class_stride;
  p.classes = (int)classes; p.top = top;
  return label_log_probs(p, dtype, true, stream);
}

static int label_log_probs_backward(const void* logits, int dtype, const void* labels, int label_dtype, const float* lse, bool rest,
                                    const float* lse_rest, const float* entropy, const float* grad_log_prob, const float* grad_entropy,
                                    void* grad_logits, int64_t batch, int64_t classes, int64_t space, int64_t batch_stride,
                                    int64_t class_stride, int64_t grad_batch_stride, int64_t grad_class_stride, void* stream) {
  const int rc = check_label_log_probs(dtype, label_dtype, batch, classes, space);
  if (rc != MVR_OK) return rc;
  if (batch == 0 || space == 0) return MVR_OK;
  if (!logits || !labels || !lse || (rest && !lse_rest) || !entropy || !grad_logits) return MVR_ERR_NULL;
  LogProbParams p = {};
  p.x = logits; p.labels = labels; p.label_type = label_dtype;
  p.entropy = const_cast<float*>(entropy); p.lse = const_cast<float*>(lse); p.lse_rest = const_cast<float*>(lse_rest);
  p.grad_log_prob = grad_log_prob; p.grad_entropy = grad_entropy; p.grad = grad_logits;
  p.batch = batch; p.space = space; p.batch_stride = batch_stride; p.class_stride = class_stride;
  p.grad_batch_stride = grad_batch_stride; p.grad_class_stride = grad_class_stride;
  p.classes = (int)classes;
  return label_log_probs(p, dtype, false, stream);
}

int mvr_label_log_probs_forward(const void* logits, int dtype, const void* labels, int label_dtype, float* log_prob, float* entropy,
                                float* lse, float* top_log_prob, int32_t* top_label, int64_t batch, int64_t classes, int64_t space,
                                int64_t batch_stride, int64_t class_stride, int top, void* stream) {
  return label_log_probs_forward(logits, dtype, labels, label_dtype, log_prob, entropy, lse, false, nullptr, top_log_prob, top_label, batch,
                                 classes, space, batch_stride, class_stride, top, stream);
}

int mvr_label_log_probs_forward_rest(const void* logits, int dtype, const void* labels, int label_dtype, float* log_prob,
                                     float* entropy, float* lse, float* lse_rest, float* top_log_prob, int32_t* top_label, int64_t batch,
                                     int64_t classes, int64_t space, int64_t batch_stride, int64_t class_stride, int top,
                                     void* stream) {
  return label_log_probs_forward(logits, dtype, labels, label_dtype, log_prob, entropy, lse, true, lse_rest, top_log_prob, top_label, batch,
                                 classes, space, batch_stride, class_stride, top, stream);
}

int mvr_label_log_probs_backward(const void* logits, int dtype, const void* labels, int label_dtype, const float* lse,
                                 const float* entropy, const float* grad_log_prob, const float* grad_entropy, void* grad_logits,
                                 int64_t batch, int64_t classes, int64_t space, int64_t batch_stride, int64_t class_stride,
                                 int64_t grad_batch_stride, int64_t grad_class_stride, void* stream) {
  return label_log_probs_backward(logits, dtype, labels, label_dtype, lse, false, nullptr, entropy, grad_log_prob, grad_entropy, grad_logits,
                                  batch, classes, space, batch_stride, class_stride, grad_batch_stride, grad_class_stride, stream);
}

int mvr_label_log_probs_backward_rest(const void* logits, int dtype, const void* labels, int label_dtype, const float* lse,
                                      const float* lse_rest, const float* entropy, const float* grad_log_prob,
                                      const float* grad_entropy, void* grad_logits, int64_t batch, int64_t classes, int64_t space,
                                      int64_t batch_stride, int64_t class_stride, int64_t grad_batch_stride,
                                      int64_t grad_class_stride, void* stream) {
  return label_log_probs_backward(logits, dtype, labels, label_dtype, lse, true, lse_rest, entropy, grad_log_prob, grad_entropy, grad_logits,
                                  batch, classes, space, batch_stride, class_stride, grad_batch_stride, grad_class_stride, stream);
}

}  // extern "C"
