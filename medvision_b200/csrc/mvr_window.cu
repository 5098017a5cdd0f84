// C ABI of attention in a sliding window (declared in include/mvr.h): argument checks, how a call is cut into CTAs, launches.  The kernels
// are those of mvr_attn_fma.cuh, mvr_attn_tc.cuh and mvr_attn_tc_bwd.cuh, each walking the tiles that its rows' windows reach, and for the
// forward of a few rows that of mvr_attn_rows.cuh.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/mvr.h"
#include "mvr_attn_host.cuh"
#include "mvr_attn_rows.cuh"

namespace {

enum Way { kFloats = 0, kTensorCores = 1, kFewRows = 2 };

struct WindowCut : OperandPieces {
  bool tc, rounded;               // rounded: half types' weights, once
  int tile;                       // rows of a CTA's tile
  long long row_tiles;            // of all sequences, per key head
  int splits, tiles_per;          // parts of the states that a row tile walks (forward, dq), and the kernel's tiles of one
  int row_splits, row_tiles_per;  // of the rows that a state tile meets (dk, dv)
  int state_tile, sink_tiles, sink_parts;
  long long delta, norm, peaks, row_peaks, part_o, part_ml, part_gq, part_gk, part_gv, bytes;
};

// Its sizes.
WindowSizes sizes_of(const mvr_attention* a, const mvr_window* w) { return window_sizes(a->T, a->L, a->Hq / a->Hk, w->before, w->after, w->sinks); }

WindowCut cut_window(const mvr_attention* a, const mvr_window* given, bool backward, Way way) {
  const WindowSizes w = sizes_of(a, given);
  WindowCut c = {};
  const bool tc = c.tc = way == kTensorCores;
  c.rounded = given->rounded_weights != 0;
  const bool pieces = tc && a->dtype == MVR_F32, wide = a->D > 64;
  c.W = (int)(pieces ? cdiv(a->D, 8) * 8 : a->D);
  const long long G = a->Hq / a->Hk, per = a->T * G, rows = a->R * a->T * a->Hq;
  c.tile = tc ? (per > kTcRows && !backward && wide ? 2 * kTcRows : kTcRows) : a->D <= 128 ? 64 : 32;
  c.row_tiles = a->R * cdiv(per, c.tile);
  c.state_tile = tc ? 128 : c.tile;
  // the kernels' own steps through the states (the forward, dq) and the rows (dk, dv)
  const int step = !tc ? c.tile : backward ? (wide ? kGradStep<128> : kGradStep<64>) : c.tile > kTcRows ? 128 : 64;
  // (a part's sums are written and read at 4 MB/us)
  c.splits = best_parts(std::max<long long>(1, c.row_tiles * a->Hk), w.span_tiles(c.tile, c.state_tile), states_step(tc, pieces, backward, wide, c.tile > kTcRows),
                        rows * a->D * 8 / 4e6, false);
  c.tiles_per = (int)cdiv(w.span_tiles(c.tile, step), c.splits);
  if (way == kFewRows) {
    // 592 CTAs, four an SM (eight: up to 15 % slower), with 128 states each at least (64: 9.4 us instead of 6.8 for 8 caches' windows of 500).
    // Their rings let an SM hold three at a time in half types and one in float, so that they run in two waves and in four.
    const long long states = w.reach(a->T) + w.sinks, ctas = std::max<long long>(1, a->N * a->Hk);
    c.splits = (int)std::max<long long>(1, std::min<long long>({64, cdiv(4 * kMultiprocessors, ctas), cdiv(states, 128)}));
  }
  c.sink_tiles = (int)cdiv(w.sinks, c.state_tile);
  c.row_splits = c.sink_parts = 1;
  const long long others = cdiv(a->L, c.state_tile) - c.sink_tiles, lead = std::min<long long>(a->L, (long long)c.sink_tiles * c.state_tile);
  if (backward) {
    // rows of a tile that the first states do not belong to; the first ones, which meet all rows, are cut into parts as long
    c.row_splits = best_parts(std::max<long long>(1, a->N * a->Hk * others), std::max<long long>(1, cdiv(w.rows_reached(c.state_tile), c.tile)), rows_step(tc, pieces, wide),
                              (double)a->N * (a->L - lead) * a->Hk * a->D * 16 / 4e6, false);
    c.row_tiles_per = w.row_tiles(c.state_tile, step, c.row_splits);
    if (c.sink_tiles > 0) c.sink_parts = w.sink_parts(step, c.row_tiles_per);
  }
  long long at = 0;
  const auto take = [&at](long long bytes) {
    const long long here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
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
      c.peaks = take(a->N * cdiv(a->L, 128) * a->Hk * 4);
      c.row_peaks = take(c.row_tiles * a->Hk * 8);
    }
    if (c.splits > 1) c.part_gq = take(c.splits * rows * a->D * 4);
    const long long states = (c.sink_parts > 1 ? c.sink_parts * lead : 0) + (c.row_splits > 1 ? c.row_splits * (a->L - lead) : 0);
    if (states > 0) {
      c.part_gk = take(a->N * states * a->Hk * a->D * 4);
      c.part_gv = take(a->N * states * a->Hk * a->D * 4);
    }
  } else if (c.splits > 1) {
    c.part_o = take(c.splits * rows * a->D * 4);
    c.part_ml = take(c.splits * rows * 8);
  }
  c.bytes = at;
  return c;
}

// Whether a forward is of few rows: those of a key head are the lanes' registers, and rows are read in vectors.  Half types up to two rows (32
// caches, windows of 2051 states, 8 key heads of 128: one row 55 us, two 57, four 73; tensor cores 70), float up to eight (16 caches of
// 2000 states, 8 heads of 64: 57 us, in float arithmetic by tiles 209).
bool few_rows(const mvr_attention* a) {
  return a->T * (a->Hq / a->Hk) <= (a->dtype == MVR_F32 ? 8 : 2) && a->D % 8 == 0 && a->N <= INT32_MAX / 64 && a->Hk <= 65535;
}
bool vectors_aligned(const void* base, const int64_t (&strides)[3], const int64_t (&sizes)[3], int element) {
  if ((uintptr_t)base % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && strides[i] * element % 16 != 0) return false;
  return true;
}

// Whether type and sizes are the tensor cores'.  Float operands are cut into pieces whole, states that no token reads among them:
// only where the tokens are not few beside the states.
bool tc_window(const mvr_attention* a, const mvr_window* w) {
  const double rows = (double)a->R * a->T * a->Hq;
  if (a->L == 0 || a->N == 0 || a->N > INT32_MAX / 4 || rows > 2e9) return false;
  const WindowSizes s = sizes_of(a, w);
  // (a few tiles of rows against one of states are as fast in float arithmetic, which rounds nothing on its way)
  if (a->T * (a->Hq / a->Hk) <= 256 && std::min<long long>(a->L, s.reach(a->T) + s.sinks) <= 64) return false;
  if (a->dtype != MVR_F32) return a->D % 8 == 0 && a->D <= 128;
  return a->D <= 64 && a->T >= a->L / 4 && rows * std::min<long long>(a->L, s.reach(1) + s.sinks) >= kPieceScores;
}

int check_window(const mvr_attention* a, const mvr_window* w, bool backward, bool sizes_only) {
  if (!a || !w) return MVR_ERR_NULL;
  if (!head_dtype(a->dtype)) return MVR_ERR_DTYPE;
  if (a->R < 0 || a->T < 0 || a->Hq < 1 || a->Hk < 1 || a->N < 0 || a->L < 0 || a->D < 1 || a->R != a->N) return MVR_ERR_SHAPE;
  if (w->before < 0 || w->after < 0 || w->sinks < 0) return MVR_ERR_WINDOW;
  if (a->Hq % a->Hk != 0) return MVR_ERR_HEADS;
  if (a->D > 256) return MVR_ERR_HEAD_SIZE;
  if (a->has_index || a->mask) return MVR_ERR_UNSUPPORTED;
  const long long most = INT32_MAX / 4;
  if (a->R > most || a->T > most || a->Hq > 65535 || a->Hk > 65535 || a->L > most) return MVR_ERR_TOO_LARGE;
  if (a->T > 0 && a->R > 0 && a->R * a->T > most / (a->Hq / a->Hk)) return MVR_ERR_TOO_LARGE;  // rows of a key head: 32 bits
  if (a->R * a->T * a->Hq * a->D / 256 > INT32_MAX - 1) return MVR_ERR_TOO_LARGE;              // CTAs of the small kernels
  if (cdiv(a->L, 32) * a->N > INT32_MAX / 64) return MVR_ERR_TOO_LARGE;                        // CTAs of dk, dv
  if (sizes_only) return MVR_OK;
  const bool any_rows = a->R > 0 && a->T > 0, any_states = a->N > 0 && a->L > 0;
  if (any_rows && !a->q) return MVR_ERR_NULL;
  if (any_states && (!a->k || !a->v)) return MVR_ERR_NULL;
  if (any_rows && (!a->out || (backward && (!a->grad_out || !a->grad_q || !a->lse)))) return MVR_ERR_NULL;
  if (any_states && backward && (!a->grad_k || !a->grad_v)) return MVR_ERR_NULL;
  return MVR_OK;
}

AttnParams window_params(const mvr_attention* a, const mvr_window* given, const WindowCut& c, char* ws) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.g = a->grad_out; p.out = a->out; p.o = a->out;
  p.gq = a->grad_q; p.gk = a->grad_k; p.gv = a->grad_v; p.lse = a->lse;
  p.q_r = a->q_strides[0]; p.q_t = a->q_strides[1]; p.q_h = a->q_strides[2];
  p.k_n = a->k_strides[0]; p.k_l = a->k_strides[1]; p.k_h = a->k_strides[2];
  p.v_n = a->v_strides[0]; p.v_l = a->v_strides[1]; p.v_h = a->v_strides[2];
  p.g_r = a->g_strides[0]; p.g_t = a->g_strides[1]; p.g_h = a->g_strides[2];
  p.lengths = a->lengths; p.lengths64 = a->lengths_64;
  p.R = (int)a->R; p.T = (int)a->T; p.Hq = (int)a->Hq; p.Hk = (int)a->Hk; p.G = (int)(a->Hq / a->Hk);
  p.N = (int)a->N; p.L = (int)a->L; p.D = (int)a->D;
  p.W = c.W;
  p.by_T.set((unsigned)std::max(1, p.T));
  p.by_G.set((unsigned)p.G);
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.before = given->before; p.after = given->after; p.sinks = (int)std::min<long long>(given->sinks, a->L);
  p.offsets = given->offsets; p.offsets64 = given->offsets_64;
  if (a->dtype != MVR_F32) p.rest = (__nv_bfloat16*)given->rest;
  p.offset = given->offset;
  p.splits = c.splits; p.tiles_per = c.tiles_per;
  p.row_splits = c.row_splits; p.row_tiles_per = c.row_tiles_per; p.sink_tiles = c.sink_tiles; p.sink_parts = c.sink_parts;
  p.delta = (float*)(ws + c.delta); p.norm = (float*)(ws + c.norm); p.peaks = (int*)(ws + c.peaks); p.row_peaks = (float2*)(ws + c.row_peaks);
  p.part_o = (float*)(ws + c.part_o); p.part_ml = (float*)(ws + c.part_ml);
  p.part_gq = (float*)(ws + c.part_gq); p.part_gk = (float*)(ws + c.part_gk); p.part_gv = (float*)(ws + c.part_gv);
  return p;
}

// CTAs of dk, dv over an image's tiles and parts.
unsigned state_ctas(const AttnParams& p, const WindowCut& c) {
  return (unsigned)((long long)p.N * ((long long)c.sink_tiles * c.sink_parts + (cdiv(p.L, c.state_tile) - c.sink_tiles) * c.row_splits));
}

template <typename T, int DP>
int fma_window(const AttnParams& p, const WindowCut& c, bool backward, cudaStream_t st) {
  const dim3 rows((unsigned)c.row_tiles, p.Hk, c.splits);
  if (!backward) return launch_shared<attn_fma_fwd<T, DP, true>>(rows, kFmaThreads, FmaTile<DP>::bytes(3), st, p);
  if (p.R > 0 && p.T > 0) {
    const int rc = launch_shared<attn_fma_dq<T, DP, true>>(rows, kFmaThreads, FmaTile<DP>::bytes(4), st, p);
    if (rc != MVR_OK) return rc;
  }
  return launch_shared<attn_fma_dkv<T, DP, true>>(dim3(state_ctas(p, c), p.Hk), kFmaThreads, FmaTile<DP>::bytes(4), st, p);
}
template <typename T>
int fma_window(const AttnParams& p, const WindowCut& c, bool backward, cudaStream_t st) {
  return p.D <= 32 ? fma_window<T, 32>(p, c, backward, st) : p.D <= 64 ? fma_window<T, 64>(p, c, backward, st)
         : p.D <= 128 ? fma_window<T, 128>(p, c, backward, st) : fma_window<T, 256>(p, c, backward, st);
}

template <typename T, int DP>
int rows_forward(const AttnParams& p, const WindowCut& c, cudaStream_t st) {
  const dim3 grid(p.N, p.Hk, c.splits);
  const int rows = p.T * p.G;
  constexpr size_t shared = kRowsShared<T>;
  if (rows <= 1) return launch_shared<attn_rows_fwd<T, DP, 1>>(grid, kRowsThreads, shared, st, p);
  if constexpr (sizeof(T) == 4) {
    if (rows > 4) return launch_shared<attn_rows_fwd<T, DP, 8>>(grid, kRowsThreads, shared, st, p);
    if (rows > 2) return launch_shared<attn_rows_fwd<T, DP, 4>>(grid, kRowsThreads, shared, st, p);
  }
  return launch_shared<attn_rows_fwd<T, DP, 2>>(grid, kRowsThreads, shared, st, p);
}
template <typename T>
int rows_forward(const AttnParams& p, const WindowCut& c, cudaStream_t st) {
  return p.D <= 32 ? rows_forward<T, 32>(p, c, st) : p.D <= 64 ? rows_forward<T, 64>(p, c, st) : p.D <= 128 ? rows_forward<T, 128>(p, c, st)
                                                                                                  : rows_forward<T, 256>(p, c, st);
}

// MODE: kWindow, or kWindowRounded where the caller wants half types' weights rounded once.
template <typename T, int DP, int TILES, int PIECES, int MODE>
int tc_window_forward_as(const AttnParams& p, const WindowCut& c, const TcMaps& maps, int* status, cudaStream_t st) {
  typedef TcForward<DP, TILES, MODE, PIECES> F;
  return launch_shared<attn_tc_fwd<T, DP, TILES, MODE, PIECES>>(dim3((unsigned)c.row_tiles, p.Hk, c.splits), F::kThreads, F::kShared, st, p, maps, status);
}
template <typename T, int DP, int TILES, int PIECES>
int tc_window_forward(const AttnParams& p, const WindowCut& c, const TcMaps& maps, int* status, cudaStream_t st) {
  if constexpr (PIECES == 1)
    if (c.rounded) return tc_window_forward_as<T, DP, TILES, PIECES, kWindowRounded>(p, c, maps, status, st);
  return tc_window_forward_as<T, DP, TILES, PIECES, kWindow>(p, c, maps, status, st);
}
template <typename T, int DP, int PIECES, int MODE>
int tc_window_states(const AttnParams& p, const WindowCut& c, const TcMaps& maps, bool boxes, int* status, cudaStream_t st) {
  typedef TcStates<DP, PIECES> S;
  const dim3 states(state_ctas(p, c), p.Hk);
  return boxes ? launch_shared<attn_tc_dkv<T, DP, true, PIECES, MODE>>(states, S::kThreads, S::kShared, st, p, maps, status)
               : launch_shared<attn_tc_dkv<T, DP, false, PIECES, MODE>>(states, S::kThreads, S::kShared, st, p, maps, status);
}
template <typename T, int DP, int PIECES>
int tc_window_backward(const AttnParams& p, const WindowCut& c, const TcMaps& maps, bool boxes, int* status, cudaStream_t st) {
  const int rc = PIECES == 1 && c.rounded ? tc_window_states<T, DP, PIECES, PIECES == 1 ? kWindowRounded : kWindow>(p, c, maps, boxes, status, st)
                                          : tc_window_states<T, DP, PIECES, kWindow>(p, c, maps, boxes, status, st);
  if (rc != MVR_OK || p.R == 0 || p.T == 0) return rc;
  typedef TcRows<DP, kWindow, PIECES> F;
  return launch_shared<attn_tc_dq<T, DP, kWindow, PIECES>>(dim3((unsigned)c.row_tiles, p.Hk, c.splits), F::kThreads, F::kShared, st, p, maps, status);
}

template <typename T>
int window_forward(const AttnParams& p, const WindowCut& c, Way way, const TcMaps& maps, int* status, cudaStream_t st) {
  int rc;
  if (way == kFewRows) {
    rc = rows_forward<T>(p, c, st);
  } else if (!c.tc) {
    rc = fma_window<T>(p, c, false, st);
  } else if constexpr (sizeof(T) == 4) {
    rc = tc_window_forward<__nv_bfloat16, 64, 1, 3>(p, c, maps, status, st);
  } else {
    rc = p.D <= 64 ? tc_window_forward<T, 64, 1, 1>(p, c, maps, status, st) : c.tile > kTcRows ? tc_window_forward<T, 128, 2, 1>(p, c, maps, status, st)
                                                                            : tc_window_forward<T, 128, 1, 1>(p, c, maps, status, st);
  }
  if (rc != MVR_OK || c.splits == 1) return rc;
  const long long outputs = (long long)p.R * p.T * p.Hq * p.D;
  if (p.D % 4 == 0 && (uintptr_t)p.out % (4 * sizeof(T)) == 0 && (uintptr_t)p.rest % 8 == 0)
    launch_dependent(attn_join<T, 4>, dim3((unsigned)cdiv(outputs, 1024)), dim3(256), 0, st, p);
  else
    launch_dependent(attn_join<T, 1>, dim3((unsigned)cdiv(outputs, 256)), dim3(256), 0, st, p);
  return launched();
}

// Sums of the parts of the states [first, first + count) of every sequence, keys' in blockIdx.y 0, values' in 1: the parts lie one behind
// another, each (N, count, Hk, D).
template <typename T, int W>
__global__ void __launch_bounds__(256) window_sum(const float* part_k, const float* part_v, T* gk, T* gv, int N, long long outer, long long first,
                                                  long long count, int parts, float scale) {
  grid_dependency();
  const float* part = blockIdx.y ? part_v : part_k;
  T* dst = blockIdx.y ? gv : gk;
  const float factor = blockIdx.y ? 1.0f : scale;
  const long long n = N * count;
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * W; i < n; i += (long long)gridDim.x * 256 * W) {
    float v[W] = {};
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
      const Vec<float, W> x = *(const Vec<float, W>*)(part + s * n + i);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += x.v[k];
    }
    const long long image = i / count;
    Vec<T, W> out;
#pragma unroll
    for (int k = 0; k < W; ++k) out.v[k] = from_float<T>(v[k] * factor);
    *(Vec<T, W>*)(dst + image * outer + first + (i - image * count)) = out;
  }
}
template <typename T>
int sum_states(const AttnParams& p, const WindowCut& c, cudaStream_t st) {
  const long long row = (long long)p.Hk * p.D, lead = std::min<long long>(p.L, (long long)c.sink_tiles * c.state_tile);
  const bool wide = p.D % 4 == 0 && (((uintptr_t)p.gk | (uintptr_t)p.gv) % (4 * sizeof(T))) == 0;
  long long before = 0;  // floats of parts that lie before
  const auto sum = [&](long long first, long long count, int parts) {
    if (parts == 1 || count == 0) return;
    const dim3 grid(blocks_of(p.N * count * row, wide ? 1024 : 256), 2);
    launch_dependent(wide ? window_sum<T, 4> : window_sum<T, 1>, grid, dim3(256), 0, st, p.part_gk + before, p.part_gv + before, (T*)p.gk, (T*)p.gv, p.N, p.L * row,
                     first * row, count * row, parts, p.scale);
    before += parts * (p.N * count * row);
  };
  sum(0, lead, c.sink_parts);
  sum(lead, p.L - lead, c.row_splits);
  return launched();
}

// plain: the call's own tensors, where the operands are in pieces.
template <typename T>
int window_backward(const AttnParams& p, const AttnParams& plain, const WindowCut& c, const TcMaps& maps, bool boxes, int* status, cudaStream_t st) {
  const long long rows = (long long)p.R * p.T * p.Hq;
  int rc = MVR_OK;
  if (c.tc && std::is_same<T, __half>::value && cudaMemsetAsync(p.peaks, 0, (size_t)p.N * cdiv(p.L, 128) * p.Hk * 4, st) != cudaSuccess) {
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
  if (!c.tc) rc = fma_window<T>(p, c, true, st);
  else if constexpr (sizeof(T) == 4) rc = tc_window_backward<__nv_bfloat16, 64, 3>(p, c, maps, boxes, status, st);
  else rc = p.D <= 64 ? tc_window_backward<T, 64, 1>(p, c, maps, boxes, status, st) : tc_window_backward<T, 128, 1>(p, c, maps, boxes, status, st);
  if (rc == MVR_OK && c.splits > 1) rc = sum_parts<T>(p.part_gq, p.gq, rows * p.D, c.splits, p.scale, st);
  if (rc == MVR_OK) rc = sum_states<T>(p, c, st);
  return rc;
}

template <typename T>
int window_as(const mvr_attention* a, const mvr_window* w, bool backward, char* workspace, int* status, cudaStream_t st) {
  TcMaps maps = {};
  bool boxes = false, tc = tc_window(a, w);
  if (!backward && few_rows(a)) {
    const int64_t rows[3] = {a->R, a->T, a->Hq}, states[3] = {a->N, a->L, a->Hk};
    if (vectors_aligned(a->q, a->q_strides, rows, sizeof(T)) && vectors_aligned(a->k, a->k_strides, states, sizeof(T)) &&
        vectors_aligned(a->v, a->v_strides, states, sizeof(T))) {
      const WindowCut c = cut_window(a, w, false, kFewRows);
      return window_forward<T>(window_params(a, w, c, workspace), c, kFewRows, maps, status, st);
    }
  }
  if constexpr (sizeof(T) == 2) {
    tc = tc && ((uintptr_t)a->out | (uintptr_t)w->rest) % 16 == 0 && rows_aligned(a->q, a->q_strides, a);
    if (backward)
      tc = tc && rows_aligned(a->grad_out, a->g_strides, a) && (((uintptr_t)a->grad_q | (uintptr_t)a->grad_k | (uintptr_t)a->grad_v) & 15) == 0;
    tc = tc && tensor_maps<T>(a, backward, 1, maps, boxes);
  }
  const Way way = tc ? kTensorCores : kFloats;
  const WindowCut c = cut_window(a, w, backward, way);
  if (c.row_tiles > INT32_MAX) return MVR_ERR_TOO_LARGE;
  AttnParams p = window_params(a, w, c, workspace);
  const AttnParams plain = p;
  if constexpr (sizeof(T) == 4) {
    if (tc) {
      mvr_attention b;
      const int rc = split_operands(a, backward, c, workspace, b, p, st);
      if (rc != MVR_OK) return rc;
      if (!tensor_maps<__nv_bfloat16>(&b, backward, 3, maps, boxes)) return MVR_ERR_LAUNCH;
    }
  }
  return backward ? window_backward<T>(p, plain, c, maps, boxes, status, st) : window_forward<T>(p, c, way, maps, status, st);
}

long long window_bytes(const mvr_attention* a, const mvr_window* w, bool backward) {
  // (which way it goes is a matter of the call's addresses too)
  long long bytes = cut_window(a, w, backward, kFloats).bytes;
  if (tc_window(a, w)) bytes = std::max(bytes, cut_window(a, w, backward, kTensorCores).bytes);
  if (!backward && few_rows(a)) bytes = std::max(bytes, cut_window(a, w, false, kFewRows).bytes);
  return bytes;
}

int window_attention(const mvr_attention* a, const mvr_window* w, bool backward, void* workspace, int64_t bytes, int* status, void* stream) {
  const int rc = check_window(a, w, backward, false);
  if (rc != MVR_OK) return rc;
  const long long need = window_bytes(a, w, backward);
  if (bytes < need || (need > 0 && !workspace)) return MVR_ERR_WORKSPACE;
  const bool any_rows = a->R > 0 && a->T > 0, any_states = a->N > 0 && a->L > 0;
  if (!any_rows && (!backward || !any_states)) return MVR_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case MVR_F32: return window_as<float>(a, w, backward, (char*)workspace, status, st);
    case MVR_F16: return window_as<__half>(a, w, backward, (char*)workspace, status, st);
    default: return window_as<__nv_bfloat16>(a, w, backward, (char*)workspace, status, st);
  }
}

}  // namespace

extern "C" {

int mvr_window_attention_workspace(const mvr_attention* a, const mvr_window* w, int backward, int64_t* bytes) {
  if (!bytes) return MVR_ERR_NULL;
  const int rc = check_window(a, w, backward != 0, true);
  if (rc != MVR_OK) return rc;
  *bytes = window_bytes(a, w, backward != 0);
  return MVR_OK;
}

int mvr_window_attention_forward(const mvr_attention* a, const mvr_window* w, void* workspace, int64_t bytes, int* status, void* stream) {
  return window_attention(a, w, false, workspace, bytes, status, stream);
}

int mvr_window_attention_backward(const mvr_attention* a, const mvr_window* w, void* workspace, int64_t bytes, int* status, void* stream) {
  return window_attention(a, w, true, workspace, bytes, status, stream);
}

}  // extern "C"
