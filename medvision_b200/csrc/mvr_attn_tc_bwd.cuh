// Attention gradients on the tensor cores (float16, bfloat16; head sizes that are multiples of 8, up to 128).
//
// Two kernels, so that every sum has one place and one order.  One keeps 128 states and walks the rows that read them (dk, dv), the
// other keeps 128 rows and walks the states (dq); both form the scores again from the forward's lse, P = 2^(S scale - lse):
//
//   states kept:  S^T = K Q^T    dP^T = V G^T    dV += P^T G    dK += dS^T Q           dS = P (dP - delta)
//   rows kept:    S   = Q K^T    dP   = G V^T    dQ += dS K
//
// Scores, dP and the sums are in tensor memory; P and dS, rounded to T, go back over the scores and dP as left operands.  A
// warpgroup takes 32 columns of a tile, one row a thread.  A tile's chain (scores, exponentials, dP, dS, products) leaves every unit
// idle for a part of it, so up to 64 columns of a head two CTAs share an SM, each 128 x 64 at a time; beyond, tensor memory holds the
// sums of one CTA only, which takes 128 x 128.  One thread issues the products in an order in which those of
// one tile run under the exponentials of the next: dV(i), S(i+1), dK(i), dP(i+1), and S(i+1), dQ(i), dP(i+1).
//
// Measured (tensor pipe, function units, issue slots busy): 2 x 2048 rows of 16 heads of 64 (4 key heads) over 8191 and 6144 states,
// bfloat16: states kept 0.33 ms (36, 36, 36 %), rows kept 0.30 ms (29, 39, 41 %).  Bound by a step's chain, as the forward is: two CTAs
// an SM instead of one of twice the columns took the first from 0.53 to 0.39 ms, boxes in place of row copies and cheaper addresses the
// rest.  One exponential per score in each kernel is the price of
// sums without atomics.
//
// float16 has few small numbers: P is scaled by 2^10 on its way to dV, and dS by a power of two that brings a bound of |dS| <= |g.v| +
// |delta| to 2^14.  Where rows are kept every row has its own, from |g| of the row (2-norms, by attn_tc_delta) and the largest |v| of the
// states of its image and key head (by the first kernel; in a window, of the tiles of 128 states that it walks).  Where states are kept it is one power a CTA, from the largest |v| of its 128 states
// and the largest |g| and |delta| of the rows that it walks: delta averages the values of all states and has to be counted by itself.  So
// no gradient depends, in its bits or its range, on rows that have nothing to do with it (in a window: on states that no token reads, tokens that
// read none, and rows that read none of the CTA's states).  Both are taken out of the sums again, exactly.
#pragma once
#include <type_traits>

#include "mvr_attn_tc.cuh"

namespace mvr {

template <int DP>
constexpr int kGradStep = DP == 64 ? 64 : 128;  // columns of a tile

__device__ __forceinline__ void group_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

__device__ __forceinline__ float finite_or_0(float x) { return x <= 3e38f ? x : 0.0f; }  // x >= 0, or NaN

// Power of two for dS, from a bound of |dS| (1 where that is 0 or not finite).
template <typename T>
__device__ __forceinline__ float slope_scale(float most) {
  if constexpr (TcType<T>::code == 1) return 1.0f;
  if (!(most > 0.0f && most <= 3e38f)) return 1.0f;
  const int e = 14 - ilogbf(most);
  return ldexpf(1.0f, e < -60 ? -60 : e > 60 ? 60 : e);
}
template <typename T>
__device__ __forceinline__ float weight_shift() { return TcType<T>::code == 1 ? 0.0f : 10.0f; }

// 32 sums of a row to a row of floats, if there is one, or of Out; `left` of them are there.
template <typename Out, int PIECES>
__device__ __forceinline__ void put_part(Out* to, float* part, const uint32_t (&v)[32], int left) {
  if (part) {
    put_floats<PIECES>(part, v, left);
  } else if constexpr (PIECES == 3) {
    put_floats<PIECES>((float*)to, v, left);
  } else {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      if (i >= left) continue;
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = pack2<Out>(__uint_as_float(v[i + 2 * e]), __uint_as_float(v[i + 2 * e + 1]));
      *(uint4*)(to + i) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// ---- states kept: dk, dv ------------------------------------------------------------------------------
template <int DP, int PIECES>
struct TcStates {
  static_assert(PIECES == 1 || DP == 64, "");
  static constexpr int kStep = kGradStep<DP>, kBlocks = DP / 64, kTileBytes = kBlocks * 128 * 128, kStepBytes = kBlocks * kStep * 128;
  static constexpr int kStageBytes = PIECES * kStepBytes;  // Q (G) of a stage
  static constexpr int kGroups = kStep * 4, kLoaders = 64, kThreads = kGroups + kLoaders + 32, kStages = DP == 64 && PIECES == 1 ? 3 : 2;
  // tensor memory: scores (P over them), dP (dS over it), third pieces of both, dV, dK
  static constexpr int kScores = 0, kSlopes = kStep, kThird = 2 * kStep, kValues = kThird + (PIECES == 1 ? 0 : kStep), kKeys = kValues + DP;
  static constexpr int kColumns = PIECES == 1 ? 2 * kStep + 2 * DP : 512;
  static constexpr int kResident = DP == 64 && PIECES == 1 ? 2 : 1;
  struct Control {
    unsigned long long states, full[kStages], empty[kStages], landed, scores, slopes, weights, grads, done;
    uint32_t tmem;
    int lost, peak[3];  // peak: largest |v|, |g|, |delta| (float bits)
    alignas(16) float lse[kStages][kStep];    // negative
    alignas(16) float delta[kStages][kStep];  // negative
  };
  static constexpr size_t kShared = 2 * PIECES * (size_t)kTileBytes + 2 * kStages * (size_t)kStageBytes + sizeof(Control) + 1024;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// BOXES: tiles of rows are boxes of the tensors (maps.q, maps.g).
// MODE: a window (kWindow, kWindowRounded) or not.  There a tile of states meets the rows whose windows reach it; the first tiles, which all tokens
// may read, are cut into more parts.
template <typename T, int DP, bool BOXES, int PIECES, int MODE = kAll>
__global__ void __launch_bounds__(TcStates<DP, PIECES>::kThreads, TcStates<DP, PIECES>::kResident)
attn_tc_dkv(const __grid_constant__ AttnParams p, const __grid_constant__ TcMaps maps, int* status) {
  typedef TcStates<DP, PIECES> F;
  typedef std::conditional_t<PIECES == 1, T, float> Out;
  // A window's slopes in two pieces, as in dq: with states read by a few rows one rounding of each was up to 1.57 times as far off as the plain
  // form, with two 1.05.  The second product costs 6 % of a training step (2 x 8192 tokens, windows of 1024 + 4, bf16: 627 to 665 us).
  constexpr bool WINDOW = MODE >= kWindow, kRest = WINDOW && PIECES == 1;
  constexpr bool kRestWeights = MODE == kWindow && PIECES == 1;  // P too: see the forward
  extern __shared__ char tc_smem[];
  char* base = tc_smem + ((1024 - (smem_at(tc_smem) & 1023)) & 1023);  // K, V, then Q and G of the stages
  typename F::Control& c = *(typename F::Control*)(base + 2 * PIECES * F::kTileBytes + 2 * F::kStages * F::kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kLoader = F::kGroups / 32, kIssuer = kLoader + F::kLoaders / 32;
  if (threadIdx.x == 0) {
    bar_init(smem_at(&c.states), 1);
    for (int i = 0; i < F::kStages; ++i) {
      bar_init(smem_at(&c.full[i]), F::kLoaders / 32);
      bar_init(smem_at(&c.empty[i]), 1);
    }
    bar_init(smem_at(&c.landed), 1);
    bar_init(smem_at(&c.scores), 1);
    bar_init(smem_at(&c.slopes), 1);
    bar_init(smem_at(&c.weights), F::kGroups / 32);
    bar_init(smem_at(&c.grads), F::kGroups / 32);
    bar_init(smem_at(&c.done), 1);
    c.lost = 0;
    c.peak[0] = c.peak[1] = c.peak[2] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == kIssuer) tmem_alloc(smem_at(&c.tmem), F::kColumns);
  const int state_tiles = (p.L + 127) / 128, hk = blockIdx.y;
  const StateTile st = WINDOW ? state_tile(p, blockIdx.x, state_tiles) : StateTile{(int)blockIdx.x / state_tiles, (int)blockIdx.x % state_tiles, (int)blockIdx.z, false};
  const int n = st.n, j0 = st.tile * 128, split = st.part;
  // one row a thread: its state, and whether it is read
  const int r = ((warp & 3) << 5) + lane, part_of = warp >> 2, j = j0 + r;
  bool in = false;
  if (warp < kLoader) in = j < states_of(p, n) && (!p.mask || p.mask[(long long)n * p.L + j] != 0);
  const bool any = __syncthreads_or(in);
  const RowTile o = image_rows(p, n);
  const int row_tiles = (o.rows + F::kStep - 1) / F::kStep, per = (row_tiles + p.row_splits - 1) / p.row_splits;
  int first = split * per * F::kStep, count = any ? max(0, min(row_tiles, (split + 1) * per) - split * per) : 0, row_lo = 0, row_hi = 0;  // first: row
  int end = o.rows;  // (a window: rows behind read none of the states, and may hold NaN)
  if (WINDOW) {
    const Places at = places_of(p, n);
    rows_of_state(p, at, j, row_lo, row_hi);  // (one state a thread)
    const TileRows r = rows_of_states(p, st, at, j0, 128, states_of(p, n), F::kStep);
    first = r.first;
    end = r.end;
    count = any ? r.count : 0;
  }
  // what lies behind D in the rows' tiles stays 0
  if (count > 0 && p.W < DP) {
    for (int e = threadIdx.x; e < 2 * F::kStages * F::kStageBytes / 16; e += F::kThreads)
      *(uint4*)(base + 2 * PIECES * F::kTileBytes + e * 16) = make_uint4(0, 0, 0, 0);
    fence_async_proxy();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = c.tmem;
  volatile int* lost = &c.lost;
  const float shift = weight_shift<T>();

  if (warp == kIssuer) {
    if (count > 0) {
      if (elect_one()) {
        bar_expect(smem_at(&c.states), 2 * PIECES * F::kTileBytes);
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece)
#pragma unroll
          for (int b = 0; b < F::kBlocks; ++b)
#pragma unroll
            for (int r = 0; r < 128; r += kTcBox) {
              const uint32_t to = smem_at(base + piece * F::kTileBytes + b * 16384 + r * 128);
              tma_load_4d(to, &maps.k, smem_at(&c.states), b * 64, hk, j0 + r, n + piece * p.N);
              tma_load_4d(to + PIECES * F::kTileBytes, &maps.v, smem_at(&c.states), b * 64, hk, j0 + r, n + piece * p.N);
            }
      }
      __syncwarp();
      const int depth = (p.D + 15) / 16;
      const uint32_t s_shape = tc_shape<T>(F::kStep, false), d_shape = tc_shape<T>(depth * 16, true);
      const char* steps = base + 2 * PIECES * F::kTileBytes;
      const uint64_t tiles_k = desc_k_major(smem_at(base)), steps_k = desc_k_major(smem_at(steps)), steps_mn = desc_mn_major(smem_at(steps), F::kStep * 128);
      const auto scores = [&](int left, int right, int to, unsigned long long* bar) {  // 128 x kStep over D, both K-major
        if (elect_one()) {
          for_pairs<PIECES>([&](int a, int b, bool first) {
            mma_rows<DP / 16>(tmem + to, tiles_k + (((left * PIECES + a) * F::kTileBytes) >> 4), steps_k + ((right * F::kStageBytes + b * F::kStepBytes) >> 4),
                              s_shape, depth, 16384, F::kStep * 128, !first);
          });
          mma_commit(smem_at(bar));
        }
        __syncwarp();
      };
      const auto sums = [&](int from, int right, int to, bool add) {  // over the rows
        if (elect_one()) {
          for_pairs<PIECES>([&](int a, int b, bool first) {
#pragma unroll
            for (int i = 0; i < F::kStep / 16; ++i) {
              const int at = a == 2 ? F::kThird + (from == F::kSlopes ? F::kStep / 2 : 0) + i * 8 : from + (i >> 1) * 32 + a * 16 + (i & 1) * 8;
              mma_ts(tmem + to, tmem + at, steps_mn + ((right * F::kStageBytes + b * F::kStepBytes + i * 2048) >> 4), d_shape, (PIECES == 1 && add) || i > 0 || !first);
            }
          });
          if (from == F::kSlopes ? kRest : kRestWeights) {
#pragma unroll
            for (int i = 0; i < F::kStep / 16; ++i)
              mma_ts(tmem + to, tmem + from + (i >> 1) * 32 + 16 + (i & 1) * 8, steps_mn + ((right * F::kStageBytes + i * 2048) >> 4), d_shape, true);
          }
        }
        __syncwarp();
      };
      const auto commit = [&](unsigned long long* bar) {
        if (elect_one()) mma_commit(smem_at(bar));
        __syncwarp();
      };
      bar_pass(smem_at(&c.states), 0, lost);
      bar_pass(smem_at(&c.full[0]), 0, lost);
      tc_fence_after();
      scores(0, 0, F::kScores, &c.scores);
      scores(1, 1, F::kSlopes, &c.slopes);
      for (int i = 0; i < count; ++i) {
        const int now = i % F::kStages, next = (i + 1) % F::kStages;
        bar_pass(smem_at(&c.weights), i & 1, lost);
        tc_fence_after();
        sums(F::kScores, 1 + 2 * now, F::kValues, i > 0);
        if (i + 1 < count) {
          bar_pass(smem_at(&c.full[next]), ((i + 1) / F::kStages) & 1, lost);
          tc_fence_after();
          scores(0, 2 * next, F::kScores, &c.scores);
        }
        bar_pass(smem_at(&c.grads), i & 1, lost);
        tc_fence_after();
        sums(F::kSlopes, 2 * now, F::kKeys, i > 0);
        commit(&c.empty[now]);
        if (i + 1 < count) scores(1, 1 + 2 * next, F::kSlopes, &c.slopes);
      }
      commit(&c.done);
      if (*lost) {
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.states), 0) && nanoseconds() - t < kWaitLimit) {}
      }
    }
  } else if (warp >= kLoader) {
    // Rows of Q and G.  Without an index a tile of rows is a box of the tensors: tokens, and the heads that share the key head.  Else
    // 16 bytes a copy, 32 rows of a warp at a time, their places (in 16 bytes from the tensors' beginnings) handed round by shuffles.
    // (TMA's gathering of four rows a copy took half as long again.)  What belongs to the rows of the next tile is looked up while the
    // copies of this one are under way.
    constexpr int kParts = F::kStep / F::kLoaders, kPieces = DP / 8, kAtOnce = 32 / kPieces;  // rows of one round of copies
    const int piece = lane % kPieces;
    const bool there = piece * 8 < p.W;
    unsigned q[kParts], g[kParts];  // ~0: no row
    float lse[kParts], delta[kParts];
    const auto look_up = [&](int i) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        const int at = first + i * F::kStep + (warp - kLoader) * 32 + k * F::kLoaders + lane;
        q[k] = g[k] = ~0u;
        lse[k] = INFINITY, delta[k] = 0.0f;  // no row: P = 0
        if (i < count && at < end) {
          const Row row = row_of(p, o, at, hk);
          if (!BOXES) q[k] = (unsigned)((row.r * p.q_r + row.t * p.q_t + row.h * p.q_h) >> 3);
          if (!BOXES) g[k] = (unsigned)((row.r * p.g_r + row.t * p.g_t + row.h * p.g_h) >> 3);
          const long long number = row_number(p, row);
          lse[k] = p.lse[number];
          delta[k] = p.delta[number];
        }
      }
    };
    const auto arrived = [&](int stage) {
      fence_async_proxy();
      bar_arrive_warp(smem_at(&c.full[stage]));
    };
    const char *q_piece = (const char*)p.q + (there ? piece * 16 : 0), *g_piece = (const char*)p.g + (there ? piece * 16 : 0);
    const uint32_t to_block = smem_at(base + 2 * PIECES * F::kTileBytes) + (piece >> 3) * (F::kStep * 128);
    look_up(0);
    bool pending = false, cleared = false;
    int i = 0;
    for (; i < count; ++i) {
      const int stage = i % F::kStages;
      if (i >= F::kStages && !bar_wait_warp(smem_at(&c.empty[stage]), (i / F::kStages - 1) & 1, lost)) break;
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        const int mine = (warp - kLoader) * 32 + k * F::kLoaders;
        c.lse[stage][mine + lane] = lse[k] == -INFINITY ? -INFINITY : shift - lse[k];
        c.delta[stage][mine + lane] = -delta[k];
        if (BOXES) continue;
#pragma unroll
        for (int e = 0; e < 32 / kAtOnce; ++e) {
          const int from = e * kAtOnce + lane / kPieces, row = mine + from;
          const unsigned qk = __shfl_sync(~0u, q[k], from), gk = __shfl_sync(~0u, g[k], from);
          const uint32_t to = to_block + 2 * stage * F::kStageBytes + row * 128 + (((piece ^ row) & 7) << 4);
          if (there) {
#pragma unroll
            for (int part = 0; part < PIECES; ++part) {
              copy16(to + part * F::kStepBytes, q_piece + (qk == ~0u ? 0 : ((long long)qk * 8 + part * p.q_piece) * 2), qk != ~0u);
              copy16(to + F::kStageBytes + part * F::kStepBytes, g_piece + (gk == ~0u ? 0 : ((long long)gk * 8 + part * p.g_piece) * 2), gk != ~0u);
            }
          }
        }
      }
      if (BOXES) {
        const uint32_t bar = smem_at(&c.full[stage]), to = smem_at(base + 2 * PIECES * F::kTileBytes) + 2 * stage * F::kStageBytes;
        __syncwarp();
        // Rows of the box behind the last that reads a state (of the last tile): zero before the products see them.  (They are 0 times 0 there, but
        // 0 times NaN otherwise.)  Such a box lands at a barrier of its own.
        cleared = WINDOW && end < o.rows && first + (i + 1) * F::kStep > end;
        if (warp != kLoader) {
          bar_arrive_warp(bar);
        } else if (elect_one()) {
          const uint32_t on = cleared ? smem_at(&c.landed) : bar;
          bar_expect(on, 2 * F::kStageBytes);
          const int token = p.by_G.quotient(first + i * F::kStep);
#pragma unroll
          for (int part = 0; part < PIECES; ++part)
#pragma unroll
            for (int b = 0; b < F::kBlocks; ++b) {
              const uint32_t at = to + part * F::kStepBytes + b * F::kStep * 128;
              tma_load_4d(at, &maps.q, on, b * 64, hk * p.G, token, n + part * p.R);
              tma_load_4d(at + F::kStageBytes, &maps.g, on, b * 64, hk * p.G, token, n + part * p.R);
            }
        }
        __syncwarp();
        if (WINDOW && cleared && warp == kLoader) {
          bar_pass(smem_at(&c.landed), 0, lost);
          char* rows = base + 2 * PIECES * F::kTileBytes + 2 * stage * F::kStageBytes;  // blocks of kStep rows, of Q and then of G
          for (int row = end - (first + i * F::kStep) + lane; row < F::kStep; row += 32)
#pragma unroll
            for (int b = 0; b < 2 * PIECES * F::kBlocks; ++b)
#pragma unroll
              for (int k = 0; k < 8; ++k) *(uint4*)(rows + (b * F::kStep + row) * 128 + (((k + lane) & 7) << 4)) = make_uint4(0, 0, 0, 0);
          arrived(stage);
        }
        look_up(i + 1);
        continue;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      look_up(i + 1);
      // the first stages are told of behind the copies of the next; from the last on, a stage is waited for at once
      if (pending) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        arrived((i - 1) % F::kStages);
      }
      pending = i + 1 < count && i + 1 < F::kStages;
      if (!pending) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        arrived(stage);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (BOXES && *lost && warp == kLoader) {  // given up: the copies under way end, or the limit passes, before the CTA does
      const unsigned long long t = nanoseconds();
      while (cleared && !bar_try(smem_at(&c.landed), 0) && nanoseconds() - t < kWaitLimit) {}
      for (int k = max(0, i - F::kStages); k < i; ++k)
        while (!bar_try(smem_at(&c.full[k % F::kStages]), (k / F::kStages) & 1) && nanoseconds() - t < kWaitLimit) {}
    }
  } else {
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    float factor = 1.0f;  // of dS
    if (count > 0 && TcType<T>::code == 0) {
      float most[3] = {};  // |v| of this thread's state, if it is read; |g|, |delta| of rows, whole tiles of them together
      const int before = o.order ? p.tiles[n] : n * ((o.rows + kTcRows - 1) / kTcRows), stop = min(end, first + count * F::kStep);
      // (a window's walk begins and ends within tiles: their rows one by one)
      const int tile0 = WINDOW ? (first + kTcRows - 1) / kTcRows : first / kTcRows, tile1 = WINDOW && stop < o.rows ? stop / kTcRows : (stop + kTcRows - 1) / kTcRows;
      for (int t = tile0 + threadIdx.x; t < tile1; t += F::kGroups) {
        const float2 peak = p.row_peaks[(long long)(before + t) * p.Hk + hk];
        most[1] = fmaxf(most[1], peak.x);
        most[2] = fmaxf(most[2], peak.y);
      }
      if (WINDOW) {
        const int head = min(stop, tile0 * kTcRows), tail = max(head, tile1 * kTcRows), alone = head - first + max(0, stop - tail);
        for (int i = threadIdx.x; i < alone; i += F::kGroups) {
          const long long number = row_number(p, row_of(p, o, first + i < head ? first + i : tail + (first + i - head), hk));
          most[1] = fmaxf(most[1], finite_or_0(p.norm[number]));
          most[2] = fmaxf(most[2], finite_or_0(fabsf(p.delta[number])));
        }
      }
      bar_pass(smem_at(&c.states), 0, lost);
      if (in && part_of == 0 && (!WINDOW || row_lo < row_hi)) {
        const char* row = base + F::kTileBytes + r * 128;
#pragma unroll
        for (int piece = 0; piece < DP / 8; ++piece) {
          const uint4 v = *(const uint4*)(row + (piece >> 3) * 16384 + (((piece ^ r) & 7) << 4));
          const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*(const __half2*)&words[k]);
            most[0] = fmaf(f.x, f.x, fmaf(f.y, f.y, most[0]));
          }
        }
        most[0] = finite_or_0(sqrtf(most[0]));
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        for (int d = 16; d; d >>= 1) most[k] = fmaxf(most[k], __shfl_xor_sync(~0u, most[k], d));
        if (lane == 0) atomicMax(&c.peak[k], __float_as_int(most[k]));
      }
      group_sync(F::kGroups);
      if (threadIdx.x == 0) atomicMax(p.peaks + (WINDOW ? (long long)n * state_tiles + st.tile : (long long)n) * p.Hk + hk, c.peak[0]);
      factor = slope_scale<T>(__int_as_float(c.peak[1]) * __int_as_float(c.peak[0]) + __int_as_float(c.peak[2]));
    }
    const float2 slope2 = make_float2(factor * exp2f(-shift), factor * exp2f(-shift)), scale2 = make_float2(p.scale_log2, p.scale_log2);
    // With pieces, each tile's sums are added up in registers (dv in the first warpgroup, dk in the second): see the forward.
    float acc[PIECES == 1 ? 1 : 64] = {};
    const auto collect = [&](int from) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t v[32];
        tmem_load32(v, tmem + lanes + from + q * 32);
        tmem_wait_load();
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[PIECES == 1 ? 0 : q * 32 + e] += __uint_as_float(v[e]);
      }
    };
    // (A state that is not read is a row of its own in both products: whatever comes of it reaches no other, and is not stored.)
    for (int i = 0; i < count; ++i) {
      const int stage = i % F::kStages;
      bar_pass(smem_at(&c.full[stage]), (i / F::kStages) & 1, lost);
      bar_pass(smem_at(&c.scores), i & 1, lost);
      tc_fence_after();
      if constexpr (PIECES == 3) {
        if (i > 0 && part_of == 0) collect(F::kValues);  // (of the tile before: its product ended before these scores)
      }
      const int col = part_of * 32;
      // rows that do not read this state
      const uint32_t bits = WINDOW ? bits_below(row_hi - (first + i * F::kStep + col)) & ~bits_below(row_lo - (first + i * F::kStep + col)) : ~0u;
      float2 w[16];
      uint32_t v[32], u[16], u1[PIECES == 1 && !kRest ? 1 : 16], u2[PIECES == 1 ? 1 : 16];
      tmem_load32(v, tmem + lanes + F::kScores + col);
      tmem_wait_load();
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 lse = *(const float4*)&c.lse[stage][col + e];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 x = fma2(make_float2(__uint_as_float(v[e + 2 * k]), __uint_as_float(v[e + 2 * k + 1])), scale2,
                                k ? make_float2(lse.z, lse.w) : make_float2(lse.x, lse.y));
          float2 y = make_float2(exp2_fast(x.x), exp2_fast(x.y));
          if (WINDOW && bits != ~0u) y = make_float2((bits >> (e + 2 * k)) & 1 ? y.x : 0.0f, (bits >> (e + 2 * k + 1)) & 1 ? y.y : 0.0f);
          w[e / 2 + k] = TcType<T>::code == 0 ? mul2(y, slope2) : y;
          if constexpr (PIECES == 1) u[e / 2 + k] = pack2<T>(y.x, y.y);
          else pieces_of(y, u[e / 2 + k], u1[e / 2 + k], u2[e / 2 + k]);
          if constexpr (kRestWeights) {
            const float2 f = floats(*(const Two<T>*)&u[e / 2 + k]);
            u1[e / 2 + k] = pack2<T>(y.x - f.x, y.y - f.y);
          }
        }
      }
      tmem_store16(tmem + lanes + F::kScores + col, u);  // (over this warpgroup's own scores)
      if constexpr (kRestWeights) tmem_store16(tmem + lanes + F::kScores + col + 16, u1);
      if constexpr (PIECES == 3) {
        tmem_store16(tmem + lanes + F::kScores + col + 16, u1);
        tmem_store16(tmem + lanes + F::kThird + col / 2, u2);
      }
      tmem_wait_store();
      tc_fence_before();
      bar_arrive_warp(smem_at(&c.weights));
      bar_pass(smem_at(&c.slopes), i & 1, lost);
      tc_fence_after();
      if constexpr (PIECES == 3) {
        if (i > 0 && part_of == 1) collect(F::kKeys);
      }
      tmem_load32(v, tmem + lanes + F::kSlopes + col);
      tmem_wait_load();
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 delta = *(const float4*)&c.delta[stage][col + e];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float2 ds = mul2(w[e / 2 + k], add2(make_float2(__uint_as_float(v[e + 2 * k]), __uint_as_float(v[e + 2 * k + 1])),
                                              k ? make_float2(delta.z, delta.w) : make_float2(delta.x, delta.y)));
          if (WINDOW && bits != ~0u) ds = make_float2((bits >> (e + 2 * k)) & 1 ? ds.x : 0.0f, (bits >> (e + 2 * k + 1)) & 1 ? ds.y : 0.0f);
          if constexpr (PIECES == 1) u[e / 2 + k] = pack2<T>(ds.x, ds.y);
          else pieces_of(ds, u[e / 2 + k], u1[e / 2 + k], u2[e / 2 + k]);
          if constexpr (kRest) {
            const float2 f = floats(*(const Two<T>*)&u[e / 2 + k]);
            u1[e / 2 + k] = pack2<T>(ds.x - f.x, ds.y - f.y);
          }
        }
      }
      tmem_store16(tmem + lanes + F::kSlopes + col, u);
      if constexpr (kRest) tmem_store16(tmem + lanes + F::kSlopes + col + 16, u1);
      if constexpr (PIECES == 3) {
        tmem_store16(tmem + lanes + F::kSlopes + col + 16, u1);
        tmem_store16(tmem + lanes + F::kThird + F::kStep / 2 + col / 2, u2);
      }
      tmem_wait_store();
      tc_fence_before();
      bar_arrive_warp(smem_at(&c.grads));
    }
    if (count > 0) bar_pass(smem_at(&c.done), 0, lost);
    if (__all_sync(~0u, *lost == 0)) {
      tc_fence_after();
      // the first half of the warpgroups stores dv, the other dk
      constexpr int kHalf = F::kGroups / 256;
      const bool keys = part_of >= kHalf;
      const long long all = (long long)p.N * p.L * p.Hk * p.D, at = (((long long)n * p.L + j) * p.Hk + hk) * p.D;
      const PartPlace place = WINDOW ? part_place(p, st, j, hk, 128) : PartPlace{p.row_splits > 1, split * all + at};
      const bool parts = place.parts;
      const float f = in ? (keys ? (parts ? 1.0f : p.scale) / factor : exp2f(-shift)) : 0.0f;
      Out* to = (Out*)(keys ? p.gk : p.gv) + at;
      float* part = parts ? (keys ? p.part_gk : p.part_gv) + place.at : nullptr;
      const auto put = [&](int q, uint32_t (&v)[32]) {
        // (a state that is not read: its sums may be NaN where rows hold NaN)
        if (j < p.L) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = in && count > 0 ? __float_as_uint(__uint_as_float(v[i]) * f) : 0;
          put_part<Out, PIECES>(to + q * 32, part ? part + q * 32 : nullptr, v, p.D - q * 32);
        }
      };
      if constexpr (PIECES == 3) {
        if (count > 0) collect(keys ? F::kKeys : F::kValues);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(acc[q * 32 + i]);
          if (q * 32 < p.D) put(q, v);
        }
      } else {
#pragma unroll 1
        for (int q = part_of % kHalf; q < DP / 32; q += kHalf) {
          if (q * 32 >= p.D) break;
          uint32_t v[32] = {};
          if (count > 0) {
            tmem_load32(v, tmem + lanes + (keys ? F::kKeys : F::kValues) + q * 32);
            tmem_wait_load();
          }
          put(q, v);
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    if (*lost) {
      if (lane == 0) {
        if (status) atomicOr(status, 2);
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.done), 0) && nanoseconds() - t < kWaitLimit) {}
      }
      __syncwarp();
    }
    tc_fence_after();
    tmem_free(tmem, F::kColumns);
  }
}

// ---- rows kept: dq ------------------------------------------------------------------------------------
template <int DP, int MODE, int PIECES>
struct TcRows {
  static constexpr int kStep = kGradStep<DP>, kBlocks = DP / 64, kTileBytes = kBlocks * 128 * 128, kStepBytes = kBlocks * kStep * 128, kSlots = 4;
  static constexpr int kRowsBytes = PIECES * kTileBytes, kSlotBytes = PIECES * kStepBytes;
  static constexpr int kGroups = kStep * 4, kThreads = kGroups + 96, kMaxTiles = kTcMaxStates / kStep;
  // tensor memory: scores, dP (dS over it), third pieces of dS, dQ
  static constexpr int kScores = 0, kSlopes = kStep, kThird = 2 * kStep, kSums = kThird + (PIECES == 1 ? 0 : kStep / 2), kColumns = DP == 64 ? 256 : 512;
  static constexpr int kResident = DP == 64 && PIECES == 1 ? 2 : 1;
  struct Control {
    unsigned long long full[kSlots], empty[kSlots], clean[kSlots], rows, scores, taken, slopes, grads, done;
    uint32_t tmem;
    int lost, tiles;
    unsigned short list[MODE == kListed ? kMaxTiles : 1];
    StateBits<kStep> bits[MODE == kListed ? kMaxTiles : 1];
  };
  static constexpr size_t kShared = 2 * (size_t)kRowsBytes + kSlots * (size_t)kSlotBytes + sizeof(Control) + 1024;
};

template <typename T, int DP, int MODE, int PIECES>
__global__ void __launch_bounds__(TcRows<DP, MODE, PIECES>::kThreads, TcRows<DP, MODE, PIECES>::kResident)
attn_tc_dq(const __grid_constant__ AttnParams p, const __grid_constant__ TcMaps maps, int* status) {
  typedef TcRows<DP, MODE, PIECES> F;
  constexpr bool MASK = MODE != kAll;
  // A window's slopes in two pieces: those of a row sum to 0, so that with few states dq is the smaller part of what is summed, and one rounding
  // of each to a half type was up to 1.2 times as far off as the rounding of dq itself.
  constexpr bool kRest = MODE == kWindow && PIECES == 1;
  typedef std::conditional_t<PIECES == 1, T, float> Out;
  extern __shared__ char tc_smem[];
  char* base = tc_smem + ((1024 - (smem_at(tc_smem) & 1023)) & 1023);  // Q, G, then the ring
  char* ring = base + 2 * F::kRowsBytes;
  typename F::Control& c = *(typename F::Control*)(ring + F::kSlots * F::kSlotBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kLoader = F::kGroups / 32, kIssuer = kLoader + 1, kCleaner = kLoader + 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::kSlots; ++i) {
      bar_init(smem_at(&c.full[i]), 1);
      bar_init(smem_at(&c.empty[i]), 1);
      bar_init(smem_at(&c.clean[i]), 1);
    }
    bar_init(smem_at(&c.rows), F::kGroups / 32);
    bar_init(smem_at(&c.scores), 1);
    bar_init(smem_at(&c.taken), F::kGroups / 32);
    bar_init(smem_at(&c.slopes), 1);
    bar_init(smem_at(&c.grads), F::kGroups / 32);
    bar_init(smem_at(&c.done), 1);
    c.lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == kIssuer) tmem_alloc(smem_at(&c.tmem), F::kColumns);
  RowTile o;
  const bool some = row_tile(p, blockIdx.x, kTcRows, o);
  const int hk = blockIdx.y, split = blockIdx.z;
  const int all = (p.L + F::kStep - 1) / F::kStep, per = (all + p.splits - 1) / p.splits;
  const int begin = split * per * F::kStep;
  int end = 0;
  if (some) end = min(states_of(p, o.n), (split + 1) * per * F::kStep);
  if (MODE == kListed && some && begin < end) list_tiles(p, o.n, begin, end, c.list, c.bits, &c.tiles);
  Places places = {};
  int states = 0;
  Span span = {};
  if (MODE == kWindow && some) {
    places = places_of(p, o.n);
    states = states_of(p, o.n);
    span = span_of(p, places, p.by_G.quotient(o.first), p.by_G.quotient(min(o.first + kTcRows, o.rows) - 1), states);
  }
  const SpanTiles<F::kStep> window(span);
  const int window_first = split * p.tiles_per;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tiles = MODE == kWindow ? max(0, min(p.tiles_per, window.count - window_first))
                    : !some || begin >= end ? 0 : MODE == kListed ? c.tiles : (end - begin + F::kStep - 1) / F::kStep;
  const uint32_t tmem = c.tmem;
  volatile int* lost = &c.lost;
  const auto first_of = [&](int i) {
    return MODE == kWindow ? window.first(window_first + i) : begin + (MODE == kListed ? (int)c.list[i] : i) * F::kStep;
  };

  if (warp == kLoader) {
    int i = 0;
    for (; i < 2 * tiles; ++i) {  // K0 V0 K1 V1 ...
      const int slot = i % F::kSlots;
      const uint32_t bar = smem_at(&c.full[slot]);
      if (i >= F::kSlots && !bar_wait_warp(smem_at(&c.empty[slot]), (i / F::kSlots - 1) & 1, lost)) break;
      const int j = first_of(i >> 1);
      if (elect_one()) {
        bar_expect(bar, F::kSlotBytes);
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece)
#pragma unroll
          for (int b = 0; b < F::kBlocks; ++b)
#pragma unroll
            for (int r = 0; r < F::kStep; r += kTcBox)
              tma_load_4d(smem_at(ring + slot * F::kSlotBytes + piece * F::kStepBytes + (b * F::kStep + r) * 128), i & 1 ? &maps.v : &maps.k, bar,
                          b * 64, hk, j + r, o.n + piece * p.N);
      }
      __syncwarp();
    }
    if (*lost)
      for (int k = max(0, i - F::kSlots); k < i; ++k) {
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.full[k % F::kSlots]), (k / F::kSlots) & 1) && nanoseconds() - t < kWaitLimit) {}
      }
  } else if (warp == kIssuer) {
    if (tiles > 0) {
      const int depth = (p.D + 15) / 16;
      const uint32_t s_shape = tc_shape<T>(F::kStep, false), d_shape = tc_shape<T>(depth * 16, true);
      const uint64_t rows_k = desc_k_major(smem_at(base)), ring_k = desc_k_major(smem_at(ring)), ring_mn = desc_mn_major(smem_at(ring), F::kStep * 128);
      const auto scores = [&](int left, int slot, int to, unsigned long long* bar) {
        if (elect_one()) {
          for_pairs<PIECES>([&](int a, int b, bool first) {
            mma_rows<DP / 16>(tmem + to, rows_k + ((left * F::kRowsBytes + a * F::kTileBytes) >> 4), ring_k + ((slot * F::kSlotBytes + b * F::kStepBytes) >> 4),
                              s_shape, depth, 16384, F::kStep * 128, !first);
          });
          mma_commit(smem_at(bar));
        }
        __syncwarp();
      };
      const auto commit = [&](unsigned long long* bar) {
        if (elect_one()) mma_commit(smem_at(bar));
        __syncwarp();
      };
      const auto wait_full = [&](int i) { bar_pass(smem_at(&c.full[i % F::kSlots]), (i / F::kSlots) & 1, lost); };
      bar_pass(smem_at(&c.rows), 0, lost);
      wait_full(0);
      wait_full(1);
      tc_fence_after();
      scores(0, 0, F::kScores, &c.scores);
      scores(1, 1, F::kSlopes, &c.slopes);
      commit(&c.empty[1]);
      for (int i = 0; i < tiles; ++i) {
        const int k = 2 * i, next = k + 2;
        if (i + 1 < tiles) {
          wait_full(next);
          bar_pass(smem_at(&c.taken), i & 1, lost);
          tc_fence_after();
          scores(0, next % F::kSlots, F::kScores, &c.scores);
          wait_full(next + 1);
        }
        if (MASK) bar_pass(smem_at(&c.clean[k % F::kSlots]), (k / F::kSlots) & 1, lost);
        bar_pass(smem_at(&c.grads), i & 1, lost);
        tc_fence_after();
        if (elect_one()) {
          for_pairs<PIECES>([&](int a, int b, bool first) {
#pragma unroll
            for (int e = 0; e < F::kStep / 16; ++e) {
              const int at = a == 2 ? F::kThird + e * 8 : F::kSlopes + (e >> 1) * 32 + a * 16 + (e & 1) * 8;
              mma_ts(tmem + F::kSums, tmem + at, ring_mn + (((k % F::kSlots) * F::kSlotBytes + b * F::kStepBytes + e * 2048) >> 4), d_shape,
                     (PIECES == 1 && i > 0) || e > 0 || !first);
            }
          });
          if constexpr (kRest) {
#pragma unroll
            for (int e = 0; e < F::kStep / 16; ++e)
              mma_ts(tmem + F::kSums, tmem + F::kSlopes + (e >> 1) * 32 + 16 + (e & 1) * 8, ring_mn + (((k % F::kSlots) * F::kSlotBytes + e * 2048) >> 4), d_shape, true);
          }
          mma_commit(smem_at(&c.empty[k % F::kSlots]));
        }
        __syncwarp();
        if (i + 1 < tiles) {
          scores(1, (next + 1) % F::kSlots, F::kSlopes, &c.slopes);
          commit(&c.empty[(next + 1) % F::kSlots]);
        }
      }
      commit(&c.done);
    }
  } else if (MASK && warp == kCleaner) {
    // rows of K that are left out may hold NaN: zero before they meet the zeros of dS
    for (int i = 0; i < tiles; ++i) {
      const int k = 2 * i, slot = k % F::kSlots;
      if (!__all_sync(~0u, bar_wait(smem_at(&c.full[slot]), (k / F::kSlots) & 1, lost))) break;
      StateBits<F::kStep> bits;
      if constexpr (MODE == kWindow) bits = bits_of_span<F::kStep>(span, first_of(i));
      else bits = c.bits[i];
      for (int piece = 0; piece < PIECES; ++piece)
        clear_rows<F::kStep, F::kBlocks>(ring + slot * F::kSlotBytes + piece * F::kStepBytes, bits, lane);
      if (lane == 0) bar_arrive(smem_at(&c.clean[slot]));
    }
  } else if (warp < kLoader) {
    const int r = threadIdx.x & 127, part_of = warp >> 2, j0 = o.first + r;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const bool mine = some && j0 < o.rows;
    Row w = {};
    long long number = 0;
    float lse = INFINITY, delta = 0.0f, factor = 1.0f;  // factor: of dS
    Span own = {};
    // (float16, a window: the largest |v| of the tiles of states that this part walks)
    int peak = 0;
    if (MODE == kWindow && TcType<T>::code == 0 && tiles > 0) {
      const int state_tiles = (p.L + 127) / 128;
      for (int i = lane; i < tiles; i += 32)
        for (int t = first_of(i) / 128; t <= min(state_tiles - 1, (first_of(i) + F::kStep - 1) / 128); ++t)
          peak = max(peak, p.peaks[((long long)o.n * state_tiles + t) * p.Hk + hk]);
      peak = __reduce_max_sync(~0u, peak);
    }
    if (mine) {
      w = row_of(p, o, j0, hk);
      if (MODE == kWindow) own = span_of(p, places, w.t, w.t, states);
      number = row_number(p, w);
      if (tiles > 0) {
        lse = p.lse[number];
        if (lse == -INFINITY) lse = INFINITY;
        delta = p.delta[number];
        if (TcType<T>::code == 0) {
          if (MODE != kWindow) peak = p.peaks[(long long)o.n * p.Hk + hk];
          factor = slope_scale<T>(p.norm[number] * __int_as_float(peak) + fabsf(delta));
        }
      }
    }
    if (tiles > 0) {
      // the first half of the warpgroups brings the rows of Q, the other those of G
      constexpr int kHalf = F::kGroups / 256;
      const bool g = part_of >= kHalf;
      const long long at = g ? w.r * p.g_r + w.t * p.g_t + w.h * p.g_h : w.r * p.q_r + w.t * p.q_t + w.h * p.q_h;
      const char* row = mine ? (const char*)(g ? p.g : p.q) + at * 2 : nullptr;
      if (kHalf == 1)
        for (int piece = 0; piece < PIECES; ++piece)
          put_row<DP>(base + g * F::kRowsBytes + piece * F::kTileBytes, r, row ? row + piece * (g ? p.g_piece : p.q_piece) * 2 : row, p.W);
      else if (part_of & 1) put_row<DP>(base + g * F::kTileBytes, r, row, p.D, DP / 16, DP / 8);
      else put_row<DP>(base + g * F::kTileBytes, r, row, p.D, 0, DP / 16);
      fence_async_proxy();
      bar_arrive_warp(smem_at(&c.rows));
    }
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), minus = make_float2(-lse, -lse), less = make_float2(-delta, -delta);
    // With pieces, each tile's sums are added up in registers (half the columns a warpgroup): see the forward.
    float acc[PIECES == 1 ? 1 : 32] = {};
    const auto collect = [&]() {
      uint32_t v[32];
      tmem_load32(v, tmem + lanes + F::kSums + part_of * 32);
      tmem_wait_load();
#pragma unroll
      for (int e = 0; e < 32; ++e) acc[PIECES == 1 ? 0 : e] += __uint_as_float(v[e]);
    };
    for (int i = 0; i < tiles; ++i) {
      uint32_t bits = ~0u;
      if (MODE == kWindow) {
        const int at = first_of(i) + part_of * 32;
        if (at < own.lo || at + 32 > own.hi) bits = span_bits(own, at);
      } else if (MODE == kListed) {
        bits = c.bits[i].w[part_of];
      } else if (i + 1 == tiles && end % F::kStep) {
        const int left = end % F::kStep - part_of * 32;
        bits = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0;
      }
      bar_pass(smem_at(&c.scores), i & 1, lost);
      tc_fence_after();
      const int col = part_of * 32;
      uint32_t v[32], u[16], u1[PIECES == 1 && !kRest ? 1 : 16], u2[PIECES == 1 ? 1 : 16];
      tmem_load32(v, tmem + lanes + F::kScores + col);
      tmem_wait_load();
      tc_fence_before();
      bar_arrive_warp(smem_at(&c.taken));
      float2 wgt[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float2 x = fma2(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale2, minus);
        const float2 y = make_float2(exp2_fast(x.x), exp2_fast(x.y));
        wgt[e] = TcType<T>::code == 0 ? mul2(y, make_float2(factor, factor)) : y;
      }
      bar_pass(smem_at(&c.slopes), i & 1, lost);
      tc_fence_after();
      if constexpr (PIECES == 3) {
        if (i > 0) collect();  // (of the tile before: its product ended before this dP)
      }
      tmem_load32(v, tmem + lanes + F::kSlopes + col);
      tmem_wait_load();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float2 ds = mul2(wgt[e], add2(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), less));
        if (bits != ~0u) ds = make_float2((bits >> (2 * e)) & 1 ? ds.x : 0.0f, (bits >> (2 * e + 1)) & 1 ? ds.y : 0.0f);
        if constexpr (PIECES == 1) u[e] = pack2<T>(ds.x, ds.y);
        else pieces_of(ds, u[e], u1[e], u2[e]);
        if constexpr (kRest) {
          const float2 f = floats(*(const Two<T>*)&u[e]);
          u1[e] = pack2<T>(ds.x - f.x, ds.y - f.y);
        }
      }
      tmem_store16(tmem + lanes + F::kSlopes + col, u);
      if constexpr (kRest) tmem_store16(tmem + lanes + F::kSlopes + col + 16, u1);
      if constexpr (PIECES == 3) {
        tmem_store16(tmem + lanes + F::kSlopes + col + 16, u1);
        tmem_store16(tmem + lanes + F::kThird + col / 2, u2);
      }
      tmem_wait_store();
      tc_fence_before();
      bar_arrive_warp(smem_at(&c.grads));
    }
    if (tiles > 0) bar_pass(smem_at(&c.done), 0, lost);
    if (__all_sync(~0u, *lost == 0)) {
      tc_fence_after();
      const long long rows = (long long)p.R * p.T * p.Hq;
      float* part = p.splits > 1 ? p.part_gq + (split * rows + number) * p.D : nullptr;
      const float f = (part ? 1.0f : p.scale) / factor;
      const auto put = [&](int q, uint32_t (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
        if (mine) put_part<Out, PIECES>((Out*)p.gq + number * p.D + q * 32, part ? part + q * 32 : nullptr, v, p.D - q * 32);
      };
      if constexpr (PIECES == 3) {
        if (tiles > 0) collect();
        uint32_t v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(acc[i]);
        if (part_of * 32 < p.D) put(part_of, v);
      } else {
#pragma unroll 1
        for (int q = part_of; q < DP / 32; q += F::kGroups / 128) {
          if (q * 32 >= p.D) break;
          uint32_t v[32] = {};
          if (tiles > 0) {
            tmem_load32(v, tmem + lanes + F::kSums + q * 32);
            tmem_wait_load();
          }
          put(q, v);
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    if (*lost) {
      if (lane == 0) {
        if (status) atomicOr(status, 2);
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.done), 0) && nanoseconds() - t < kWaitLimit) {}
      }
      __syncwarp();
    }
    tc_fence_after();
    tmem_free(tmem, F::kColumns);
  }
}

// delta = g.o per row; for float16 |g| (2-norm) too, and the largest of both of a tile of rows (what is not finite bounds nothing), so that
// where states are kept a CTA looks at as many bounds as it has tiles of rows: looking at the rows themselves cost it 9 us of 150 in
// 128 x 49 rows of two images.  A CTA takes a tile, a row 4, 8 or 16 lanes.
constexpr int kDeltaThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kDeltaThreads) attn_tc_delta(const __grid_constant__ AttnParams p) {
  grid_dependency();
  RowTile o;
  if (!row_tile(p, blockIdx.x, kTcRows, o) || o.n >= p.N) return;
  __shared__ int peak[2];
  if (threadIdx.x < 2) peak[threadIdx.x] = 0;
  __syncthreads();
  const int hk = blockIdx.y, lane = threadIdx.x & 31, per = p.D / 8;  // a lane takes 8 elements of a row
  const int width = per <= 4 ? 4 : per <= 8 ? 8 : 16, piece = lane % width;
  float most = 0.0f, most_delta = 0.0f;
  for (int j = threadIdx.x / width; j < kTcRows && o.first + (j & ~(32 / width - 1)) < o.rows; j += kDeltaThreads / width) {
    const bool mine = o.first + j < o.rows;
    Row w = {};
    if (mine) w = row_of(p, o, o.first + j, hk);
    const long long row = row_number(p, w);
    float v = 0.0f, square = 0.0f;
    if (mine && piece < per) {
      const Vec<T, 8> g = *(const Vec<T, 8>*)((const T*)p.g + w.r * p.g_r + w.t * p.g_t + w.h * p.g_h + piece * 8);
      const Vec<T, 8> out = *(const Vec<T, 8>*)((const T*)p.o + row * p.D + piece * 8);
      Vec<__nv_bfloat16, 8> rest = {};
      if (p.rest) rest = *(const Vec<__nv_bfloat16, 8>*)(p.rest + row * p.D + piece * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = to_float(g.v[e]);
        v += a * (to_float(out.v[e]) + to_float(rest.v[e]));
        if (TcType<T>::code == 0) square += a * a;
      }
    }
    for (int d = width / 2; d; d >>= 1) {
      v += __shfl_xor_sync(~0u, v, d);
      if (TcType<T>::code == 0) square += __shfl_xor_sync(~0u, square, d);
    }
    if (mine && piece == 0) {
      p.delta[row] = v;
      if (TcType<T>::code == 0) {
        p.norm[row] = sqrtf(square);
        if (p.lse[row] != -INFINITY) {  // (it reads a state)
          most = fmaxf(most, finite_or_0(sqrtf(square)));
          most_delta = fmaxf(most_delta, finite_or_0(fabsf(v)));
        }
      }
    }
  }
  if constexpr (TcType<T>::code == 0) {
    if (piece == 0) {
      atomicMax(&peak[0], __float_as_int(most));
      atomicMax(&peak[1], __float_as_int(most_delta));
    }
    __syncthreads();
    if (threadIdx.x == 0) p.row_peaks[(long long)blockIdx.x * p.Hk + hk] = make_float2(__int_as_float(peak[0]), __int_as_float(peak[1]));
  }
}

}  // namespace mvr
