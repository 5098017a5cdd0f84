// Attention forward on the tensor cores (float16, bfloat16; head sizes that are multiples of 8, up to 128).
//
// A CTA holds TILES tiles of 128 rows of queries and walks the states of their image 64 or 128 at a time.  One warp brings tiles of
// keys and values into a ring in shared memory by TMA, one thread issues the products, and a warpgroup for every 64 columns of a
// tile, one row a thread, keeps the running maximum and sum:
//
//   S = Q K^T (128 x 64 or 128, tensor memory)  ->  P = 2^(S scale - m), rounded to T, over S  ->  O += P V (tensor memory)
//
// The maximum that P is formed about is only moved when it grows by more than 2^8, in float16 2^4: then O, in tensor memory, is scaled
// first.  float16 has few small numbers, so there P is 2^11 times as large: up to 2^15, and a weight is off by at most 2^-36 of the
// largest beside its relative rounding, which 2^21 states, the most of a call, bring to 2^-15.  (About 1 itself a weight below 2^-25
// would be 0, and 2^18 of them a percent of the result.)  The sum is formed of P before it is rounded; the factor is in both and
// goes out with the normaliser.  One CTA's chain of products, exponentials and products leaves
// every unit idle for a part of it.  Up to 64 columns of a head four CTAs share an SM, each with a tile of rows and 64 states at a
// time.  Beyond, two row tiles of one CTA alternate, which read every tile of states once for both, or, where rows are few, two CTAs
// with a tile each.  Few rows: the states are cut into parts as well (attn_join).
//
// Measured (tensor pipe, function units, issue slots busy): 2 x 4096 rows of 16 heads of 128 over 8192 states, bfloat16: 0.53 ms in a
// short run, 1.04 PFLOP/s (counters, in 0.56 ms: 49, 37, 41 %); 2 x 2048 rows of 16 heads of 64 (4 key heads) over 8191 and 6144:
// 0.23 ms, 0.53 PFLOP/s (26, 39, 45 %); one token of 32 heads of 128 (8 key heads) in each of 32 caches of 8448 to 16384 states:
// 0.27 ms, 6.0 TB/s.  None of the units is the limit of the first two: a step's chain (wait, fetch, maximum, exponentials, store) takes
// 2100 to 2500 cycles of a CTA, and tensor memory holds no more CTAs.  Of eight pairs of exponentials two as polynomials were best
// (none: 3 % slower, four: 6 %).
//
// States that are left out (lengths, mask) are compacted to a list of tiles, with a bit a state, before the walk; tiles without a state
// are not read.  Their scores are replaced, and their rows of V, which may hold NaN, are zeroed in shared memory by a warp of its
// own before the product reads them.
#pragma once
#include "mvr_attn.cuh"
#include "mvr_tc.cuh"

namespace mvr {

constexpr int kPolynomials = 2;  // of eight pairs of exponentials, how many are polynomials (halves: their error is below the rounding)

// P of the largest score (as a power of two), and how much further one may rise before the maximum is moved.
template <typename T> constexpr float kWeightShift = TcType<T>::code == 0 ? 11.0f : 0.0f;
template <typename T> constexpr float kLazy = TcType<T>::code == 0 ? 4.0f : 8.0f;

constexpr int kTcRows = 128, kTcBox = 64;   // rows of a tile; states of a TMA box
constexpr int kTcMaxStates = 32768;         // states that one CTA can list

// Which of STEP states may be read.
template <int STEP>
struct StateBits {
  uint32_t w[STEP / 32];
  __device__ __forceinline__ bool any() const {
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < STEP / 32; ++k) r |= w[k];
    return r != 0;
  }
  __device__ __forceinline__ bool all() const {
    uint32_t r = ~0u;
#pragma unroll
    for (int k = 0; k < STEP / 32; ++k) r &= w[k];
    return r == ~0u;
  }
};

template <int DP, int TILES, bool MASK, int PIECES>
struct TcForward {
  static_assert(PIECES == 1 || (DP == 64 && TILES == 1), "");
  static constexpr int kStep = TILES == 2 ? 128 : 64, kHalves = kStep / 64, kMaxTiles = kTcMaxStates / kStep;
  static constexpr int kBlocks = DP / 64, kTileBytes = kBlocks * kTcRows * 128, kStepBytes = kBlocks * kStep * 128;
  static constexpr int kRowsBytes = PIECES * kTileBytes, kSlotBytes = PIECES * kStepBytes;  // of a row tile and of a place of the ring
  static constexpr int kSlots = PIECES == 1 ? 4 : 2;
  static constexpr int kSoftmax = TILES * kHalves * 128, kThreads = kSoftmax + (TILES == 2 ? 96 : 64);
  // tensor memory: scores (P over them), third pieces of P, O
  static constexpr int kScores = 0, kThird = TILES * kStep, kOut = kThird + (PIECES == 1 ? 0 : 32);
  static constexpr int kColumns = TILES == 2 ? 512 : DP == 64 && PIECES == 1 ? 128 : 256;
  static constexpr int kResident = TILES == 2 ? 1 : DP == 64 && PIECES == 1 ? 4 : 2;
  struct Control {
    unsigned long long full[kSlots], empty[kSlots], clean[kSlots];
    unsigned long long queries[TILES], scores[TILES], weights[TILES], out[TILES], halves[TILES];
    uint32_t tmem;
    int lost, tiles, regions;
    int order[TILES == 1 ? kTcRows : 1];          // regions of the image, where the index is not grouped
    float top[kHalves == 2 ? 2 : 1][TILES][2][128];  // what the two halves of a row tell each other
    unsigned short list[MASK ? kMaxTiles : 1];
    StateBits<kStep> bits[MASK ? kMaxTiles : 1];
  };
  static constexpr size_t kShared = TILES * (size_t)kRowsBytes + kSlots * (size_t)kSlotBytes + sizeof(Control) + 1024;
};

struct TcMaps {
  CUtensorMap k, v;  // (D, heads, states, images; pieces one behind another)
  CUtensorMap q, g;  // (D, heads, tokens, regions): set where tiles of rows are boxes of the queries and their gradient
};

// List of the tiles of STEP states in [begin, end) that have one to read, with their bits.  All threads; the result after a barrier.
template <int STEP>
__device__ __forceinline__ void list_tiles(const AttnParams& p, int n, int begin, int end, unsigned short* list, StateBits<STEP>* bits,
                                           int* count) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, tiles = (end - begin + STEP - 1) / STEP;
  for (int i = threadIdx.x >> 5; i < tiles; i += warps) {
    StateBits<STEP> b;
#pragma unroll
    for (int k = 0; k < STEP / 32; ++k) {
      const int j = begin + i * STEP + k * 32 + lane;
      b.w[k] = __ballot_sync(~0u, j < end && (!p.mask || p.mask[(long long)n * p.L + j] != 0));
    }
    if (lane == 0) bits[i] = b;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int at = 0;
    for (int base = 0; base < tiles; base += 32) {
      const int i = base + lane;
      StateBits<STEP> b = {};
      if (i < tiles) b = bits[i];
      const bool any = b.any();
      const uint32_t who = __ballot_sync(~0u, any);
      __syncwarp();
      if (any) {  // (at + rank <= i: what is overwritten has been read)
        const int to = at + __popc(who & ((1u << lane) - 1));
        list[to] = (unsigned short)i;
        bits[to] = b;
      }
      at += __popc(who);
      __syncwarp();
    }
    if (lane == 0) *count = at;
  }
}

// Rows of states that are left out become 0 in a tile of STEP rows in shared memory.  One warp, a row a lane (row by row, eight lanes a
// row, took longer than the products of a half-masked tile).
template <int STEP, int BLOCKS>
__device__ __forceinline__ void clear_rows(char* tile, const StateBits<STEP>& b, int lane) {
  if (b.all()) return;
#pragma unroll
  for (int w = 0; w < STEP / 32; ++w) {
    if ((b.w[w] >> lane) & 1) continue;
    char* row = tile + (w * 32 + lane) * 128;
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
      for (int c = 0; c < 8; ++c) *(uint4*)(row + k * (STEP * 128) + (((c + lane) & 7) << 4)) = make_uint4(0, 0, 0, 0);
  }
  fence_async_proxy();
  __syncwarp();
}

// A row of 2-byte elements into a K-major tile in the 128-byte swizzle; zeros behind D, and for no row at all.
template <int DP>
__device__ __forceinline__ void put_row(char* tile, int r, const void* src, int D, int first = 0, int last = DP / 8) {
#pragma unroll
  for (int c = first; c < last; ++c) {
    const uint4 v = src && c * 8 < D ? ((const uint4*)src)[c] : make_uint4(0, 0, 0, 0);
    *(uint4*)(tile + (c >> 3) * (kTcRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
}

// `left` floats of 32 to a row; sixteen bytes at a time where every row starts at a multiple of them.
template <int PIECES>
__device__ __forceinline__ void put_floats(float* to, const uint32_t (&v)[32], int left) {
  if (PIECES == 1 || ((uintptr_t)to & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if (i + 4 <= left) {
        *(uint4*)(to + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < left) to[i + e] = __uint_as_float(v[i + e]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < left) to[i] = __uint_as_float(v[i]);
  }
}

// PIECES 3: float tensors, whose operands lie in pieces (T is bfloat16).
template <typename T, int DP, int TILES, bool MASK, int PIECES>
__global__ void __launch_bounds__(TcForward<DP, TILES, MASK, PIECES>::kThreads, TcForward<DP, TILES, MASK, PIECES>::kResident)
attn_tc_fwd(const __grid_constant__ AttnParams p, const __grid_constant__ TcMaps maps, int* status) {
  typedef TcForward<DP, TILES, MASK, PIECES> F;
  extern __shared__ char tc_smem[];
  char* base = tc_smem + ((1024 - (smem_at(tc_smem) & 1023)) & 1023);
  char* ring = base + TILES * F::kRowsBytes;
  typename F::Control& c = *(typename F::Control*)(ring + F::kSlots * F::kSlotBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kLoader = F::kSoftmax / 32, kIssuer = kLoader + 1, kCleaner = kLoader + 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::kSlots; ++i) {
      bar_init(smem_at(&c.full[i]), 1);
      bar_init(smem_at(&c.empty[i]), 1);
      bar_init(smem_at(&c.clean[i]), 1);
    }
    for (int t = 0; t < TILES; ++t) {
      bar_init(smem_at(&c.queries[t]), 4 * F::kHalves);
      bar_init(smem_at(&c.scores[t]), 1);
      bar_init(smem_at(&c.weights[t]), 4 * F::kHalves);
      bar_init(smem_at(&c.halves[t]), 8);
      bar_init(smem_at(&c.out[t]), 1);
    }
    c.lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Tensor memory is taken only when the kernel before has ended, and the next kernel may come only when it has been taken: no CTA
  // holds it while it waits for another that still needs some.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == kIssuer) tmem_alloc(smem_at(&c.tmem), F::kColumns);
  RowTile o;
  const int hk = blockIdx.y, split = blockIdx.z;
  bool some;
  if (TILES == 1 && p.index) {
    // few regions: the CTA looks for those of its image itself, which is faster than a kernel that groups them
    const int n = blockIdx.x;
    if (warp == 0) {
      int at = 0;
      for (int r0 = 0; r0 < p.R; r0 += 32) {
        const bool mine = r0 + lane < p.R && image_index(p.index, p.index_type, p.index_stride, r0 + lane, p.N) == n;
        const uint32_t who = __ballot_sync(~0u, mine);
        if (mine) c.order[at + __popc(who & ((1u << lane) - 1))] = r0 + lane;
        at += __popc(who);
      }
      if (lane == 0) {
        c.regions = at;
        if (n == p.N && at > 0 && hk == 0 && split == 0 && status) atomicOr(status, 1);
      }
    }
    __syncthreads();
    o = {n, 0, c.regions * p.T * p.G, c.order};
    some = o.rows > 0;
  } else {
    some = row_tile(p, blockIdx.x, TILES * kTcRows, o);
  }
  const int all = (p.L + F::kStep - 1) / F::kStep, per = (all + p.splits - 1) / p.splits;
  const int begin = split * per * F::kStep;
  int end = 0;
  if (some) end = min(states_of(p, o.n), (split + 1) * per * F::kStep);
  if (MASK && some && begin < end) list_tiles(p, o.n, begin, end, c.list, c.bits, &c.tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tiles = !some || begin >= end ? 0 : MASK ? c.tiles : (end - begin + F::kStep - 1) / F::kStep;
  const int used = !some ? 0 : TILES == 2 && o.first + kTcRows < o.rows ? 2 : 1;  // row tiles that have rows
  const uint32_t tmem = c.tmem;
  volatile int* lost = &c.lost;
  const auto first_of = [&](int i) { return begin + (MASK ? (int)c.list[i] : i) * F::kStep; };

  const auto clean = [&](int tile, int slot) {
    for (int piece = 0; piece < PIECES; ++piece)
      clear_rows<F::kStep, F::kBlocks>(ring + slot * F::kSlotBytes + piece * F::kStepBytes, c.bits[MASK ? tile : 0], lane);
    if (lane == 0) bar_arrive(smem_at(&c.clean[slot]));
  };

  if (warp == kLoader) {
    constexpr int kBehind = F::kSlots == 4 ? 2 : 0;
    const auto clean_values = [&](int item) {
      bar_pass(smem_at(&c.full[item % F::kSlots]), (item / F::kSlots) & 1, lost);
      clean(item >> 1, item % F::kSlots);
    };
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
      // One row tile: registers go further with six warps a CTA, so this one clears rows of V as well, a tile behind where the ring
      // holds two.
      if (MASK && TILES == 1 && (i & 1) && i >= kBehind) clean_values(i - kBehind);
    }
    if (MASK && TILES == 1 && kBehind > 0 && i == 2 * tiles && tiles > 0) clean_values(i - 1);
    // given up: the copies under way end before the CTA does
    if (*lost)
      for (int k = max(0, i - F::kSlots); k < i; ++k) {
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.full[k % F::kSlots]), (k / F::kSlots) & 1) && nanoseconds() - t < kWaitLimit) {}
      }
  } else if (warp == kIssuer) {
    if (tiles > 0) {
      const int depth = (p.D + 15) / 16;
      const uint32_t s_shape = tc_shape<T>(F::kStep, false, p.scale < 0.0f), o_shape = tc_shape<T>(depth * 16, true);
      const uint64_t queries = desc_k_major(smem_at(base)), keys = desc_k_major(smem_at(ring)), values = desc_mn_major(smem_at(ring), F::kStep * 128);
      const auto multiply = [&](int t, int slot) {
        for_pairs<PIECES>([&](int a, int b, bool first) {
          mma_rows<DP / 16>(tmem + F::kScores + t * F::kStep, queries + ((t * F::kRowsBytes + a * F::kTileBytes) >> 4),
                            keys + ((slot * F::kSlotBytes + b * F::kStepBytes) >> 4), s_shape, depth, kTcRows * 128, F::kStep * 128, !first);
        });
      };
      const auto scores = [&](int t, int slot) {  // S_t = Q_t K^T
        if (elect_one()) {
          multiply(t, slot);
          mma_commit(smem_at(&c.scores[t]));
        }
        __syncwarp();
      };
      const auto commit = [&](unsigned long long* bar) {
        if (elect_one()) mma_commit(smem_at(bar));
        __syncwarp();
      };
      for (int t = 0; t < used; ++t) bar_pass(smem_at(&c.queries[t]), 0, lost);
      bar_pass(smem_at(&c.full[0]), 0, lost);
      tc_fence_after();
      for (int t = 0; t < used; ++t) scores(t, 0);
      commit(&c.empty[0]);
      for (int j = 0; j < tiles; ++j) {
        const int v = 2 * j + 1, k = v + 1, vs = v % F::kSlots, ks = k % F::kSlots;
        bar_pass(smem_at(&c.full[vs]), (v / F::kSlots) & 1, lost);
        if (MASK) bar_pass(smem_at(&c.clean[vs]), (v / F::kSlots) & 1, lost);
        if (j + 1 < tiles) bar_pass(smem_at(&c.full[ks]), (k / F::kSlots) & 1, lost);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if (t >= used) break;
          bar_pass(smem_at(&c.weights[t]), j & 1, lost);
          tc_fence_after();
          if (elect_one()) {
            for_pairs<PIECES>([&](int a, int b, bool first) {
#pragma unroll
              for (int i = 0; i < F::kStep / 16; ++i) {  // O_t += P_t V
                const int at = PIECES == 1 ? t * F::kStep + (i >> 2) * 64 + (i & 3) * 8
                                           : a == 2 ? F::kThird + i * 8 : (i >> 1) * 32 + a * 16 + (i & 1) * 8;
                mma_ts(tmem + F::kOut + t * DP, tmem + F::kScores + at, values + ((vs * F::kSlotBytes + b * F::kStepBytes + i * 2048) >> 4), o_shape,
                       (PIECES == 1 && j > 0) || i > 0 || !first);
              }
            });
            if (j + 1 < tiles) {
              multiply(t, ks);
              mma_commit(smem_at(&c.scores[t]));
            }
            if (t + 1 == used) {
              mma_commit(smem_at(&c.empty[vs]));
              if (j + 1 < tiles) mma_commit(smem_at(&c.empty[ks]));
            }
          }
          __syncwarp();
        }
      }
      for (int t = 0; t < TILES; ++t) commit(&c.out[t]);
    }
  } else if (MASK && TILES == 2 && warp == kCleaner) {
    for (int j = 0; j < tiles; ++j) {
      const int v = 2 * j + 1, slot = v % F::kSlots;
      if (!bar_wait(smem_at(&c.full[slot]), (v / F::kSlots) & 1, lost)) break;
      clean(j, slot);
    }
  } else if (warp < kLoader) {
    const int t = warp / (4 * F::kHalves), half = F::kHalves == 2 ? (warp >> 2) & 1 : 0, r = threadIdx.x & 127, j0 = o.first + t * kTcRows + r;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21, s_at = tmem + lanes + F::kScores + t * F::kStep + half * 64, o_at = tmem + lanes + F::kOut + t * DP;
    if (t < used) {
      Row w = {};
      const bool mine = j0 < o.rows;
      if (mine) w = row_of(p, o, j0, hk);
      if (tiles > 0) {
        const char* q = mine ? (const char*)p.q + (w.r * p.q_r + w.t * p.q_t + w.h * p.q_h) * 2 : nullptr;
        if (F::kHalves == 1)
          for (int piece = 0; piece < PIECES; ++piece) put_row<DP>(base + piece * F::kTileBytes, r, q ? q + piece * p.q_piece * 2 : q, p.W);
        else if (half) put_row<DP>(base + t * F::kTileBytes, r, q, p.D, DP / 16, DP / 8);
        else put_row<DP>(base + t * F::kTileBytes, r, q, p.D, 0, DP / 16);
        fence_async_proxy();
        bar_arrive_warp(smem_at(&c.queries[t]));
      }
      const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);  // (not 0: a score that is left out is -inf)
      float m = -INFINITY, l = 0.0f;  // m: in the units of S, the same in both halves; l: of this half
      const auto reference = [&](float m) { return m == -INFINITY ? 0.0f : fmaf(m, scale, -kWeightShift<T>); };  // P = 2^(S scale - this)
      // With pieces, O of each tile is added up in registers: the tensor cores' additions cut off what they do not hold, which over a
      // hundred tiles comes to some 4e-6, five times the error of float sums.
      float acc[PIECES == 1 ? 1 : 64] = {};
      const auto collect = [&]() {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t v[32];
          tmem_load32(v, o_at + q * 32);
          tmem_wait_load();
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[PIECES == 1 ? 0 : q * 32 + i] += __uint_as_float(v[i]);
        }
      };
      // A warp without a row only keeps step: what lies in its rows of P reaches no other row of O.  (A single token leaves three
      // warps of four idle.)
      if (F::kHalves == 1 && !__any_sync(~0u, mine)) {
        for (int j = 0; j < tiles; ++j) {
          bar_pass(smem_at(&c.scores[t]), j & 1, lost);
          bar_arrive_warp(smem_at(&c.weights[t]));
        }
      } else {
      for (int j = 0; j < tiles; ++j) {
        uint32_t bits[2] = {~0u, ~0u};
        if (MASK) {
          bits[0] = c.bits[j].w[half * 2];
          bits[1] = c.bits[j].w[half * 2 + 1];
        } else if (j + 1 == tiles && end % F::kStep) {
          const int left = end % F::kStep - half * 64;
          bits[0] = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0;
          bits[1] = left >= 64 ? ~0u : left > 32 ? (1u << (left - 32)) - 1 : 0;
        }
        bar_pass(smem_at(&c.scores[t]), j & 1, lost);
        tc_fence_after();
        if constexpr (PIECES == 3) {
          if (j > 0) collect();  // (of the tile before: its product ended before these scores)
        }
        // scores of 32 states, those that are left out as -inf
        const auto settle = [&](uint32_t (&v)[32], int q) {
          if (bits[q] != ~0u) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = (bits[q] >> i) & 1 ? v[i] : __float_as_uint(-INFINITY);
          }
        };
        const auto most = [&](const uint32_t (&v)[32]) {  // of 32 scores; two chains
          float a = -INFINITY, c = __uint_as_float(v[0]);
#pragma unroll
          for (int i = 1; i < 29; i += 4) {
            a = max3(a, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
            c = max3(c, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
          }
          a = max3(a, __uint_as_float(v[29]), __uint_as_float(v[30]));
          return max3(a, c, __uint_as_float(v[31]));
        };
        // (fetched twice: keeping them costs more registers than a thread has)
        uint32_t x[32];
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          tmem_load32(x, s_at + q * 32);
          tmem_wait_load();
          settle(x, q);
          top = max3(top, most(x), top);
        }
        // the row's maximum, of both halves
        if constexpr (F::kHalves == 2) {
          c.top[j & 1][t][half][r] = top;
          bar_arrive_warp(smem_at(&c.halves[t]));
          bar_pass(smem_at(&c.halves[t]), j & 1, lost);
          top = max3(top, c.top[j & 1][t][half ^ 1][r], top);
        }
        if (top == INFINITY) top = NAN;  // (as inf - inf is; the sums are NaN from here on)
        // move the maximum?  (the first tile: there is no O yet)
        const bool move = !(top <= m) && (m == -INFINITY || !((top - m) * scale <= kLazy<T>));  // (NaN moves it)
        if (__any_sync(~0u, move)) {
          const float shrink = move ? (m == -INFINITY ? 0.0f : exp2_fast((m - top) * scale)) : 1.0f;
          if (move) m = top;
          l *= shrink;
          if constexpr (PIECES == 3) {
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] *= shrink;
          } else if (j > 0) {
#pragma unroll 1
            for (int q = half; q < DP / 32; q += F::kHalves) {
              uint32_t v[32];
              tmem_load32(v, o_at + q * 32);
              tmem_wait_load();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * shrink);
              tmem_store32(o_at + q * 32, v);
            }
          }
        }
        const float ref = reference(m);
        const float2 scale2 = make_float2(scale, scale), minus = make_float2(-ref, -ref);
        float2 sums[2] = {};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          tmem_load32(x, s_at + q * 32);
          tmem_wait_load();
          settle(x, q);
          uint32_t v[16], v1[PIECES == 1 ? 1 : 16], v2[PIECES == 1 ? 1 : 16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 a = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, minus);
            const float2 e = PIECES == 1 && i % 8 < kPolynomials ? exp2_polynomial(a) : make_float2(exp2_fast(a.x), exp2_fast(a.y));
            sums[i & 1] = add2(sums[i & 1], e);
            if constexpr (PIECES == 1) v[i] = pack2<T>(e.x, e.y);
            else pieces_of(e, v[i], v1[i], v2[i]);
          }
          // (over this half's own scores; with pieces, over the 32 that have just been read)
          if constexpr (PIECES == 1) {
            tmem_store16(s_at + q * 16, v);
          } else {
            tmem_store16(s_at + q * 32, v);
            tmem_store16(s_at + q * 32 + 16, v1);
            tmem_store16(tmem + lanes + F::kThird + q * 16, v2);
          }
        }
        const float2 sum = add2(sums[0], sums[1]);
        l += sum.x + sum.y;
        tmem_wait_store();
        tc_fence_before();
        bar_arrive_warp(smem_at(&c.weights[t]));
      }
      }
      // the halves' sums together (a + b is b + a: the same in both)
      if constexpr (F::kHalves == 2) {
        c.top[tiles & 1][t][half][r] = l;
        bar_arrive_warp(smem_at(&c.halves[t]));
        bar_pass(smem_at(&c.halves[t]), tiles & 1, lost);
        l += c.top[tiles & 1][t][half ^ 1][r];
      }
      if (tiles > 0) bar_pass(smem_at(&c.out[t]), 0, lost);
      if (__all_sync(~0u, *lost == 0)) {
        tc_fence_after();
        if constexpr (PIECES == 3) {
          if (tiles > 0) collect();
        }
        const long long row = row_number(p, w), rows = (long long)p.R * p.T * p.Hq;
        if (m == -INFINITY) l = 0.0f;  // no state, or only scores of -inf
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (mine && !half) {
          if (p.splits > 1) {
            p.part_ml[(split * rows + row) * 2] = m == -INFINITY ? m : reference(m);
            p.part_ml[(split * rows + row) * 2 + 1] = l;
          } else if (p.lse) {
            p.lse[row] = l == 0.0f ? -INFINITY : reference(m) + log2f(l);
          }
        }
        const auto put = [&](int q, uint32_t (&v)[32]) {
          if (mine && (p.splits > 1 || PIECES == 3)) {
            float* to = (p.splits > 1 ? p.part_o + (split * rows + row) * p.D : (float*)p.out + row * p.D) + q * 32;
            const float f = p.splits > 1 ? 1.0f : inv;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            put_floats<PIECES>(to, v, p.D - q * 32);
          } else if (mine) {
            T* to = (T*)p.out + row * p.D + q * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (q * 32 + i >= p.D) continue;
              uint32_t u[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                u[e] = pack2<T>(__uint_as_float(v[i + 2 * e]) * inv, __uint_as_float(v[i + 2 * e + 1]) * inv);
              *(uint4*)(to + i) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        };
        if constexpr (PIECES == 3) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(acc[q * 32 + i]);
            if (q * 32 < p.D) put(q, v);
          }
        } else {
#pragma unroll 1
          for (int q = half; q < DP / 32; q += F::kHalves) {
            if (q * 32 >= p.D) break;
            uint32_t v[32] = {};
            if (tiles > 0) {
              tmem_load32(v, o_at + q * 32);
              tmem_wait_load();
            }
            put(q, v);
            __syncwarp();
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    if (*lost) {  // products may still be under way: they end before tensor memory is freed
      if (lane == 0) {
        if (status) atomicOr(status, 2);
        const unsigned long long t = nanoseconds();
        while (!bar_try(smem_at(&c.out[0]), 0) && nanoseconds() - t < kWaitLimit) {}
      }
      __syncwarp();
    }
    tc_fence_after();
    tmem_free(tmem, F::kColumns);
  }
}

}  // namespace mvr
