// Group norm with its activation over channels-last tensors (N, S, C), groups of consecutive channels:
//   xhat = (x - mean) rstd    z = xhat w + b    y = act(z)            mean, variance of an image's group: S * C / groups values
//   dz = dy act'(z)    db = sum dz    dw = sum dz xhat    dx = rstd (dz w - m1 - xhat m2)    m1, m2: the group's means of dz w, dz w xhat
//
// A CTA takes a block of whole groups and a chunk of an image's rows, a thread one vector of channels of every `depth`th row, so that what
// belongs to a channel stays in registers.  Two ways:
//   passes    one kernel for the chunks' sums per group, one that joins an image's chunks and walks the rows again, backwards: what was
//             read last is the likeliest still in L2.  All CTAs run at once, so that a chunk is as long as the work allows and its sums
//             are few (296 of an SM's two; some 38 KB that every CTA of the second kernel reads)
//   clusters  where the rows of a block fit the shared memory of one to eight CTAs: these tell each other their sums and walk the rows a
//             second time where they lie
// No atomics: each sum has one place and one order.
//
// Measured, bfloat16 rows of 32 channels, groups of 4, silu, 2 x 128^3 rows (268 MB): moments 52 us (5.1 TB/s), elements 106 (5.0), slopes' sums
// 119 (4.5), dx 152 (5.3); of a copy's rate 70 to 80 %, issue slots 40 % busy and the function units 43 to 64: what is left is a thread's
// chain of loads, exponentials and stores at 24 warps an SM (loads a step ahead do not fit the registers backward).  The second read comes
// from memory: 63 MB of L2 are near an SM, and all chunks are walked at once.  2 x 48^3 rows of 64 halves: 20 us forward, 38 backward.
// 2 x 512 rows of 256 halves by clusters 4.8 us, in passes 7.3.
//
// Statistics.  A thread sums x - k and (x - k)^2 about its own first value k of a channel, over its r rows.  If k lies far from the others,
// the thread's sum of squares about its mean is itself at least (r - 1) / r of that distance's square, so that cancellation costs no
// more than some r of its last bits, whatever the data's offset; the same holds where a thread joins threads or chunks about the first
// one's mean.  Channels, threads and chunks are joined by their means' differences, for
// which a mean is kept as two floats: rounded to one, means near 1e5 of values with a deviation of 2 put an error of 1e-4 into their variance,
// and 2e-3 into every xhat of a group.  What a mean's rounding left is taken out of a channel's bias, of its sum of dz xhat and of dx's constant
// part, so that it costs no value an operation.
#pragma once
#include "mvr_types.cuh"

namespace mvr {

enum { kNoActivation = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// Mean, as a float and what its rounding left, sum of squares about it, and of how many values.
struct alignas(16) Moments {
  float mean, rest, square, count;
};

struct NormParams {
  const void *x, *dy, *weight, *bias;  // (N, S, C) twice; (C), or null: 1 and 0
  void *out, *dx, *dweight, *dbias;
  float *mean, *rstd, *rest;           // (N, groups); rest: what the mean's rounding left, or null
  Moments* moments;                    // (N, chunks, groups): forward
  float2 *sums, *slopes;               // (N, chunks, groups): sums of dz w, dz w xhat; (N, chunks, C): of dz, dz xhat
  long long S, rows;                   // rows of a chunk, or of a CTA of a cluster
  int N, C, groups, width;             // width: channels of a group
  int parameters;                      // type of weight and bias: 0 float, 1 half, 3 bfloat16
  int chunks;                          // of an image; or CTAs of a cluster
  int blocks, block_groups, columns;   // of an image; groups and vectors of a block
  int lanes, depth;                    // a CTA takes `lanes` vectors of `depth` rows at a time (clusters, nearly always: all of a block)
  Divisor by_width;
  int channel_ctas;                    // dx: the first CTAs sum the gradients of weights and biases
  float eps;
};

constexpr int kNormThreads = 384;

__device__ __forceinline__ float parameter(const NormParams& p, const void* from, int c) {
  return p.parameters == 0 ? ((const float*)from)[c] : p.parameters == 1 ? to_float(((const __half*)from)[c]) : to_float(((const __nv_bfloat16*)from)[c]);
}
// V neighbouring ones, all under way together.
template <typename PT, int V>
__device__ __forceinline__ void load_parameters(float (&to)[V], const void* from, int c) {
  PT v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = ((const PT*)from)[c + k];
#pragma unroll
  for (int k = 0; k < V; ++k) to[k] = to_float(v[k]);
}
template <int V>
__device__ __forceinline__ void parameters_of(const NormParams& p, float (&weight)[V], float (&bias)[V], int c) {
#pragma unroll
  for (int k = 0; k < V; ++k) weight[k] = 1.0f, bias[k] = 0.0f;
  if (p.parameters == 0) {
    if (p.weight) load_parameters<float>(weight, p.weight, c);
    if (p.bias) load_parameters<float>(bias, p.bias, c);
  } else if (p.parameters == 1) {
    if (p.weight) load_parameters<__half>(weight, p.weight, c);
    if (p.bias) load_parameters<__half>(bias, p.bias, c);
  } else {
    if (p.weight) load_parameters<__nv_bfloat16>(weight, p.weight, c);
    if (p.bias) load_parameters<__nv_bfloat16>(bias, p.bias, c);
  }
}
__device__ __forceinline__ float weight_of(const NormParams& p, int c) { return p.weight ? parameter(p, p.weight, c) : 1.0f; }
__device__ __forceinline__ void put_parameter(const NormParams& p, void* to, int c, float v) {
  if (p.parameters == 0) ((float*)to)[c] = v;
  else if (p.parameters == 1) ((__half*)to)[c] = from_float<__half>(v);
  else ((__nv_bfloat16*)to)[c] = from_float<__nv_bfloat16>(v);
}

// ---- pairs of values ----------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(z), and act'(z).  Half types: exponentials and inverses by the function units (2^-20 of the result up to |z| = 10), the normal
// distribution by formula 7.1.26 of Abramowitz and Stegun (1.5e-7), which shares its exponential with the slope.
template <typename T, int ACT>
__device__ __forceinline__ float2 activate(float2 z, float2& slope) {
  constexpr bool kExact = sizeof(T) == 4;
  if constexpr (ACT == kRelu) {
    slope = make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
    return make_float2(z.x > 0.0f || z.x != z.x ? z.x : 0.0f, z.y > 0.0f || z.y != z.y ? z.y : 0.0f);
  } else if constexpr (ACT == kSilu) {
    float2 gate;
    if constexpr (kExact) {
      gate = make_float2(1.0f / (1.0f + expf(-z.x)), 1.0f / (1.0f + expf(-z.y)));
    } else {
      const float2 t = mul2(z, two(-1.4426950408889634f)), d = add2(make_float2(exp2_of(t.x), exp2_of(t.y)), two(1.0f));
      gate = make_float2(inverse_of(d.x), inverse_of(d.y));
    }
    const float2 y = mul2(z, gate);
    slope = fma2(y, fma2(gate, two(-1.0f), two(1.0f)), gate);
    return y;
  } else if constexpr (ACT == kGelu) {
    float2 gate, bell;  // distribution and density times sqrt(2 pi)
    if constexpr (kExact) {
      gate = make_float2(normcdff(z.x), normcdff(z.y));
      bell = make_float2(expf(-0.5f * z.x * z.x), expf(-0.5f * z.y * z.y));
    } else {
      const float2 square = mul2(mul2(z, z), two(-0.7213475204444817f)), d = fma2(make_float2(fabsf(z.x), fabsf(z.y)), two(0.3275911f * 0.7071067811865476f), two(1.0f));
      bell = make_float2(exp2_of(square.x), exp2_of(square.y));
      const float2 t = make_float2(inverse_of(d.x), inverse_of(d.y));
      float2 s = fma2(t, two(0.5f * 1.061405429f), two(0.5f * -1.453152027f));
      s = fma2(s, t, two(0.5f * 1.421413741f));
      s = fma2(s, t, two(0.5f * -0.284496736f));
      s = fma2(s, t, two(0.5f * 0.254829592f));
      s = mul2(mul2(s, t), bell);  // the part beyond |z|
      gate = make_float2(z.x < 0.0f ? s.x : 1.0f - s.x, z.y < 0.0f ? s.y : 1.0f - s.y);
    }
    slope = fma2(mul2(z, two(0.3989422804014327f)), bell, gate);
    return mul2(z, gate);
  } else {
    slope = two(1.0f);
    return z;
  }
}

// load(i) and then use(i, what it gave) for i < count, U loads under way together (a store between them would hold the next one up).
template <int U, typename L, typename F>
__device__ __forceinline__ void walk(int count, L&& load, F&& use) {
  for (int i = 0; i < count; i += U) {
    decltype(load(0)) v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < count) v[u] = load(i + u);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < count) use(i + u, v[u]);
  }
}

// ---- who takes what -----------------------------------------------------------------------------------
struct NormPlace {
  int n, chunk, block, lane, depth;
  int group;                   // first group of the block
  long long begin, end, row;   // of the chunk; the thread's first row
  int count;                   // of its rows
};
__device__ __forceinline__ NormPlace norm_place(const NormParams& p, int n, int block, int chunk) {
  NormPlace t;
  t.n = n;
  t.block = block;
  t.chunk = chunk;
  t.group = block * p.block_groups;
  t.depth = threadIdx.x / p.lanes;
  t.lane = threadIdx.x - t.depth * p.lanes;
  t.begin = chunk * p.rows;
  t.end = max(t.begin, min(p.S, t.begin + p.rows));
  t.row = t.begin + t.depth;
  t.count = t.depth < p.depth && t.row < t.end ? (int)((t.end - t.row + p.depth - 1) / p.depth) : 0;
  return t;
}
__device__ __forceinline__ NormPlace norm_place(const NormParams& p, int cta) {  // (passes)
  const int image = cta / p.blocks, n = image / p.chunks;
  return norm_place(p, n, cta - image * p.blocks, image - n * p.chunks);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* mine, int rank) {  // the same place in another CTA of the cluster
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  return at;
}
__device__ __forceinline__ Moments of_cluster(const Moments* mine, int rank) {
  Moments v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.mean), "=f"(v.rest), "=f"(v.square), "=f"(v.count) : "r"(at_rank(mine, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 of_cluster(const float2* mine, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at_rank(mine, rank)) : "memory");
  return v;
}

// A team of neighbouring threads, at most a warp, for every group of a block.
struct NormTeam {
  int size, lane, first, teams;
  __device__ __forceinline__ NormTeam(int groups, int entries) {  // (of a group)
    size = 32;
    while (size > 1 && (kNormThreads / size < groups || size >= 2 * entries)) size >>= 1;
    lane = threadIdx.x & (size - 1);
    first = threadIdx.x / size;
    teams = kNormThreads / size;
  }
  __device__ __forceinline__ float sum(float v) const {  // (all threads of a warp)
    for (int d = size >> 1; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
  }
  // f(g, there) for every group; all threads call it alike often
  template <typename F>
  __device__ __forceinline__ void each(int groups, F&& f) const {
    for (int g = first; g - first < groups; g += teams) f(g < groups ? g : groups - 1, g < groups);
  }
};

// ---- moments ------------------------------------------------------------------------------------------
__device__ __forceinline__ Moments moments_of(float a, float b, float square, float count) {  // mean: a + b
  const float mean = a + b, of_b = mean - a;
  return {mean, (a - (mean - of_b)) + (b - of_b), square, count};
}
__device__ __forceinline__ float distance(const Moments& a, const Moments& b) { return (a.mean - b.mean) + (a.rest - b.rest); }

// (an empty `a` only with an empty `b`: rows are dealt out from the first thread, CTA and chunk on)
__device__ __forceinline__ Moments joined(const Moments& a, const Moments& b) {
  const float count = a.count + b.count, d = distance(b, a), shift = d * b.count * inverse_of(fmaxf(count, 1.0f));
  return moments_of(a.mean, a.rest + shift, fmaf(shift * d, a.count, a.square + b.square), count);
}
__device__ __forceinline__ float2 joined(float2 a, float2 b) { return add2(a, b); }

// (rows, columns) of shared memory joined down to the first row, by halves.  All threads, behind a barrier; ends in one.
template <typename E>
__device__ __forceinline__ void join_rows(E* at, int rows, int columns) {
  while (rows > 1) {
    const int half = (rows + 1) >> 1;
    for (int i = threadIdx.x; i < (rows - half) * columns; i += kNormThreads) at[i] = joined(at[i], at[half * columns + i]);
    __syncthreads();
    rows = half;
  }
}

// Entries in a row, n of them, by a team; in its first thread.
__device__ __forceinline__ Moments team_join(const NormTeam& team, const Moments* from, int n) {
  Moments m = {};
  if (team.lane < n) m = from[team.lane];
  for (int i = team.lane + team.size; i < n; i += team.size) m = joined(m, from[i]);
  for (int d = 1; d < team.size; d <<= 1) {  // (neighbours first: a thread without an entry is behind those with one)
    const Moments other = {__shfl_down_sync(~0u, m.mean, d), __shfl_down_sync(~0u, m.rest, d), __shfl_down_sync(~0u, m.square, d), __shfl_down_sync(~0u, m.count, d)};
    if (team.lane + d < team.size) m = joined(m, other);
  }
  return m;
}

// A sum of squares about a mean, whose rounding may have left it below 0; NaN (of values that are not finite) stays.
__device__ __forceinline__ float not_negative(float square) { return square < 0.0f ? 0.0f : square; }

// A thread's sums about a pivot, of a vector of channels.
template <typename T, int V>
struct NormMoments {
  typedef FloatPairs<T, V> P;
  P pivot, sum, square;
  __device__ __forceinline__ void start(const Vec<T, V>& v) {
    pivot = P(v);
#pragma unroll
    for (int k = 0; k < P::kPairs; ++k) sum.v[k] = square.v[k] = two(0.0f);
  }
  __device__ __forceinline__ void add(const Vec<T, V>& v) {
    const P x(v);
#pragma unroll
    for (int k = 0; k < P::kPairs; ++k) {
      const float2 d = fma2(pivot.v[k], two(-1.0f), x.v[k]);
      sum.v[k] = add2(sum.v[k], d);
      square.v[k] = fma2(d, d, square.v[k]);
    }
  }
  __device__ __forceinline__ Moments of(int k, float count, float inverse) const {
    const float s = k & 1 ? sum.v[k >> 1].y : sum.v[k >> 1].x, q = k & 1 ? square.v[k >> 1].y : square.v[k >> 1].x,
                c = k & 1 ? pivot.v[k >> 1].y : pivot.v[k >> 1].x, mean = s * inverse;
    return moments_of(c, mean, not_negative(fmaf(-mean, s, q)), count);
  }
  // SPAN neighbouring channels from k on, together
  template <int SPAN>
  __device__ __forceinline__ Moments of(int k, float count, float inverse) const {
    const Moments first = of(k, count, inverse);
    if constexpr (SPAN == 1) return first;
    float shift = 0.0f, square = first.square;
#pragma unroll
    for (int i = 1; i < SPAN; ++i) shift += distance(of(k + i, count, inverse), first);
    shift *= 1.0f / SPAN;
    square = fmaf(count * shift, shift, square);
#pragma unroll
    for (int i = 1; i < SPAN; ++i) {
      const Moments v = of(k + i, count, inverse);
      const float d = distance(v, first) - shift;
      square += fmaf(count * d, d, v.square);
    }
    return moments_of(first.mean, first.rest + shift, square, count * SPAN);
  }
  template <int SPAN>
  __device__ __forceinline__ void tell(Moments* to, int rows) const {
    const float inverse = rows > 0 ? 1.0f / rows : 0.0f;
#pragma unroll
    for (int k = 0; k < V; k += SPAN) to[k / SPAN] = rows > 0 ? of<SPAN>(k, (float)rows, inverse) : Moments{};
  }
};

// What the CTA's threads have summed, per group of the block: put(g, moments), by one thread each.  `told`: shared memory, an entry for
// every run of a thread's channels that lie in one group.  Ends in a barrier.
template <typename T, int V, bool WHOLE, typename F>
__device__ __forceinline__ void group_moments(const NormParams& p, const NormPlace& t, const NormMoments<T, V>& m, Moments* told, int columns, F&& put) {
  constexpr int kHalf = V % 2 == 0 ? V / 2 : 1;
  const int each = WHOLE ? 1 : p.width == kHalf ? V / kHalf : V;  // entries of a thread
  if (t.depth < p.depth && t.lane < columns) {
    Moments* mine = told + (t.depth * columns + t.lane) * each;
    if (WHOLE) m.template tell<V>(mine, t.count);
    else if (p.width == kHalf) m.template tell<kHalf>(mine, t.count);
    else m.template tell<1>(mine, t.count);
  }
  __syncthreads();
  join_rows(told, p.depth, columns * each);
  // (a block wider than the CTA is one group, taken part by part)
  const int groups = columns < p.columns ? 1 : p.block_groups, entries = columns * each / groups;
  if (entries == 1) {
    for (int g = threadIdx.x; g < groups; g += kNormThreads) put(g, told[g]);
  } else {
    const NormTeam team(groups, entries);
    team.each(groups, [&](int g, bool there) {
      const Moments all = team_join(team, told + g * entries, entries);
      if (there && team.lane == 0) put(g, all);
    });
  }
  __syncthreads();
}

template <typename T, int V, bool WHOLE>
__global__ void __launch_bounds__(kNormThreads, 2) norm_stats(const __grid_constant__ NormParams p) {
  extern __shared__ Moments norm_told[];
  __shared__ Moments parts;
  typedef Vec<T, V> Vector;
  grid_dependency();
  const NormPlace t = norm_place(p, blockIdx.x);
  const T* x = (const T*)p.x + (t.n * p.S + t.row) * p.C + (long long)t.group * p.width + t.lane * V;
  const long long step = (long long)p.depth * p.C;
  Moments* to = p.moments + ((long long)t.n * p.chunks + t.chunk) * p.groups + t.group;
  for (int c0 = 0; c0 < p.columns; c0 += p.lanes) {  // (once, but for groups wider than the CTA)
    const int columns = min(p.lanes, p.columns - c0);
    NormMoments<T, V> m;
    if (t.count > 0 && t.lane < columns) {
      const T* at = x + (long long)c0 * V;
      m.start(*(const Vector*)at);
      walk<4>(t.count - 1, [&](int) { return *(const Vector*)(at += step); }, [&](int, const Vector& v) { m.add(v); });
    }
    group_moments<T, V, WHOLE>(p, t, m, norm_told, columns, [&](int g, const Moments& v) {
      if (columns == p.columns) {
        to[g] = v;
      } else {  // the parts of one group, by one thread
        parts = c0 == 0 ? v : joined(parts, v);
        if (c0 + columns == p.columns) to[g] = parts;
      }
    });
  }
}

// ---- normalised rows ----------------------------------------------------------------------------------
// What belongs to a thread's channels: z = (x - mean) factor + bias (less the mean's rest times factor).
template <typename T, int V, bool WHOLE>
struct NormChannels {
  typedef FloatPairs<T, V> P;
  static constexpr int kOwn = WHOLE ? 1 : P::kPairs;
  float2 mean[kOwn];  // of the vector's group, or of the channels'
  P factor, bias;
  // weights and biases of the vector `column` of the block (asked for before what they have to wait for)
  __device__ __forceinline__ NormChannels(const NormParams& p, const NormPlace& t, int column) {
    float w[V], b[V];
    parameters_of<V>(p, w, b, t.group * p.width + column * V);
#pragma unroll
    for (int k = 0; k < P::kPairs; ++k) {
      factor.v[k] = make_float2(w[2 * k], w[V == 1 ? 0 : 2 * k + 1]);
      bias.v[k] = make_float2(b[2 * k], b[V == 1 ? 0 : 2 * k + 1]);
    }
  }
  // `means`, `rstds`, `rests` (or null: 0): of the groups of the block
  __device__ __forceinline__ void set(const NormParams& p, int column, const float* means, const float* rstds, const float* rests) {
    if constexpr (WHOLE) {
      const int g = p.by_width.quotient(column * V);
      mean[0] = two(means[g]);
      const float2 r = two(rstds[g]), less = two(rests ? -rests[g] : 0.0f);
#pragma unroll
      for (int k = 0; k < P::kPairs; ++k) {
        factor.v[k] = mul2(factor.v[k], r);
        bias.v[k] = fma2(factor.v[k], less, bias.v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < P::kPairs; ++k) {
        const int g = p.by_width.quotient(column * V + 2 * k), h = p.by_width.quotient(column * V + 2 * k + 1);
        mean[k] = make_float2(means[g], means[h]);
        factor.v[k] = mul2(factor.v[k], make_float2(rstds[g], rstds[h]));
        if (rests) bias.v[k] = fma2(factor.v[k], make_float2(-rests[g], -rests[h]), bias.v[k]);
      }
    }
  }
  __device__ __forceinline__ float2 centred(int k, float2 x) const { return fma2(mean[WHOLE ? 0 : k], two(-1.0f), x); }
};

template <typename T, int ACT, int V, bool WHOLE>
__device__ __forceinline__ Vec<T, V> normalised(const Vec<T, V>& v, const NormChannels<T, V, WHOLE>& c) {
  FloatPairs<T, V> x(v);
#pragma unroll
  for (int k = 0; k < FloatPairs<T, V>::kPairs; ++k) {
    float2 slope;
    x.v[k] = activate<T, ACT>(fma2(c.centred(k, x.v[k]), c.factor.v[k], c.bias.v[k]), slope);
  }
  return x.vector();
}

// A store of what this kernel does not read again.
template <typename V>
__device__ __forceinline__ void put_once(V* to, const V& v) {
  if constexpr (sizeof(V) == 16) __stcs((uint4*)to, *(const uint4*)&v);
  else *to = v;
}

__device__ __forceinline__ void keep_statistics(const NormParams& p, const NormPlace& t, int g, float mean, float rstd, float rest) {
  const long long at = (long long)t.n * p.groups + t.group + g;
  p.mean[at] = mean;
  p.rstd[at] = rstd;
  if (p.rest) p.rest[at] = rest;
}
// Of the groups of a block, as the forward has left them.
struct NormStatistics {
  const float *means, *rstds, *rests;
  __device__ __forceinline__ NormStatistics(const NormParams& p, const NormPlace& t) {
    const long long at = (long long)t.n * p.groups + t.group;
    means = p.mean + at;
    rstds = p.rstd + at;
    rests = p.rest ? p.rest + at : nullptr;
  }
};

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 2) norm_apply(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) float norm_groups[];  // the block's means, their inverse deviations, what the threads have joined
  typedef Vec<T, V> Vector;
  grid_dependency();
  const NormPlace t = norm_place(p, blockIdx.x);
  float *means = norm_groups, *rstds = means + p.block_groups, *rests = rstds + p.block_groups;
  NormChannels<T, V, WHOLE> c(p, t, t.lane);
  // an image's chunks: a thread takes every so many of a group's, then the threads are joined
  Moments* told = (Moments*)(norm_groups + ((3 * p.block_groups + 3) & ~3));
  const Moments* from = p.moments + (long long)t.n * p.chunks * p.groups + t.group;
  const int parts = min(p.chunks, max(1, kNormThreads / p.block_groups));
  for (int i = threadIdx.x; i < parts * p.block_groups; i += kNormThreads) {
    const int part = i / p.block_groups, g = i - part * p.block_groups;
    Moments first = {};
    float count = 0.0f, sum = 0.0f, square = 0.0f;
    walk<8>((p.chunks - part + parts - 1) / parts, [&](int k) { return from[(long long)(part + k * parts) * p.groups + g]; }, [&](int k, const Moments& v) {
      if (k == 0) first = v;
      const float d = distance(v, first);  // (about the first chunk's mean)
      count += v.count;
      sum = fmaf(v.count, d, sum);
      square += fmaf(v.count * d, d, v.square);
    });
    const float shift = sum / count;
    told[i] = moments_of(first.mean, first.rest + shift, not_negative(fmaf(-shift, sum, square)), count);
  }
  __syncthreads();
  join_rows(told, parts, p.block_groups);
  for (int g = threadIdx.x; g < p.block_groups; g += kNormThreads) {
    const Moments all = told[g];
    means[g] = all.mean;
    rests[g] = all.rest;
    rstds[g] = 1.0f / sqrtf(all.square / all.count + p.eps);
    if (t.chunk == 0) keep_statistics(p, t, g, means[g], rstds[g], rests[g]);
  }
  __syncthreads();
  if (t.count == 0) return;
  const long long step = (long long)p.depth * p.C, first = (t.n * p.S + t.row) * p.C + (long long)t.group * p.width;
  for (int column = t.lane; column < p.columns; column += p.lanes) {
    if (column != t.lane) c = NormChannels<T, V, WHOLE>(p, t, column);
    c.set(p, column, means, rstds, rests);
    const long long last = first + (t.count - 1) * step + (long long)column * V;
    const T* x = (const T*)p.x + last + step;
    T* out = (T*)p.out + last + step;
    walk<6>(t.count, [&](int) { return *(const Vector*)(x -= step); }, [&](int, const Vector& v) { put_once((Vector*)(out -= step), normalised<T, ACT>(v, c)); });
  }
}

// Shared memory of a CTA of a cluster: what its threads have summed, its groups' sums, its groups' two or three numbers, then the rows.
struct NormShared {
  char *told, *groups;
  float *first, *second, *third;
  char* rows;
  __device__ __forceinline__ NormShared(const NormParams& p, char* base, int told_bytes) {
    told = base;
    groups = told + told_bytes;
    first = (float*)(groups + 16 * p.block_groups);
    second = first + p.block_groups;
    third = second + p.block_groups;
    rows = base + bytes(told_bytes, p.block_groups);
  }
  static __host__ __device__ __forceinline__ int bytes(int told, int groups) { return (told + groups * 28 + 15) & ~15; }
};

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 2) norm_cluster(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) char norm_bytes[];
  typedef Vec<T, V> Vector;
  const NormShared sh(p, norm_bytes, p.depth * p.lanes * (WHOLE ? 1 : V) * (int)sizeof(Moments));
  const int image = blockIdx.x / p.chunks, n = image / p.blocks;  // (block, image, CTA of the cluster)
  const NormPlace t = norm_place(p, n, image - n * p.blocks, blockIdx.x - image * p.chunks);
  grid_dependency();
  const long long step = (long long)p.depth * p.C, first = (t.n * p.S + t.row) * p.C + (long long)t.group * p.width + t.lane * V;
  Vector* rows = (Vector*)sh.rows + t.depth * p.lanes + t.lane;  // of this thread
  const int next = p.depth * p.lanes;
  NormChannels<T, V, WHOLE> c(p, t, t.lane);
  NormMoments<T, V> m;
  if (t.count > 0) {
    const T* x = (const T*)p.x + first;
    m.start(rows[0] = *(const Vector*)x);
    walk<4>(t.count - 1, [&](int) { return *(const Vector*)(x += step); }, [&](int i, const Vector& v) { m.add(rows[(i + 1) * next] = v); });
  }
  Moments* groups = (Moments*)sh.groups;
  group_moments<T, V, WHOLE>(p, t, m, (Moments*)sh.told, p.columns, [&](int g, const Moments& v) { groups[g] = v; });
  if (p.chunks > 1) cluster_sync();
  for (int g = threadIdx.x; g < p.block_groups; g += kNormThreads) {
    Moments all = groups[g];
    if (p.chunks > 1) {
      walk<8>(p.chunks, [&](int i) { return of_cluster(groups + g, i); }, [&](int i, const Moments& v) { all = i == 0 ? v : joined(all, v); });
    }
    sh.first[g] = all.mean;
    sh.second[g] = 1.0f / sqrtf(all.square / all.count + p.eps);
    sh.third[g] = all.rest;
    if (t.chunk == 0) keep_statistics(p, t, g, sh.first[g], sh.second[g], sh.third[g]);
  }
  __syncthreads();
  if (t.count > 0) {
    c.set(p, t.lane, sh.first, sh.second, sh.third);
    T* out = (T*)p.out + first;
    walk<4>(t.count, [&](int i) { return rows[i * next]; }, [&](int i, const Vector& v) { *(Vector*)(out + i * step) = normalised<T, ACT>(v, c); });
  }
  if (p.chunks > 1) cluster_sync();  // (no CTA ends while another reads its shared memory)
}

// ---- backward -----------------------------------------------------------------------------------------
template <typename Vector>
struct Both {
  Vector x, dy;
};
template <typename Vector, typename T>
__device__ __forceinline__ Both<Vector> load_both(const T*& x, const T*& dy, long long step) {
  const Both<Vector> v = {*(const Vector*)x, *(const Vector*)dy};
  x += step;
  dy += step;
  return v;
}

// Sums of dz and dz (x - mean), of a vector of channels.
template <typename T, int V>
struct NormSlopes {
  typedef FloatPairs<T, V> P;
  P dz, product;
  __device__ __forceinline__ NormSlopes() {
#pragma unroll
    for (int k = 0; k < P::kPairs; ++k) dz.v[k] = product.v[k] = two(0.0f);
  }
  template <int ACT, bool WHOLE>
  __device__ __forceinline__ void add(const Vec<T, V>& x, const Vec<T, V>& dy, const NormChannels<T, V, WHOLE>& c) {
    const P a(x), g(dy);
#pragma unroll
    for (int k = 0; k < P::kPairs; ++k) {
      const float2 centred = c.centred(k, a.v[k]);
      float2 slope;
      activate<T, ACT>(fma2(centred, c.factor.v[k], c.bias.v[k]), slope);
      const float2 d = mul2(g.v[k], slope);
      dz.v[k] = add2(dz.v[k], d);
      product.v[k] = fma2(d, centred, product.v[k]);
    }
  }
};

// The CTA's sums per channel (dz, dz xhat), over `columns` vectors from vector c0 of the block on: channel(c, sums) by one thread each, with
// them in `told`[c].  `told`: shared memory, two floats a channel of every thread.  Ends in a barrier.
template <typename T, int V, typename F>
__device__ __forceinline__ void channel_sums(const NormParams& p, const NormPlace& t, const NormSlopes<T, V>& mine, float2* told, int columns, int c0,
                                             const NormStatistics& of, F&& channel) {
  const int channels = columns * V;
  if (t.depth < p.depth && t.lane < columns) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      told[t.depth * channels + t.lane * V + k] = k & 1 ? make_float2(mine.dz.v[k >> 1].y, mine.product.v[k >> 1].y) : make_float2(mine.dz.v[k >> 1].x, mine.product.v[k >> 1].x);
  }
  __syncthreads();
  join_rows(told, p.depth, channels);
  for (int c = threadIdx.x; c < channels; c += kNormThreads) {
    float2 s = told[c];
    const int g = p.by_width.quotient(c0 * V + c);
    s.y = (of.rests ? fmaf(-of.rests[g], s.x, s.y) : s.y) * of.rstds[g];
    told[c] = s;
    channel(c0 * V + c, s);
  }
  __syncthreads();
}

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 2) norm_sums(const __grid_constant__ NormParams p) {
  extern __shared__ float2 norm_slopes[];
  typedef Vec<T, V> Vector;
  grid_dependency();
  const NormPlace t = norm_place(p, blockIdx.x);
  const NormStatistics of(p, t);
  const long long step = (long long)p.depth * p.C, first = (t.n * p.S + t.row) * p.C + (long long)t.group * p.width + t.lane * V;
  const long long number = (long long)t.n * p.chunks + t.chunk;
  float2 before = two(0.0f);  // (of the parts of one group)
  for (int c0 = 0; c0 < p.columns; c0 += p.lanes) {
    const int columns = min(p.lanes, p.columns - c0);
    NormSlopes<T, V> s;
    if (t.count > 0 && t.lane < columns) {
      NormChannels<T, V, WHOLE> c(p, t, c0 + t.lane);
      c.set(p, c0 + t.lane, of.means, of.rstds, of.rests);
      const T *x = (const T*)p.x + first + (long long)c0 * V, *dy = (const T*)p.dy + first + (long long)c0 * V;
      walk<3>(t.count, [&](int) { return load_both<Vector>(x, dy, step); }, [&](int, const Both<Vector>& v) { s.template add<ACT>(v.x, v.dy, c); });
    }
    channel_sums<T, V>(p, t, s, norm_slopes, columns, c0, of, [&](int c, float2 v) { p.slopes[number * p.C + (long long)t.group * p.width + c] = v; });
    const int groups = columns < p.columns ? 1 : p.block_groups, width = columns * V / groups;
    const NormTeam team(groups, width);
    team.each(groups, [&](int g, bool there) {
      float2 all = two(0.0f);
      for (int k = team.lane; k < width; k += team.size) all = fma2(two(weight_of(p, t.group * p.width + c0 * V + g * width + k)), norm_slopes[g * width + k], all);
      before = make_float2(before.x * (c0 > 0) + team.sum(all.x), before.y * (c0 > 0) + team.sum(all.y));
      if (there && team.lane == 0 && c0 + columns == p.columns) p.sums[number * p.groups + t.group + g] = before;
    });
    __syncthreads();
  }
}

// Gradients of weights and biases of 32 channels: sums over all images' chunks.
__device__ __forceinline__ void parameter_gradients(const NormParams& p, int cta, float2* shared) {
  const int channel = cta * 32 + (threadIdx.x & 31);
  const long long entries = (long long)p.N * p.chunks;
  float2 s = two(0.0f);
  if (channel < p.C) {
#pragma unroll 4
    for (long long e = threadIdx.x >> 5; e < entries; e += kNormThreads / 32) s = add2(s, p.slopes[e * p.C + channel]);
  }
  shared[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || channel >= p.C) return;
  for (int i = 1; i < kNormThreads / 32; ++i) s = add2(s, shared[i * 32 + threadIdx.x]);
  if (p.dweight) put_parameter(p, p.dweight, channel, s.y);
  if (p.dbias) put_parameter(p, p.dbias, channel, s.x);
}
static __global__ void __launch_bounds__(kNormThreads) norm_parameters(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[kNormThreads];
  grid_dependency();
  parameter_gradients(p, blockIdx.x, shared);
}

// dx = dz factor - rstd m1 - (x - mean) rstd^2 m2, with the mean's rest in the part that is the same for all rows
template <typename T, int V, bool WHOLE>
struct NormReturn {
  float2 first[NormChannels<T, V, WHOLE>::kOwn], second[NormChannels<T, V, WHOLE>::kOwn];  // negative
  // m1, m2: of the groups of the block
  __device__ __forceinline__ NormReturn(const NormParams& p, int column, const float* m1, const float* m2, const NormStatistics& of) {
#pragma unroll
    for (int k = 0; k < 2 * NormChannels<T, V, WHOLE>::kOwn; ++k) {
      const int g = p.by_width.quotient(column * V + (k < V ? k : 0));
      const float rstd = of.rstds[g], b = -rstd * rstd * m2[g], a = fmaf(-rstd, m1[g], of.rests ? -of.rests[g] * b : 0.0f);
      if (k & 1) first[k >> 1].y = a, second[k >> 1].y = b;
      else first[k >> 1].x = a, second[k >> 1].x = b;
    }
    if (WHOLE) first[0].y = first[0].x, second[0].y = second[0].x;
  }
  template <int ACT>
  __device__ __forceinline__ Vec<T, V> gradient(const Vec<T, V>& x, const Vec<T, V>& dy, const NormChannels<T, V, WHOLE>& c) const {
    const FloatPairs<T, V> a(x);
    FloatPairs<T, V> g(dy);
#pragma unroll
    for (int k = 0; k < FloatPairs<T, V>::kPairs; ++k) {
      const float2 centred = c.centred(k, a.v[k]);
      float2 slope;
      activate<T, ACT>(fma2(centred, c.factor.v[k], c.bias.v[k]), slope);
      g.v[k] = fma2(centred, second[WHOLE ? 0 : k], fma2(mul2(g.v[k], slope), c.factor.v[k], first[WHOLE ? 0 : k]));
    }
    return g.vector();
  }
};

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 2) norm_dx(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) float norm_groups[];  // m1, m2 of the block's groups (and what the parameters' CTAs sum)
  typedef Vec<T, V> Vector;
  grid_dependency();
  if ((int)blockIdx.x < p.channel_ctas) {
    parameter_gradients(p, blockIdx.x, (float2*)norm_groups);
    return;
  }
  const NormPlace t = norm_place(p, blockIdx.x - p.channel_ctas);
  const NormStatistics of(p, t);
  float *m1 = norm_groups, *m2 = m1 + p.block_groups;
  NormChannels<T, V, WHOLE> c(p, t, t.lane);
  const float all = (float)p.S * p.width;
  float2* told = (float2*)(m2 + p.block_groups);
  const float2* from = p.sums + (long long)t.n * p.chunks * p.groups + t.group;
  const int parts = min(p.chunks, max(1, kNormThreads / p.block_groups));
  for (int i = threadIdx.x; i < parts * p.block_groups; i += kNormThreads) {
    const int part = i / p.block_groups, g = i - part * p.block_groups;
    float2 sum = two(0.0f);
    walk<8>((p.chunks - part + parts - 1) / parts, [&](int k) { return from[(long long)(part + k * parts) * p.groups + g]; },
            [&](int, const float2& v) { sum = add2(sum, v); });
    told[i] = sum;
  }
  __syncthreads();
  join_rows(told, parts, p.block_groups);
  for (int g = threadIdx.x; g < p.block_groups; g += kNormThreads) m1[g] = told[g].x / all, m2[g] = told[g].y / all;
  __syncthreads();
  if (t.count == 0) return;
  const long long step = (long long)p.depth * p.C, first = (t.n * p.S + t.row) * p.C + (long long)t.group * p.width;
  for (int column = t.lane; column < p.columns; column += p.lanes) {
    if (column != t.lane) c = NormChannels<T, V, WHOLE>(p, t, column);
    c.set(p, column, of.means, of.rstds, of.rests);
    const NormReturn<T, V, WHOLE> back(p, column, m1, m2, of);
    const long long last = first + (t.count - 1) * step + (long long)column * V;
    const T *x = (const T*)p.x + last, *dy = (const T*)p.dy + last;
    T* dx = (T*)p.dx + last + step;
    walk<3>(t.count, [&](int) { return load_both<Vector>(x, dy, -step); },
            [&](int, const Both<Vector>& v) { put_once((Vector*)(dx -= step), back.template gradient<ACT>(v.x, v.dy, c)); });
  }
}

// All of a block of groups: dx, and the block's channels' sums of the image (a chunk an image).
template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 2) norm_cluster_backward(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) char norm_bytes[];
  typedef Vec<T, V> Vector;
  const NormShared sh(p, norm_bytes, p.depth * p.lanes * V * (int)sizeof(float2));
  const int image = blockIdx.x / p.chunks, n = image / p.blocks;
  const NormPlace t = norm_place(p, n, image - n * p.blocks, blockIdx.x - image * p.chunks);
  grid_dependency();
  const NormStatistics of(p, t);
  const long long step = (long long)p.depth * p.C, first = (t.n * p.S + t.row) * p.C + (long long)t.group * p.width + t.lane * V;
  Vector* rows = (Vector*)sh.rows + (t.depth * p.lanes + t.lane) * 2;  // of this thread: x and dy
  const int next = p.depth * p.lanes * 2;
  NormChannels<T, V, WHOLE> c(p, t, t.lane);
  c.set(p, t.lane, of.means, of.rstds, of.rests);
  NormSlopes<T, V> s;
  if (t.count > 0) {
    const T *x = (const T*)p.x + first, *dy = (const T*)p.dy + first;
    walk<2>(t.count, [&](int) { return load_both<Vector>(x, dy, step); }, [&](int i, const Both<Vector>& v) {
      rows[i * next] = v.x;
      rows[i * next + 1] = v.dy;
      s.template add<ACT>(v.x, v.dy, c);
    });
  }
  float2* told = (float2*)sh.told;
  channel_sums<T, V>(p, t, s, told, p.columns, 0, of, [&](int, float2) {});
  if (p.chunks > 1) cluster_sync();
  const float all = (float)p.S * p.width;
  const NormTeam team(p.block_groups, p.width);
  team.each(p.block_groups, [&](int g, bool there) {
    float2 sum = two(0.0f);
    for (int k = team.lane; k < p.width; k += team.size) {
      const int at = g * p.width + k;
      float2 v = told[at];
      if (p.chunks > 1) {
        v = of_cluster(told + at, 0);
        for (int i = 1; i < p.chunks; ++i) v = add2(v, of_cluster(told + at, i));
      }
      if (there && t.chunk == 0) p.slopes[(long long)t.n * p.C + t.group * p.width + at] = v;
      sum = fma2(two(weight_of(p, t.group * p.width + at)), v, sum);
    }
    sum = make_float2(team.sum(sum.x), team.sum(sum.y));
    if (there && team.lane == 0) sh.first[g] = sum.x / all, sh.second[g] = sum.y / all;
  });
  __syncthreads();
  if (t.count > 0) {
    const NormReturn<T, V, WHOLE> back(p, t.lane, sh.first, sh.second, of);
    T* dx = (T*)p.dx + first;
    walk<2>(t.count, [&](int i) { return Both<Vector>{rows[i * next], rows[i * next + 1]}; },
            [&](int i, const Both<Vector>& v) { *(Vector*)(dx + i * step) = back.template gradient<ACT>(v.x, v.dy, c); });
  }
  if (p.chunks > 1) cluster_sync();
}

}  // namespace mvr
