// Group norm with its activation over channels-last tensors (N, S, C), groups of consecutive channels:
//   xhat = (x - mean) rstd    z = xhat w + b    y = act(z)            mean, variance of an image's group: S * C / groups values
//   dz = dy act'(z)    db = sum dz    dw = sum dz xhat    dx = rstd (dz w - m1 - xhat m2)    m1, m2: the group's means of dz w, dz w xhat
//
// Every pass walks rows with one vector of channels a thread, so that what belongs to a channel stays in registers.  Forward: per-channel
// mean and sum of squares of every chunk of rows, their union per group, then the elements.  Backward: per-channel sums of dz and dz xhat
// of every chunk, their union, then dx.  No atomics: each sum has one place and one order.
//
// Statistics.  A thread sums x - k and (x - k)^2 about its own first value k of a channel, over its r rows.  If k lies far from the others,
// the thread's sum of squares about its mean is itself at least (r - 1) / r of that distance's square, so that cancellation costs no
// more than some r of its last bits, whatever the data's offset.  Threads, chunks and channels are joined by their means' differences, for
// which a mean is kept as two floats: rounded to one, means near 1e5 of values with a deviation of 2 put an error of 1e-4 into their variance.
#pragma once
#include "mvr_types.cuh"

namespace mvr {

enum { kNoActivation = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// Mean, as a float and what its rounding left, and sum of squares about it.
struct alignas(16) Moments {
  float mean, rest, square, unused;
};

struct NormParams {
  const void *x, *dy, *weight, *bias;  // (N, S, C) twice; (C), or null: 1 and 0
  void *out, *dx, *dweight, *dbias;
  float *mean, *rstd;                  // (N, groups)
  Moments* moments;                    // (N, chunks, C): forward
  float2* part;                        // (N, chunks, C): backward, sums of dz and dz xhat
  float2* means;                       // (N, groups): m1, m2
  long long S, rows;                   // rows of a chunk, or of a CTA of a cluster
  int N, C, groups, width;             // width: channels of a group
  int parameters;                      // type of weight and bias: 0 float, 1 half, 3 bfloat16
  int chunks;                          // of an image; or CTAs of a cluster
  int columns, lanes, depth;           // vectors of a row; of those a CTA takes `lanes`, `depth` rows at a time
  int blocks;                          // of lanes in a row
  float eps;
};

constexpr int kNormThreads = 256;

__device__ __forceinline__ float parameter(const NormParams& p, const void* from, int c) {
  return p.parameters == 0 ? ((const float*)from)[c] : p.parameters == 1 ? to_float(((const __half*)from)[c]) : to_float(((const __nv_bfloat16*)from)[c]);
}
__device__ __forceinline__ float weight_of(const NormParams& p, int c) { return p.weight ? parameter(p, p.weight, c) : 1.0f; }
__device__ __forceinline__ void put_parameter(const NormParams& p, void* to, int c, float v) {
  if (p.parameters == 0) ((float*)to)[c] = v;
  else if (p.parameters == 1) ((__half*)to)[c] = from_float<__half>(v);
  else ((__nv_bfloat16*)to)[c] = from_float<__nv_bfloat16>(v);
}

// act(z), and act'(z).
template <typename T, int ACT>
__device__ __forceinline__ float activate(float z, float& slope) {
  constexpr bool kExact = sizeof(T) == 4;  // (the fast forms are off by 2^-20 up to |z| = 10, a 2^-9 of half a step of float16)
  if (ACT == kRelu) {
    slope = z > 0.0f ? 1.0f : 0.0f;
    return z > 0.0f || z != z ? z : 0.0f;
  }
  if (ACT == kSilu) {
    const float gate = kExact ? 1.0f / (1.0f + expf(-z)) : __fdividef(1.0f, 1.0f + __expf(-z));
    slope = gate * fmaf(z, 1.0f - gate, 1.0f);
    return z * gate;
  }
  if (ACT == kGelu) {
    const float gate = normcdff(z);
    slope = fmaf(z * 0.3989422804014327f, kExact ? expf(-0.5f * z * z) : __expf(-0.5f * z * z), gate);
    return z * gate;
  }
  slope = 1.0f;
  return z;
}

// A thread's place: its channels [channel, channel + V) and the rows of its chunk that it walks.
struct NormPlace {
  int n, chunk, block, lane, depth, channel;
  long long begin, end, row;  // of the chunk; its first one
  bool in;
};
// CTA `cta` of the grid: block of lanes, chunk, image.
template <int V>
__device__ __forceinline__ NormPlace norm_place(const NormParams& p, int cta, bool backwards = false) {
  NormPlace t;
  const int number = cta / p.blocks, chunk = number % p.chunks;
  t.block = cta - number * p.blocks;
  t.n = number / p.chunks;
  t.chunk = backwards ? p.chunks - 1 - chunk : chunk;
  t.depth = threadIdx.x / p.lanes;
  t.lane = threadIdx.x - t.depth * p.lanes;
  const int column = t.block * p.lanes + t.lane;
  t.in = t.depth < p.depth && column < p.columns;
  t.channel = column * V;
  t.begin = t.chunk * p.rows;
  t.end = max(t.begin, min(p.S, t.begin + p.rows));
  t.row = t.begin + t.depth;
  return t;
}

// Per channel, what every depth has; f(values, their distance, place, channel) joins them.
template <int V, typename E, typename F>
__device__ __forceinline__ void by_channel(const NormParams& p, const NormPlace& t, E* norm_shared, const E (&mine)[V], F&& f) {
  const int width = p.lanes * V;  // norm_shared: (depth, width)
  if (t.depth < p.depth) {
#pragma unroll
    for (int k = 0; k < V; ++k) norm_shared[t.depth * width + t.lane * V + k] = mine[k];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += kNormThreads)
    if (t.block * width + c < p.C) f(norm_shared + c, width, c, t.block * width + c);
}

// ---- forward ------------------------------------------------------------------------------------------
__device__ __forceinline__ Moments moments_of(float a, float b, float square) {  // mean: a + b
  const float mean = a + b, of_b = mean - a;
  return {mean, (a - (mean - of_b)) + (b - of_b), square, 0.0f};
}
__device__ __forceinline__ float distance(const Moments& a, const Moments& b) { return (a.mean - b.mean) + (a.rest - b.rest); }

// Sums about a pivot, of V channels.
template <int V>
struct NormMoments {
  float pivot[V] = {}, sum[V] = {}, square[V] = {};
  int count = 0;
  template <typename T>
  __device__ __forceinline__ void start(const Vec<T, V>& v) {
    count = 1;
#pragma unroll
    for (int k = 0; k < V; ++k) pivot[k] = to_float(v.v[k]);
  }
  template <typename T>
  __device__ __forceinline__ void add(const Vec<T, V>& v) {
    ++count;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = to_float(v.v[k]) - pivot[k];
      sum[k] += d;
      square[k] = fmaf(d, d, square[k]);
    }
  }
  __device__ __forceinline__ void get(Moments (&to)[V]) const {
    const float inverse = count > 0 ? 1.0f / count : 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) to[k] = moments_of(pivot[k], sum[k] * inverse, fmaxf(0.0f, fmaf(-sum[k] * inverse, sum[k], square[k])));
  }
};
// Of `rows` rows that `depth` threads took in turns, together.
__device__ __forceinline__ Moments join_moments(const Moments* v, int width, int depth, int rows) {
  const auto rows_of = [&](int i) { return (float)((rows - i + depth - 1) / depth); };
  const Moments first = v[0];
  float mean = 0.0f, m2 = 0.0f;  // (mean: from the first one's)
  const int some = min(depth, rows);
  for (int i = 0; i < some; ++i) mean = fmaf(rows_of(i), distance(v[i * width], first), mean);
  mean /= (float)max(1, rows);
  for (int i = 0; i < some; ++i) {
    const float d = distance(v[i * width], first) - mean;
    m2 += fmaf(rows_of(i) * d, d, v[i * width].square);
  }
  return moments_of(first.mean, first.rest + mean, m2);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) norm_stats(const __grid_constant__ NormParams p) {
  extern __shared__ Moments norm_moments[];
  grid_dependency();
  const NormPlace t = norm_place<V>(p, blockIdx.x);
  typedef Vec<T, V> Vector;
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  NormMoments<V> m;
  if (t.in) {
    long long r = t.row;
    if (r < t.end) m.start(*(const Vector*)(x + r * p.C));
#pragma unroll 4
    for (r += p.depth; r < t.end; r += p.depth) m.add(*(const Vector*)(x + r * p.C));
  }
  Moments mine[V];
  m.get(mine);
  by_channel<V>(p, t, norm_moments, mine, [&](const Moments* v, int width, int, int channel) {
    p.moments[((long long)t.n * p.chunks + t.chunk) * p.C + channel] = join_moments(v, width, p.depth, (int)(t.end - t.begin));
  });
}

__device__ __forceinline__ float norm_sum(float v, float* shared) {  // over the CTA, the same in all threads
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  float total = 0.0f;
  for (int i = 0; i < kNormThreads / 32; ++i) total += shared[i];
  return total;
}

// Statistics of a group of an image, from its channels' chunks.
static __global__ void __launch_bounds__(kNormThreads) norm_finish(const __grid_constant__ NormParams p) {
  __shared__ float shared[kNormThreads / 32];
  grid_dependency();
  const int n = blockIdx.x / p.groups, g = blockIdx.x - n * p.groups, entries = p.chunks * p.width;
  const Moments* part = p.moments + (long long)n * p.chunks * p.C + g * p.width;
  const auto at = [&](int e, float& rows) {
    const int chunk = e / p.width;
    rows = (float)min(p.rows, p.S - chunk * p.rows);
    return part[(long long)chunk * p.C + (e - chunk * p.width)];
  };
  const Moments first = part[0];
  const float all = (float)p.S * p.width;
  float sum = 0.0f, rows;
  for (int e = threadIdx.x; e < entries; e += kNormThreads) {
    const Moments v = at(e, rows);
    sum = fmaf(rows, distance(v, first), sum);
  }
  const float mean = norm_sum(sum, shared) / all;
  float m2 = 0.0f;
  for (int e = threadIdx.x; e < entries; e += kNormThreads) {
    const Moments v = at(e, rows);
    const float d = distance(v, first) - mean;
    m2 += fmaf(rows * d, d, v.square);
  }
  m2 = norm_sum(m2, shared);
  if (threadIdx.x == 0) {
    p.mean[n * p.groups + g] = first.mean + (first.rest + mean);
    p.rstd[n * p.groups + g] = 1.0f / sqrtf(m2 / all + p.eps);
  }
}

// What belongs to a thread's channels.  mean, rstd: of the groups from `first` on.
template <int V>
struct NormChannels {
  float mean[V], rstd[V], weight[V], bias[V];
  __device__ __forceinline__ NormChannels(const NormParams& p, const NormPlace& t, const float* means, const float* rstds, int first) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = t.in ? t.channel + k : first * p.width, g = c / p.width - first;
      mean[k] = means[g];
      rstd[k] = rstds[g];
      weight[k] = weight_of(p, c);
      bias[k] = p.bias ? parameter(p, p.bias, c) : 0.0f;
    }
  }
};

template <typename T, int ACT, int V>
__device__ __forceinline__ Vec<T, V> normalised(Vec<T, V> v, const NormChannels<V>& c) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float slope;
    v.v[k] = from_float<T>(activate<T, ACT>(fmaf((to_float(v.v[k]) - c.mean[k]) * c.rstd[k], c.weight[k], c.bias[k]), slope));
  }
  return v;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_apply(const __grid_constant__ NormParams p) {
  grid_dependency();
  // (an image's last chunks were read last, and are the likeliest still in L2)
  const NormPlace t = norm_place<V>(p, blockIdx.x, true);
  const NormChannels<V> c(p, t, p.mean + (long long)t.n * p.groups, p.rstd + (long long)t.n * p.groups, 0);
  if (!t.in) return;
  typedef Vec<T, V> Vector;
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  T* out = (T*)p.out + t.n * p.S * p.C + t.channel;
#pragma unroll 4
  for (long long r = t.row; r < t.end; r += p.depth) *(Vector*)(out + r * p.C) = normalised<T, ACT>(*(const Vector*)(x + r * p.C), c);
}

// ---- clusters -----------------------------------------------------------------------------------------
// Where an image's block of whole groups fits the shared memory of a cluster's CTAs (or of one CTA), one kernel does it all: each CTA
// brings its rows into shared memory, the CTAs tell each other their channels' sums, and the rows are read a second time where they lie.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 of_cluster(const float2* mine, int rank) {  // the same place in CTA `rank` of the cluster
  uint32_t at;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ Moments of_cluster(const Moments* mine, int rank) {
  uint32_t at;
  Moments v = {};
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.mean), "=f"(v.rest), "=f"(v.square), "=f"(v.unused) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
// Shared memory of a CTA: what each depth tells (depth, lanes V), its channels (lanes V), its groups' two numbers, then the rows.
template <typename E, int V>
struct NormShared {
  E *told, *channels;
  float *first, *second;
  char* rows;
  __device__ __forceinline__ NormShared(const NormParams& p, char* base) {
    const int width = p.lanes * V, groups = width / p.width;
    told = (E*)base;
    channels = told + p.depth * width;
    first = (float*)(channels + width);
    second = first + groups;
    rows = base + bytes(p.depth, width, groups);
  }
  static __host__ __device__ __forceinline__ int bytes(int depth, int width, int groups) { return ((int)sizeof(E) * (depth + 1) * width + groups * 8 + 15) & ~15; }
};

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_cluster(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) char norm_bytes[];
  typedef Vec<T, V> Vector;
  const NormShared<Moments, V> sh(p, norm_bytes);
  // (block, image, CTA of the cluster)
  NormPlace t = norm_place<V>(p, blockIdx.x / p.chunks % p.blocks + p.blocks * (blockIdx.x % p.chunks + p.chunks * (blockIdx.x / p.chunks / p.blocks)));
  const int width = p.lanes * V, groups = width / p.width, first = t.block * groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency();
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  T* out = (T*)p.out + t.n * p.S * p.C + t.channel;
  Vector* rows = (Vector*)sh.rows + t.depth * p.lanes + t.lane;  // of this thread
  NormMoments<V> m;
  if (t.in) {
    int i = 0;
    if (t.row < t.end) m.start(rows[0] = *(const Vector*)(x + t.row * p.C));
#pragma unroll 4
    for (long long r = t.row + p.depth; r < t.end; r += p.depth) m.add(rows[++i * p.depth * p.lanes] = *(const Vector*)(x + r * p.C));
  }
  Moments mine[V];
  m.get(mine);
  by_channel<V>(p, t, sh.told, mine, [&](const Moments* v, int w, int c, int) { sh.channels[c] = join_moments(v, w, p.depth, (int)(t.end - t.begin)); });
  if (p.chunks > 1) cluster_sync();
  else __syncthreads();
  // a warp per group: its channels of all CTAs
  const float all = (float)p.S * p.width;
  for (int g = warp; g < groups; g += kNormThreads / 32) {
    const int entries = p.chunks * p.width;
    const auto at = [&](int e, float& count) {
      const int rank = e / p.width;
      count = (float)max(0ll, min(p.rows, p.S - rank * p.rows));
      const Moments* from = sh.channels + g * p.width + (e - rank * p.width);
      return p.chunks > 1 ? of_cluster(from, rank) : *from;
    };
    float count, sum = 0.0f, m2 = 0.0f;
    const Moments pivot = at(0, count);
    for (int e = lane; e < entries; e += 32) {
      const Moments v = at(e, count);
      if (count > 0.0f) sum = fmaf(count, distance(v, pivot), sum);
    }
    const float shift = warp_sum(sum) / all, mean = pivot.mean + (pivot.rest + shift);
    for (int e = lane; e < entries; e += 32) {
      const Moments v = at(e, count);
      const float d = distance(v, pivot) - shift;
      if (count > 0.0f) m2 += fmaf(count * d, d, v.square);
    }
    m2 = warp_sum(m2);
    if (lane == 0) {
      const float rstd = 1.0f / sqrtf(m2 / all + p.eps);
      sh.first[g] = mean;
      sh.second[g] = rstd;
      if (t.chunk == 0) {
        p.mean[(long long)t.n * p.groups + first + g] = mean;
        p.rstd[(long long)t.n * p.groups + first + g] = rstd;
      }
    }
  }
  __syncthreads();
  const NormChannels<V> c(p, t, sh.first, sh.second, first);
  if (t.in) {
    int i = 0;
    for (long long r = t.row; r < t.end; r += p.depth) *(Vector*)(out + r * p.C) = normalised<T, ACT>(rows[i++ * p.depth * p.lanes], c);
  }
  if (p.chunks > 1) cluster_sync();  // (no CTA ends while another reads its shared memory)
}

// ---- backward -----------------------------------------------------------------------------------------
template <typename T, int ACT, int V>
__device__ __forceinline__ void add_slopes(float2 (&sums)[V], const Vec<T, V>& x, const Vec<T, V>& dy, const NormChannels<V>& c) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float xhat = (to_float(x.v[k]) - c.mean[k]) * c.rstd[k];
    float slope;
    activate<T, ACT>(fmaf(xhat, c.weight[k], c.bias[k]), slope);
    const float dz = to_float(dy.v[k]) * slope;
    sums[k].x += dz;
    sums[k].y = fmaf(dz, xhat, sums[k].y);
  }
}
template <typename T, int ACT, int V>
__device__ __forceinline__ Vec<T, V> input_gradient(const Vec<T, V>& x, const Vec<T, V>& dy, const NormChannels<V>& c, const float2 (&m)[V]) {
  Vec<T, V> o;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float xhat = (to_float(x.v[k]) - c.mean[k]) * c.rstd[k];
    float slope;
    activate<T, ACT>(fmaf(xhat, c.weight[k], c.bias[k]), slope);
    o.v[k] = from_float<T>(c.rstd[k] * (fmaf(to_float(dy.v[k]) * slope, c.weight[k], -m[k].x) - xhat * m[k].y));
  }
  return o;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_sums(const __grid_constant__ NormParams p) {
  extern __shared__ float2 norm_shared[];
  grid_dependency();
  const NormPlace t = norm_place<V>(p, blockIdx.x);
  const NormChannels<V> c(p, t, p.mean + (long long)t.n * p.groups, p.rstd + (long long)t.n * p.groups, 0);
  typedef Vec<T, V> Vector;
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  const T* dy = (const T*)p.dy + t.n * p.S * p.C + t.channel;
  float2 mine[V] = {};
  if (t.in) {
#pragma unroll 2
    for (long long r = t.row; r < t.end; r += p.depth) add_slopes<T, ACT>(mine, *(const Vector*)(x + r * p.C), *(const Vector*)(dy + r * p.C), c);
  }
  by_channel<V>(p, t, norm_shared, mine, [&](const float2* v, int width, int, int channel) {
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = 0; i < p.depth; ++i) s = add2(s, v[i * width]);
    p.part[((long long)t.n * p.chunks + t.chunk) * p.C + channel] = s;
  });
}

// A group's m1 and m2 of an image (the first N * groups CTAs, if `means`), and 32 channels' gradients of weights and biases over all
// images' chunks (the others).
static __global__ void __launch_bounds__(kNormThreads) norm_sums_finish(const __grid_constant__ NormParams p, int group_ctas) {
  __shared__ float shared[kNormThreads / 32];
  __shared__ float2 totals[kNormThreads];
  grid_dependency();
  if ((int)blockIdx.x < group_ctas) {
    const int n = blockIdx.x / p.groups, g = blockIdx.x - n * p.groups, entries = p.chunks * p.width;
    const float2* part = p.part + (long long)n * p.chunks * p.C + g * p.width;
    float2 s = make_float2(0.0f, 0.0f);
    for (int e = threadIdx.x; e < entries; e += kNormThreads) {
      const int chunk = e / p.width, c = e - chunk * p.width;
      const float w = weight_of(p, g * p.width + c);
      s = fma2(make_float2(w, w), part[(long long)chunk * p.C + c], s);
    }
    const float all = (float)p.S * p.width, m1 = norm_sum(s.x, shared), m2 = norm_sum(s.y, shared);
    if (threadIdx.x == 0) p.means[blockIdx.x] = make_float2(m1 / all, m2 / all);
    return;
  }
  const int channel = (blockIdx.x - group_ctas) * 32 + (threadIdx.x & 31);
  const long long entries = (long long)p.N * p.chunks;
  float2 s = make_float2(0.0f, 0.0f);
  if (channel < p.C) {
#pragma unroll 8
    for (long long e = threadIdx.x >> 5; e < entries; e += kNormThreads / 32) s = add2(s, p.part[e * p.C + channel]);
  }
  totals[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || channel >= p.C) return;
  for (int i = 1; i < kNormThreads / 32; ++i) s = add2(s, totals[i * 32 + threadIdx.x]);
  if (p.dweight) put_parameter(p, p.dweight, channel, s.y);
  if (p.dbias) put_parameter(p, p.dbias, channel, s.x);
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_dx(const __grid_constant__ NormParams p) {
  grid_dependency();
  const NormPlace t = norm_place<V>(p, blockIdx.x, true);
  const NormChannels<V> c(p, t, p.mean + (long long)t.n * p.groups, p.rstd + (long long)t.n * p.groups, 0);
  if (!t.in) return;
  float2 m[V];
#pragma unroll
  for (int k = 0; k < V; ++k) m[k] = p.means[(long long)t.n * p.groups + (t.channel + k) / p.width];
  typedef Vec<T, V> Vector;
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  const T* dy = (const T*)p.dy + t.n * p.S * p.C + t.channel;
  T* dx = (T*)p.dx + t.n * p.S * p.C + t.channel;
#pragma unroll 2
  for (long long r = t.row; r < t.end; r += p.depth)
    *(Vector*)(dx + r * p.C) = input_gradient<T, ACT>(*(const Vector*)(x + r * p.C), *(const Vector*)(dy + r * p.C), c, m);
}

// All of a block of groups: dx, and the block's channels' sums of the image (p.part, a chunk an image).
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_cluster_backward(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) char norm_bytes[];
  typedef Vec<T, V> Vector;
  const NormShared<float2, V> sh(p, norm_bytes);
  NormPlace t = norm_place<V>(p, blockIdx.x / p.chunks % p.blocks + p.blocks * (blockIdx.x % p.chunks + p.chunks * (blockIdx.x / p.chunks / p.blocks)));
  const int width = p.lanes * V, groups = width / p.width, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency();
  const NormChannels<V> c(p, t, p.mean + (long long)t.n * p.groups, p.rstd + (long long)t.n * p.groups, 0);
  const T* x = (const T*)p.x + t.n * p.S * p.C + t.channel;
  const T* dy = (const T*)p.dy + t.n * p.S * p.C + t.channel;
  T* dx = (T*)p.dx + t.n * p.S * p.C + t.channel;
  Vector* rows = (Vector*)sh.rows + (t.depth * p.lanes + t.lane) * 2;  // of this thread: x and dy
  const int step = p.depth * p.lanes * 2;
  float2 mine[V] = {};
  if (t.in) {
    int i = 0;
#pragma unroll 2
    for (long long r = t.row; r < t.end; r += p.depth, ++i)
      add_slopes<T, ACT>(mine, rows[i * step] = *(const Vector*)(x + r * p.C), rows[i * step + 1] = *(const Vector*)(dy + r * p.C), c);
  }
  by_channel<V>(p, t, sh.told, mine, [&](const float2* v, int w, int at, int) {
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = 0; i < p.depth; ++i) s = add2(s, v[i * w]);
    sh.channels[at] = s;
  });
  if (p.chunks > 1) cluster_sync();
  else __syncthreads();
  const float all = (float)p.S * p.width;
  for (int g = warp; g < groups; g += kNormThreads / 32) {
    float2 sum = make_float2(0.0f, 0.0f);
    for (int k = lane; k < p.width; k += 32) {
      const int at = g * p.width + k, channel = t.block * width + at;
      float2 s = make_float2(0.0f, 0.0f);
      for (int rank = 0; rank < p.chunks; ++rank) s = add2(s, p.chunks > 1 ? of_cluster(sh.channels + at, rank) : sh.channels[at]);
      if (t.chunk == 0) p.part[(long long)t.n * p.C + channel] = s;
      const float w = weight_of(p, channel);
      sum = fma2(make_float2(w, w), s, sum);
    }
    const float m1 = warp_sum(sum.x), m2 = warp_sum(sum.y);
    if (lane == 0) {
      sh.first[g] = m1 / all;
      sh.second[g] = m2 / all;
    }
  }
  __syncthreads();
  if (t.in) {
    float2 m[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int g = (t.channel + k) / p.width - t.block * groups;
      m[k] = make_float2(sh.first[g], sh.second[g]);
    }
    int i = 0;
    for (long long r = t.row; r < t.end; r += p.depth, ++i) *(Vector*)(dx + r * p.C) = input_gradient<T, ACT>(rows[i * step], rows[i * step + 1], c, m);
  }
  if (p.chunks > 1) cluster_sync();
}

}  // namespace mvr
