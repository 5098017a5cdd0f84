// C ABI of an encoder block's operators beside attention (declared in include/mvr.h): group norm with its activation, rotary positions.
// Argument checks, kernel selection and launches; no torch types, device pointers and sizes only.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <numeric>

#include "../../include/mvr.h"
#include "mvr_norm.cuh"
#include "mvr_rotary.cuh"

namespace {

using namespace mvr;

bool element_type(int t) { return t == MVR_F32 || t == MVR_F16 || t == MVR_BF16; }
int size_of(int t) { return t == MVR_F32 ? 4 : 2; }
int launched() { return cudaGetLastError() == cudaSuccess ? MVR_OK : MVR_ERR_LAUNCH; }
long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

constexpr int kMultiprocessors = 148;

// ---- group norm ---------------------------------------------------------------------------------------

// How a call is cut: by clusters of `chunks` CTAs, each with its rows in shared memory, or in passes over chunks of rows.
struct NormCut {
  bool clusters, whole;  // whole: every vector lies in one group
  int V, block_groups, blocks, columns, lanes, depth, chunks;
  long long rows;
  size_t shared;
  long long sums, slopes, bytes;
};

// Whether rows can be taken in vectors of V channels: a block of whole groups and whole vectors is one group, or fits a CTA's threads.
bool vectors_fit(const mvr_group_norm* a, int V) {
  const long long width = a->C / a->groups, groups = V / std::gcd(width, (long long)V);
  return a->C % V == 0 && (groups == 1 || groups * width / V <= kNormThreads);
}
int vector_of(const mvr_group_norm* a, bool backward) {
  uintptr_t all = (uintptr_t)a->x | (uintptr_t)(backward ? a->grad_x : a->out);
  if (backward) all |= (uintptr_t)a->grad_out;
  const int whole = 16 / size_of(a->dtype);
  if (vectors_fit(a, whole) && all % 16 == 0) return whole;
  if (whole == 8 && vectors_fit(a, 4) && all % 8 == 0) return 4;
  return 1;
}

constexpr size_t kNormShared = 200 * 1024;

NormCut cut_norm(const mvr_group_norm* a, bool backward, int V) {
  NormCut c = {};
  c.V = V;
  const int width = (int)(a->C / a->groups), element = size_of(a->dtype), operands = backward ? 2 : 1;
  c.whole = width % V == 0;
  const int told = backward ? V * (int)sizeof(float2) : (c.whole ? 1 : V) * (int)sizeof(Moments);  // bytes of a thread's sums
  const double bytes = (double)a->N * a->S * a->C * element;
  // Times in us, measured from 0.5 to 268 MB of x.  Passes: 8.5 + 0.43 a MB (0.54 beyond L2), backward 9 + 1.0 (float: 0.65).  Clusters: 2 (4),
  // 1.3 more where CTAs tell each other their sums, and for each wave 2.2 (3) and 0.06 a KB that an SM brings into shared memory (pieces of
  // a row below 32 bytes: 0.1).  A wave: two CTAs an SM, of clusters of 4 and 8 as many as 128 and 96 SMs hold.  (2 x 4096 rows of 128 halves:
  // clusters 7.2, passes 10.3; 2 x 32768 of 64: 13.2, 11.4; 8 x 1000 of 512: 8.0, 12.0.)
  double least = backward ? 9 + bytes * (element == 2 ? 1.0e-6 : 0.65e-6) : 8.5 + bytes * (bytes < 60e6 ? 0.43e-6 : 0.54e-6);
  for (int groups = 1; groups <= a->groups; ++groups) {
    const long long channels = (long long)groups * width;
    if (channels / V > kNormThreads) break;
    if (a->groups % groups != 0 || channels % V != 0) continue;
    for (int size = 1; size <= 8; size *= 2) {
      const long long rows = cdiv(a->S, size);
      const int lanes = (int)(channels / V), depth = (int)std::min<long long>(kNormThreads / lanes, rows);
      const long long data = cdiv(rows, depth) * depth * channels * element * operands, ctas = a->N * (a->groups / groups) * size;
      if (data > (long long)kNormShared || ctas > INT32_MAX) continue;
      const size_t shared = (size_t)(NormShared::bytes(depth * lanes * told, groups) + data);
      if (shared > kNormShared || (size > 1 && (size - 1) * rows >= a->S)) continue;
      const int multiprocessors = size == 8 ? 96 : size == 4 ? 128 : kMultiprocessors;
      const long long on_sm = cdiv(ctas, multiprocessors), resident = std::min<long long>(2, 220 * 1024 / (long long)(shared + 1024));
      const double time = (backward ? 4 : 2) + (size > 1 ? 1.3 : 0) + (double)cdiv(on_sm, resident) * (backward ? 3 : 2.2) +
                          (double)on_sm * data * (channels * element < 32 ? 0.1e-3 : 0.06e-3);
      if (time < least) {
        least = time;
        c.clusters = true;
        c.block_groups = groups;
        c.lanes = c.columns = lanes;
        c.depth = depth;
        c.chunks = size;
        c.rows = rows;
        c.shared = shared;
      }
    }
  }
  if (!c.clusters) {
    // blocks of up to 512 bytes of a row, if groups are not wider, and 64 groups
    for (int groups = 1; groups <= a->groups; ++groups) {
      if (a->groups % groups != 0 || (long long)groups * width % V != 0) continue;
      if (c.block_groups > 0 && (groups > 64 || (long long)groups * width * element > 512)) break;
      c.block_groups = groups;
    }
    c.columns = (int)((long long)c.block_groups * width / V);
    c.lanes = std::min(c.columns, kNormThreads);
    c.depth = kNormThreads / c.lanes;
    // all CTAs at once, two an SM, each with two rows a thread at least; and no more sums than a CTA of the second pass can look at
    const long long blocks = a->groups / c.block_groups, all = std::max<long long>(1, 2 * kMultiprocessors / std::max<long long>(1, a->N * blocks));
    c.chunks = (int)std::max<long long>(1, std::min({all, cdiv(a->S, 2 * c.depth), 8192LL / c.block_groups}));
    c.rows = cdiv(std::max<long long>(1, a->S), c.chunks);
    c.chunks = (int)std::max<long long>(1, cdiv(a->S, c.rows));
    c.shared = (size_t)c.depth * c.lanes * told;
  }
  c.blocks = (int)(a->groups / c.block_groups);
  long long at = 0;
  const auto take = [&at](long long n) {
    const long long here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  if (!c.clusters) c.sums = take(a->N * c.chunks * a->groups * (backward ? 8 : 16));
  if (backward) c.slopes = take(a->N * (c.clusters ? 1 : c.chunks) * a->C * 8);
  c.bytes = at;
  return c;
}

int check_norm(const mvr_group_norm* a, bool backward, bool sizes_only) {
  if (!a) return MVR_ERR_NULL;
  if (!element_type(a->dtype) || (a->parameter_dtype != MVR_F32 && a->parameter_dtype != a->dtype)) return MVR_ERR_DTYPE;
  if (a->N < 0 || a->S < 0 || a->C < 1) return MVR_ERR_SHAPE;
  if (a->groups < 1 || a->C % a->groups != 0) return MVR_ERR_GROUPS;
  if (a->activation < MVR_ACT_NONE || a->activation > MVR_ACT_GELU) return MVR_ERR_ACTIVATION;
  if (!(a->eps >= 0.0f)) return MVR_ERR_SHAPE;
  if (a->C > 1 << 20 || a->N > INT32_MAX / 64 || (a->N > 0 && a->C * a->N > INT32_MAX) || a->S > (1LL << 40)) return MVR_ERR_TOO_LARGE;
  if (a->S > 0 && a->N > 0 && a->S > INT64_MAX / 64 / a->C / a->N) return MVR_ERR_TOO_LARGE;
  if (sizes_only) return MVR_OK;
  const bool any = a->N > 0 && a->S > 0;
  if (any && (!a->x || !a->mean || !a->rstd || (backward ? !a->grad_out || !a->grad_x : !a->out))) return MVR_ERR_NULL;
  return MVR_OK;
}

NormParams norm_params(const mvr_group_norm* a, const NormCut& c, char* ws) {
  NormParams p = {};
  p.x = a->x; p.dy = a->grad_out; p.weight = a->weight; p.bias = a->bias;
  p.out = a->out; p.dx = a->grad_x; p.dweight = a->grad_weight; p.dbias = a->grad_bias;
  p.mean = a->mean; p.rstd = a->rstd; p.rest = a->mean_rest;
  p.moments = (Moments*)(ws + c.sums); p.sums = (float2*)(ws + c.sums); p.slopes = (float2*)(ws + c.slopes);
  p.S = a->S; p.rows = c.rows;
  p.N = (int)a->N; p.C = (int)a->C; p.groups = (int)a->groups; p.width = (int)(a->C / a->groups);
  p.parameters = a->parameter_dtype;
  p.by_width.set((unsigned)p.width);
  p.chunks = c.chunks; p.blocks = c.blocks; p.block_groups = c.block_groups; p.columns = c.columns; p.lanes = c.lanes; p.depth = c.depth;
  p.eps = a->eps;
  return p;
}

// Lets a kernel have as much shared memory as any call of it asks for, once per device, and launches it, in clusters of `size` CTAs.
template <auto KERNEL>
int launch_norm(const NormParams& p, long long ctas, size_t shared, int size, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MVR_ERR_LAUNCH;
  const uint64_t bit = 1ull << (device & 63);
  if (device >= 64 || !(done.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNormShared) != cudaSuccess) {
      cudaGetLastError();
      return MVR_ERR_LAUNCH;
    }
    if (device < 64) done.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kNormThreads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, KERNEL, p);
  return launched();
}

template <typename T, int V, bool WHOLE, int ACT>
int norm_as(NormParams& p, const NormCut& c, bool backward, cudaStream_t st) {
  const long long ctas = (long long)p.N * c.chunks * c.blocks;
  const int channel_ctas = p.dweight || p.dbias ? (int)cdiv(p.C, 32) : 0;
  // (the second passes: three numbers a group, or two, and what the threads have joined)
  const size_t joined = std::max<size_t>(kNormThreads, c.block_groups), groups = (size_t)c.block_groups * 12 + 16;
  int rc;
  if (!backward) {
    if (c.clusters) return launch_norm<norm_cluster<T, V, WHOLE, ACT>>(p, ctas, c.shared, c.chunks, st);
    rc = launch_norm<norm_stats<T, V, WHOLE>>(p, ctas, c.shared, 1, st);
    return rc != MVR_OK ? rc : launch_norm<norm_apply<T, V, WHOLE, ACT>>(p, ctas, groups + joined * sizeof(Moments), 1, st);
  }
  if (c.clusters) {
    rc = launch_norm<norm_cluster_backward<T, V, WHOLE, ACT>>(p, ctas, c.shared, c.chunks, st);
    if (rc != MVR_OK || channel_ctas == 0) return rc;
    p.chunks = 1;
    launch_dependent(norm_parameters, dim3((unsigned)channel_ctas), dim3(kNormThreads), 0, st, p);
    return launched();
  }
  rc = launch_norm<norm_sums<T, V, WHOLE, ACT>>(p, ctas, c.shared, 1, st);
  p.channel_ctas = channel_ctas;
  return rc != MVR_OK ? rc : launch_norm<norm_dx<T, V, WHOLE, ACT>>(p, ctas + channel_ctas, groups + joined * sizeof(float2), 1, st);
}
template <typename T, int V, int ACT>
int norm_as(NormParams& p, const NormCut& c, bool backward, cudaStream_t st) {
  if constexpr (V > 1)
    if (!c.whole) return norm_as<T, V, false, ACT>(p, c, backward, st);
  return norm_as<T, V, true, ACT>(p, c, backward, st);
}
template <typename T, int V>
int norm_with(NormParams& p, const NormCut& c, int activation, bool backward, cudaStream_t st) {
  switch (activation) {
    case MVR_ACT_NONE: return norm_as<T, V, kNoActivation>(p, c, backward, st);
    case MVR_ACT_RELU: return norm_as<T, V, kRelu>(p, c, backward, st);
    case MVR_ACT_SILU: return norm_as<T, V, kSilu>(p, c, backward, st);
    default: return norm_as<T, V, kGelu>(p, c, backward, st);
  }
}

long long norm_bytes(const mvr_group_norm* a, bool backward) {
  // (the vector is a matter of the call's addresses)
  long long most = 0;
  for (int V : {1, 4, 8})
    if (V * size_of(a->dtype) <= 16 && vectors_fit(a, V)) most = std::max(most, cut_norm(a, backward, V).bytes);
  return most;
}

int group_norm(const mvr_group_norm* a, bool backward, void* workspace, int64_t bytes, void* stream) {
  const int rc = check_norm(a, backward, false);
  if (rc != MVR_OK) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a->N == 0 || a->S == 0) {
    if (!backward) return MVR_OK;
    for (void* to : {a->grad_weight, a->grad_bias})  // sums of nothing
      if (to && cudaMemsetAsync(to, 0, (size_t)a->C * size_of(a->parameter_dtype), st) != cudaSuccess) {
        cudaGetLastError();
        return MVR_ERR_LAUNCH;
      }
    return MVR_OK;
  }
  const int V = vector_of(a, backward);
  const NormCut c = cut_norm(a, backward, V);
  if (bytes < c.bytes || (c.bytes > 0 && !workspace)) return MVR_ERR_WORKSPACE;
  if ((long long)a->N * c.chunks * c.blocks > INT32_MAX - (1 << 16)) return MVR_ERR_TOO_LARGE;
  NormParams p = norm_params(a, c, (char*)workspace);
  switch (a->dtype) {
    case MVR_F32: return V == 4 ? norm_with<float, 4>(p, c, a->activation, backward, st) : norm_with<float, 1>(p, c, a->activation, backward, st);
    case MVR_F16:
      return V == 8 ? norm_with<__half, 8>(p, c, a->activation, backward, st) : V == 4 ? norm_with<__half, 4>(p, c, a->activation, backward, st)
                                                                                : norm_with<__half, 1>(p, c, a->activation, backward, st);
    default:
      return V == 8 ? norm_with<__nv_bfloat16, 8>(p, c, a->activation, backward, st)
             : V == 4 ? norm_with<__nv_bfloat16, 4>(p, c, a->activation, backward, st) : norm_with<__nv_bfloat16, 1>(p, c, a->activation, backward, st);
  }
}

// ---- rotary positions ---------------------------------------------------------------------------------

int check_rotary(const mvr_rotary* a) {
  if (!a) return MVR_ERR_NULL;
  if (!element_type(a->dtype)) return MVR_ERR_DTYPE;
  if (a->N < 0 || a->L < 0 || a->D < 1 || a->heads[0] < 1 || a->heads[1] < 0) return MVR_ERR_SHAPE;
  if (a->axes < 1 || a->axes > MVR_MAX_AXES) return MVR_ERR_AXES;
  long long pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0) return MVR_ERR_AXES;
    pairs += a->sections[i];
    if (2 * pairs > a->D) return MVR_ERR_AXES;
  }
  if (pairs > kRotaryPairs) return MVR_ERR_HEAD_SIZE;
  if (!(a->base >= 1.0) || !std::isfinite(a->base)) return MVR_ERR_AXES;
  if (a->position_dtype != MVR_INDEX_F32 && a->position_dtype != MVR_INDEX_I32 && a->position_dtype != MVR_INDEX_I64) return MVR_ERR_DTYPE;
  if (a->D > 1 << 14 || a->heads[0] > 1 << 16 || a->heads[1] > 1 << 16 || a->L > 1 << 30 || a->N > INT32_MAX) return MVR_ERR_TOO_LARGE;
  if (a->N == 0 || a->L == 0) return MVR_OK;
  if (a->N * a->L > (1LL << 40)) return MVR_ERR_TOO_LARGE;
  for (int i = 0; i < 2; ++i)
    for (int k = 1; k < 3; ++k)
      if (a->heads[i] > 0 && (a->strides[i][k] > INT32_MAX || a->strides[i][k] < INT32_MIN)) return MVR_ERR_TOO_LARGE;
  if (!a->x[0] || !a->out[0] || (a->heads[1] > 0 && (!a->x[1] || !a->out[1])) || !a->positions) return MVR_ERR_NULL;
  return MVR_OK;
}

template <typename T>
int rotary_as(RotaryParams& p, const mvr_rotary* a, cudaStream_t st) {
  // vectors of 16 bytes, where rows and addresses allow them
  constexpr int V = 16 / (int)sizeof(T);
  bool vectors = a->D % V == 0;
  for (int i = 0; i < 2; ++i) {
    if (a->heads[i] == 0) continue;
    vectors = vectors && ((uintptr_t)a->x[i] | (uintptr_t)a->out[i]) % 16 == 0;
    const int64_t sizes[3] = {a->N, a->L, a->heads[i]};
    for (int k = 0; k < 3; ++k) vectors = vectors && (sizes[k] == 1 || a->strides[i][k] % V == 0);
  }
  const int N = (int)a->N;
  const bool good = !vectors ? launch_rotary<T, 1, kScalar>(p, N, a->interleaved, st) : a->interleaved ? launch_rotary<T, V, kNeighbour>(p, N, true, st)
                    : p.pairs % V == 0 ? launch_rotary<T, V, kApart>(p, N, false, st) : launch_rotary<T, V, kOwn>(p, N, false, st);
  return good ? MVR_OK : MVR_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int mvr_group_norm_workspace(const mvr_group_norm* a, int backward, int64_t* bytes) {
  if (!bytes) return MVR_ERR_NULL;
  const int rc = check_norm(a, backward != 0, true);
  if (rc != MVR_OK) return rc;
  *bytes = a->N == 0 || a->S == 0 ? 0 : norm_bytes(a, backward != 0);
  return MVR_OK;
}

int mvr_group_norm_forward(const mvr_group_norm* a, void* workspace, int64_t bytes, void* stream) { return group_norm(a, false, workspace, bytes, stream); }

int mvr_group_norm_backward(const mvr_group_norm* a, void* workspace, int64_t bytes, void* stream) { return group_norm(a, true, workspace, bytes, stream); }

int mvr_rotary_positions(const mvr_rotary* a, void* stream) {
  const int rc = check_rotary(a);
  if (rc != MVR_OK) return rc;
  if (a->N == 0 || a->L == 0) return MVR_OK;
  RotaryParams p = {};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = a->x[i];
    p.out[i] = a->out[i];
    p.heads[i] = (int)a->heads[i];
    p.s_n[i] = a->strides[i][0]; p.s_l[i] = (int)a->strides[i][1]; p.s_h[i] = (int)a->strides[i][2];
  }
  p.positions = a->positions;
  p.position_type = a->position_dtype == MVR_INDEX_F32 ? 0 : a->position_dtype == MVR_INDEX_I32 ? 1 : 2;
  p.p_n = a->position_strides[0]; p.p_l = a->position_strides[1]; p.p_a = a->position_strides[2];
  p.L = (int)a->L;
  p.D = (int)a->D;
  p.sign = a->inverse ? -1.0f : 1.0f;
  for (int i = 0; i < kRotaryAxes; ++i) {
    const int n = i < a->axes ? (int)a->sections[i] : 0;
    // 1 / 2 pi times powers of base^(-1 / n), in 2^-64 (and what lies below): by whole-number products, since a call of powl for each, and
    // conversions from long double, take longer than the kernel of a few tokens
    const long double ratio = n > 1 ? powl(a->base, -1.0L / n) : 1.0L;
    const unsigned __int128 factor = ratio < 1.0L ? (unsigned __int128)(unsigned long long)(ratio * 18446744073709551616.0L) : (unsigned __int128)1 << 64;
    unsigned long long turns = 0x28be60db9391054aull, below = 0x7f09d5f47d4d3770ull;
    for (int k = 0; k < n; ++k) {
      p.turns[p.pairs + k] = turns;
      const unsigned __int128 next = turns * factor + ((below * factor) >> 64);
      turns = (unsigned long long)(next >> 64);
      below = (unsigned long long)next;
    }
    p.ends[i] = p.pairs += n;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == MVR_F32 ? rotary_as<float>(p, a, st) : a->dtype == MVR_F16 ? rotary_as<__half>(p, a, st) : rotary_as<__nv_bfloat16>(p, a, st);
}

}  // extern "C"
