// C ABI of an encoder block's operators beside attention (declared in include/mvr.h): group norm with its activation, rotary positions.
// Argument checks, kernel selection and launches; no torch types, device pointers and sizes only.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>

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
  bool clusters;
  int V, columns, lanes, depth, blocks, chunks;
  long long rows;
  size_t shared;
  long long part, means, bytes;
};

int vector_of(const mvr_group_norm* a, bool backward) {
  uintptr_t all = (uintptr_t)a->x | (uintptr_t)(backward ? a->grad_x : a->out);
  if (backward) all |= (uintptr_t)a->grad_out;
  const int whole = 16 / size_of(a->dtype);
  if (a->C % whole == 0 && all % 16 == 0) return whole;
  if (whole == 8 && a->C % 4 == 0 && all % 8 == 0) return 4;
  return 1;
}

constexpr size_t kNormShared = 200 * 1024;

NormCut cut_norm(const mvr_group_norm* a, bool backward, int V) {
  NormCut c = {};
  c.V = V;
  c.columns = (int)(a->C / V);
  const int width = (int)(a->C / a->groups), elements = backward ? 2 : 1, entry = (int)(backward ? sizeof(float2) : sizeof(Moments));
  const double bytes = (double)a->N * a->S * a->C * size_of(a->dtype);
  // Passes: 3 launches, and memory at some 5 MB/us; the second read finds what fits L2.
  double least = 7 + bytes * (backward ? 3 : 2) / 5e6 + bytes * elements / (bytes * elements < 80e6 ? 10e6 : 5e6);
  for (int groups = 1; groups <= a->groups; ++groups) {
    const long long channels = (long long)groups * width;
    if (a->groups % groups != 0 || channels % V != 0 || channels / V > kNormThreads) continue;
    for (int size = 1; size <= 8; size *= 2) {
      const int lanes = (int)(channels / V), depth = (int)std::min<long long>(kNormThreads / lanes, std::max<long long>(1, cdiv(a->S, size)));
      const long long rows = cdiv(a->S, size), data = cdiv(rows, depth) * depth * lanes * V * size_of(a->dtype) * elements;
      const size_t shared = (size_t)(((depth + 1) * channels * entry + groups * 8 + 15) / 16 * 16 + data);
      if (shared > kNormShared || (size > 1 && rows < 2 * depth)) continue;
      const long long ctas = a->N * (a->groups / groups) * size;
      if (ctas > INT32_MAX) continue;
      // An SM's CTAs together take a wave; each waits some 3 us for its loads and its group's sums, 1.5 more in a cluster.  Row pieces below
      // 64 bytes use the memory badly.
      const int resident = (int)std::min<long long>(8, 220 * 1024 / (long long)(shared + 1024));
      const double waves = std::max(1.0, (double)ctas / (kMultiprocessors * resident)), piece = (double)channels * size_of(a->dtype);
      const double time = 2 + std::ceil(waves) * (3 + (size > 1 ? 1.5 : 0)) +
                          std::max(bytes * (elements + 1) / 5e6, waves * resident * (double)data * (elements + 1) / elements / 40e3) * (piece < 32 ? 2 : piece < 64 ? 1.3 : 1);
      if (time < least) {
        least = time;
        c.clusters = true;
        c.lanes = lanes;
        c.depth = depth;
        c.blocks = (int)(a->groups / groups);
        c.chunks = size;
        c.rows = rows;
        c.shared = shared;
      }
    }
  }
  if (!c.clusters) {
    c.lanes = std::min(c.columns, kNormThreads);
    c.depth = kNormThreads / c.lanes;
    c.blocks = (int)cdiv(c.columns, c.lanes);
    // some six CTAs an SM, each with four rows a thread at least
    const long long most = std::max<long long>(1, cdiv(a->S, 4 * c.depth)), want = cdiv(6 * kMultiprocessors, std::max<long long>(1, a->N * c.blocks));
    c.chunks = (int)std::min<long long>({most, std::max<long long>(1, want), 1 << 16});
    c.rows = cdiv(std::max<long long>(1, a->S), c.chunks);
    c.chunks = (int)std::max<long long>(1, cdiv(a->S, c.rows));
    c.shared = (size_t)c.depth * c.lanes * V * entry;
  }
  long long at = 0;
  const auto take = [&at](long long n) {
    const long long here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  if (!c.clusters || backward) c.part = take(a->N * (c.clusters ? 1 : c.chunks) * a->C * entry);
  if (!c.clusters && backward) c.means = take(a->N * a->groups * 8);
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
  p.mean = a->mean; p.rstd = a->rstd;
  p.moments = (Moments*)(ws + c.part); p.part = (float2*)(ws + c.part); p.means = (float2*)(ws + c.means);
  p.S = a->S; p.rows = c.rows;
  p.N = (int)a->N; p.C = (int)a->C; p.groups = (int)a->groups; p.width = (int)(a->C / a->groups);
  p.parameters = a->parameter_dtype;
  p.chunks = c.chunks; p.columns = c.columns; p.lanes = c.lanes; p.depth = c.depth; p.blocks = c.blocks;
  p.eps = a->eps;
  return p;
}

// A kernel of clusters, with as much shared memory as it asks for (the limit is raised once per device).
template <auto KERNEL>
int launch_cluster(const NormParams& p, const NormCut& c, cudaStream_t st) {
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
  cfg.gridDim = dim3((unsigned)((long long)p.N * c.blocks * c.chunks));
  cfg.blockDim = dim3(kNormThreads);
  cfg.dynamicSmemBytes = c.shared;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = c.chunks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, KERNEL, p);
  return launched();
}

template <typename T, int V, int ACT>
int norm_as(const NormParams& p, const NormCut& c, bool backward, cudaStream_t st) {
  const dim3 grid((unsigned)((long long)p.N * c.chunks * c.blocks)), threads(kNormThreads);
  const int group_ctas = p.N * p.groups, channel_ctas = p.dweight || p.dbias ? (int)cdiv(p.C, 32) : 0;
  if (!backward) {
    if (c.clusters) return launch_cluster<norm_cluster<T, V, ACT>>(p, c, st);
    launch_dependent(norm_stats<T, V>, grid, threads, c.shared, st, p);
    launch_dependent(norm_finish, dim3((unsigned)group_ctas), threads, 0, st, p);
    launch_dependent(norm_apply<T, V, ACT>, grid, threads, 0, st, p);
    return launched();
  }
  if (c.clusters) {
    const int rc = launch_cluster<norm_cluster_backward<T, V, ACT>>(p, c, st);
    if (rc != MVR_OK || channel_ctas == 0) return rc;
    NormParams sums = p;
    sums.chunks = 1;
    launch_dependent(norm_sums_finish, dim3((unsigned)channel_ctas), threads, 0, st, sums, 0);
    return launched();
  }
  launch_dependent(norm_sums<T, V, ACT>, grid, threads, c.shared, st, p);
  launch_dependent(norm_sums_finish, dim3((unsigned)(group_ctas + channel_ctas)), threads, 0, st, p, group_ctas);
  launch_dependent(norm_dx<T, V, ACT>, grid, threads, 0, st, p);
  return launched();
}
template <typename T, int V>
int norm_with(const NormParams& p, const NormCut& c, int activation, bool backward, cudaStream_t st) {
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
    if (V * size_of(a->dtype) <= 16 && a->C % V == 0) most = std::max(most, cut_norm(a, backward, V).bytes);
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
  if ((long long)a->N * c.chunks * c.blocks > INT32_MAX) return MVR_ERR_TOO_LARGE;
  const NormParams p = norm_params(a, c, (char*)workspace);
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
  if (!(a->base > 0.0) || !std::isfinite(a->base)) return MVR_ERR_AXES;
  if (a->position_dtype != MVR_INDEX_F32 && a->position_dtype != MVR_INDEX_I32 && a->position_dtype != MVR_INDEX_I64) return MVR_ERR_DTYPE;
  if (a->D > 1 << 20 || a->heads[0] > 1 << 20 || a->heads[1] > 1 << 20 || a->L > INT32_MAX || a->N > INT32_MAX) return MVR_ERR_TOO_LARGE;
  if (a->N == 0 || a->L == 0) return MVR_OK;
  if (a->N * a->L > (1LL << 40)) return MVR_ERR_TOO_LARGE;
  if (!a->x[0] || !a->out[0] || (a->heads[1] > 0 && (!a->x[1] || !a->out[1])) || !a->positions) return MVR_ERR_NULL;
  return MVR_OK;
}

template <typename T>
int rotary_as(RotaryParams& p, const mvr_rotary* a, cudaStream_t st) {
  // the widest vector that columns, rows and addresses allow
  int V = 16 / (int)sizeof(T);
  for (; V > 1; V /= 2) {
    bool good = a->D % V == 0 && (a->interleaved ? 2 * p.pairs : p.pairs) % V == 0;
    for (int i = 0; i < 2; ++i) {
      if (a->heads[i] == 0) continue;
      good = good && ((uintptr_t)a->x[i] | (uintptr_t)a->out[i]) % (V * sizeof(T)) == 0;
      const int64_t sizes[3] = {a->N, a->L, a->heads[i]};
      for (int k = 0; k < 3; ++k) good = good && (sizes[k] == 1 || a->strides[i][k] % V == 0);
    }
    if (good) break;
  }
  int rc;
  switch (V) {
    case 8: if constexpr (sizeof(T) == 2) { rc = launch_rotary<T, 8>(p, a->interleaved, st); break; }
    case 4: rc = launch_rotary<T, 4>(p, a->interleaved, st); break;
    case 2: rc = launch_rotary<T, 2>(p, a->interleaved, st); break;
    default: rc = launch_rotary<T, 1>(p, a->interleaved, st);
  }
  return rc ? MVR_ERR_TOO_LARGE : launched();
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
    p.s_n[i] = a->strides[i][0]; p.s_l[i] = a->strides[i][1]; p.s_h[i] = a->strides[i][2];
  }
  p.positions = a->positions;
  p.position_type = a->position_dtype == MVR_INDEX_F32 ? 0 : a->position_dtype == MVR_INDEX_I32 ? 1 : 2;
  p.p_n = a->position_strides[0]; p.p_l = a->position_strides[1]; p.p_a = a->position_strides[2];
  p.tokens = a->N * a->L;
  p.L = (int)a->L;
  p.D = (int)a->D;
  p.sign = a->inverse ? -1.0f : 1.0f;
  for (int i = 0; i < kRotaryAxes; ++i) {
    const int n = i < a->axes ? (int)a->sections[i] : 0;
    for (int k = 0; k < n; ++k) p.turns[p.pairs + k] = std::pow(a->base, -(double)k / n) * 0.15915494309189533577;  // / 2 pi
    p.ends[i] = p.pairs += n;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == MVR_F32 ? rotary_as<float>(p, a, st) : a->dtype == MVR_F16 ? rotary_as<__half>(p, a, st) : rotary_as<__nv_bfloat16>(p, a, st);
}

}  // extern "C"
