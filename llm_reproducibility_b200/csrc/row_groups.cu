// Rows grouped by id (a stable counting sort) and the router that produces the ids.
//
// Router: one warp per token.  The token's E scores sit in registers, element e in lane e % 32; each of k rounds takes the
// largest key over the warp and, among equal keys, the lowest index (two warp-wide integer reductions).  A score's key
// is its bit pattern made monotone, so the order is total and exact whatever the type.  Softmax statistics are fp32.
//
// Grouping: ONE cluster of up to 8 CTAs x 32 warps.  Warp w of the cluster owns the w-th contiguous run of rows, counts
// its rows per group (lanes with the same id find each other with match.any, one of them adds), the counts are turned
// into first places -- over the warps of a CTA in shared memory, over the CTAs through distributed shared memory, over
// the groups with a scan -- and a second walk over the same rows hands out the places in row order.  No atomics: the
// order is the stable one whatever the timing.  Both walks read the ids from L2; the bound is the latency of the
// cluster's few SMs, not bytes.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "tbik_internal.h"

namespace tbik {
namespace {

namespace cg = cooperative_groups;

constexpr int kGroupThreads = 1024;
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kRouteWarps = 8;  // tokens per block of the router's own launch

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Monotone key of a score: larger score, larger key; -0 equals +0; every NaN is the largest key; 0 is below them all.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

struct RouteParams {
  const void* logits;
  int64_t ld, T;
  int E, k, renormalize;
  float* weights;
  int32_t* ids;
};

// One token by one warp; V = ceil(E / 32) rounded up to a power of two.
template <typename T, int V>
__device__ __forceinline__ void route_token(const RouteParams& p, int64_t t, int lane) {
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  uint32_t key[V];
  uint32_t best = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = j * 32 + lane;
    key[j] = e < p.E ? key_of(to_float(row[e])) : 0u;
    best = max(best, key[j]);
  }
  const float peak = value_of(__reduce_max_sync(0xFFFFFFFFu, best));
  const bool empty = peak == -INFINITY;  // every expert masked
  float total = 0.0f;
  if (!p.renormalize) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[j] != 0u) total += expf(value_of(key[j]) - peak);
    total = warp_sum(total);
  }
  float mine = 0.0f;
  int my_id = 0;
  for (int r = 0; r < p.k; ++r) {
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll
    for (int j = V - 1; j >= 0; --j)
      if (key[j] == top) at = j * 32 + lane;
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    if (lane == r) {
      mine = value_of(top);
      my_id = static_cast<int>(at);
    }
    if (static_cast<int>(at & 31u) == lane) {  // the lane that gave it up looks for its next one
      best = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j == static_cast<int>(at >> 5)) key[j] = 0u;
        best = max(best, key[j]);
      }
    }
  }
  float w = (lane < p.k && !empty) ? expf(mine - peak) : 0.0f;
  if (p.renormalize) total = warp_sum(w);
  if (lane < p.k) {
    p.weights[t * p.k + lane] = empty ? 0.0f : w / total;
    p.ids[t * p.k + lane] = my_id;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (t < p.T) route_token<T, V>(p, t, threadIdx.x & 31);
}

struct GroupParams {
  const int32_t* ids;
  int64_t M;
  int groups;
  int32_t *order, *position, *offsets;
};

// Places of the rows of one cluster's batch.  smem: [warps][G + 1] counts, then [G + 1] CTA totals, [G + 1] first
// places, [32] warp sums of the scan.
__device__ __forceinline__ void group_cluster(const GroupParams& p, int32_t* smem) {
  cg::cluster_group cluster = cg::this_cluster();
  const int nb = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.groups + 1;  // the last bucket: rows of no group
  int32_t* counts = smem;
  int32_t* totals = smem + kGroupWarps * B;
  int32_t* first = totals + B;
  int32_t* sums = first + B;
  for (int i = threadIdx.x; i < kGroupWarps * B; i += kGroupThreads) counts[i] = 0;
  __syncthreads();

  const int64_t per_warp = ((p.M + nb * kGroupWarps - 1) / (nb * kGroupWarps) + 31) / 32 * 32;
  const int64_t row0 = (static_cast<int64_t>(rank) * kGroupWarps + warp) * per_warp;
  const int64_t row1 = row0 + per_warp < p.M ? row0 + per_warp : p.M;
  int32_t* mine = counts + warp * B;
  constexpr int U = 4;  // steps whose ids are requested together
  // walk(f): f(row, bucket, lanes of the step with the same bucket, lanes with a row) for every row of this warp, 32 at a time
  auto walk = [&](auto&& f) {
    for (int64_t r = row0; r < row1; r += 32 * U) {
      int32_t id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = r + u * 32 + lane;
        id[u] = i < row1 ? __ldcg(p.ids + i) : 0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = r + u * 32 + lane;
        const unsigned live = __ballot_sync(0xFFFFFFFFu, i < row1);
        if (i < row1) {
          const int b = (id[u] < 0 || id[u] >= p.groups) ? p.groups : id[u];
          f(i, b, __match_any_sync(live, b), live);
        }
        __syncwarp();
      }
    }
  };
  walk([&](int64_t, int b, unsigned peers, unsigned) {
    if (lane == __ffs(peers) - 1) mine[b] += __popc(peers);
  });
  __syncthreads();
  for (int b = threadIdx.x; b < B; b += kGroupThreads) {
    int32_t run = 0;
    for (int w = 0; w < kGroupWarps; ++w) {
      const int32_t c = counts[w * B + b];
      counts[w * B + b] = run;
      run += c;
    }
    totals[b] = run;
  }
  cluster.sync();
  // scan over the buckets: thread t holds buckets 2t and 2t + 1
  int32_t all[2] = {0, 0}, before[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int b = 2 * static_cast<int>(threadIdx.x) + u;
    if (b < B) {
      for (int c = 0; c < nb; ++c) {
        const int32_t v = cluster.map_shared_rank(totals, c)[b];
        all[u] += v;
        if (c < rank) before[u] += v;
      }
    }
  }
  int32_t run = all[0] + all[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(0xFFFFFFFFu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  if (warp == 0) {
    int32_t s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t v = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += v;
    }
    sums[lane] = s;
  }
  __syncthreads();
  int32_t start = run - all[0] - all[1] + (warp > 0 ? sums[warp - 1] : 0);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int b = 2 * static_cast<int>(threadIdx.x) + u;
    if (b < B) {
      first[b] = start + before[u];
      if (rank == 0) p.offsets[b] = start;
    }
    start += all[u];
  }
  cluster.sync();  // nobody leaves while its totals may still be read; also publishes `first` to the block
  walk([&](int64_t i, int b, unsigned peers, unsigned live) {
    const int32_t at = first[b] + mine[b] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp(live);  // everyone has read the count before it moves on
    if (lane == __ffs(peers) - 1) mine[b] += __popc(peers);
    p.order[at] = static_cast<int32_t>(i);
    p.position[i] = at;
  });
}

__global__ void __launch_bounds__(kGroupThreads) group_kernel(const GroupParams p) {
  extern __shared__ int32_t group_smem[];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the router's ids, when this launch follows it
  group_cluster(p, group_smem);
}

// Few tokens: router and grouping in one launch of one cluster.
template <typename T, int V>
__global__ void __launch_bounds__(kGroupThreads) route_group_kernel(const RouteParams r, const GroupParams p) {
  extern __shared__ int32_t group_smem[];
  const int warps = gridDim.x * kGroupWarps;
  for (int64_t t = blockIdx.x * kGroupWarps + (threadIdx.x >> 5); t < r.T; t += warps) route_token<T, V>(r, t, threadIdx.x & 31);
  __threadfence();
  cg::this_cluster().sync();
  group_cluster(p, group_smem);
}

struct RouteBackParams {
  const void* logits;
  int64_t ld, T;
  int E, k, renormalize;
  const float* weights;
  const int32_t* ids;
  const float* dweights;
  void* dlogits;
  int64_t ldd;
};

// dl_e = p_e (dp_e - sum_j p_j dp_j), the Jacobian of the softmax over the set it ran over: the chosen k (renormalize: p
// is the weight, everything else gets 0) or all E.  One warp per token; the chosen experts' terms meet in a row of
// shared memory.
template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32) route_backward_kernel(const RouteBackParams p) {
  __shared__ float rows[kRouteWarps][TBIK_MAX_GROUPS];
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  float* s = rows[threadIdx.x >> 5];
  for (int e = lane; e < p.E; e += 32) s[e] = 0.0f;
  float w = 0.0f, dw = 0.0f;
  int id = -1;
  if (lane < p.k) {
    w = p.weights[t * p.k + lane];
    dw = p.dweights[t * p.k + lane];
    id = p.ids[t * p.k + lane];
  }
  const float inner = warp_sum(w * dw);
  __syncwarp();
  if (id >= 0 && id < p.E) s[id] = p.renormalize ? w * (dw - inner) : dw;
  __syncwarp();
  T* out = static_cast<T*>(p.dlogits) + t * p.ldd;
  if (p.renormalize) {
    for (int e = lane; e < p.E; e += 32) out[e] = from_float<T>(s[e]);
    return;
  }
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  uint32_t best = 0;
  for (int e = lane; e < p.E; e += 32) best = max(best, key_of(to_float(row[e])));
  const float peak = value_of(__reduce_max_sync(0xFFFFFFFFu, best));
  const bool empty = peak == -INFINITY;
  float total = 0.0f;
  for (int e = lane; e < p.E; e += 32) total += expf(to_float(row[e]) - peak);
  total = warp_sum(total);
  for (int e = lane; e < p.E; e += 32)
    out[e] = from_float<T>(empty ? 0.0f : expf(to_float(row[e]) - peak) / total * (s[e] - inner));
}

// ---------------------------------------------------------------- host side
constexpr int kDevices = 64;

size_t group_smem_bytes(int groups) { return (static_cast<size_t>(kGroupWarps + 2) * (groups + 1) + 32) * sizeof(int32_t); }

// CTAs of the cluster: one per 2048 rows, at most 8.  Few rows are done sooner without the cluster's barriers.
int cluster_size(int64_t M) {
  int c = 1;
  while (c < kMaxCluster && M > 2048 * c) c *= 2;
  return c;
}

template <typename... Params>
int launch_cluster(void (*kernel)(Params...), const char* what, int ctas, size_t smem, bool after, cudaStream_t stream,
                   const Params&... params) {
  // the attribute belongs to (kernel, device); setting it again is cheap and idempotent
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return set_cuda_error(e, what);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kGroupThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params...);
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, what);
}

int check_group(int64_t M, int groups, const void* ids, const void* order, const void* position, const void* offsets,
                const char* what) {
  if (groups < 1 || groups > TBIK_MAX_GROUPS) return set_error(TBIK_ERR_SHAPE, what);
  if (M < 0 || M >= (int64_t(1) << 31)) return set_error(TBIK_ERR_SHAPE, what);
  if (!offsets || (M > 0 && (!ids || !order || !position))) return set_error(TBIK_ERR_ARG, what);
  return TBIK_OK;
}

template <typename T, int V>
int route_launch(const RouteParams& r, const GroupParams& g, cudaStream_t stream) {
  const size_t smem = group_smem_bytes(g.groups);
  // One launch while the cluster's 32 warps per CTA take at most two tokens each; beyond that the router gets the GPU.
  const int ctas = cluster_size(g.M);
  int fused = ctas;
  while (fused < kMaxCluster && r.T > 2 * fused * kGroupWarps) fused *= 2;
  if (r.T <= 2 * fused * kGroupWarps)
    return launch_cluster(route_group_kernel<T, V>, "route_group_kernel launch", fused, smem, false, stream, r, g);
  route_kernel<T, V><<<static_cast<unsigned>((r.T + kRouteWarps - 1) / kRouteWarps), kRouteWarps * 32, 0, stream>>>(r);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "route_kernel launch");
  return launch_cluster(group_kernel, "group_kernel launch", ctas, smem, true, stream, g);
}

template <typename T>
int route_width(const RouteParams& r, const GroupParams& g, cudaStream_t stream) {
  if (r.E <= 32) return route_launch<T, 1>(r, g, stream);
  if (r.E <= 64) return route_launch<T, 2>(r, g, stream);
  if (r.E <= 128) return route_launch<T, 4>(r, g, stream);
  if (r.E <= 256) return route_launch<T, 8>(r, g, stream);
  if (r.E <= 512) return route_launch<T, 16>(r, g, stream);
  return route_launch<T, 32>(r, g, stream);
}

int check_route(int64_t T, int E, int k, int dtype) {
  if (dtype != TBIK_DTYPE_BF16 && dtype != TBIK_DTYPE_FP16 && dtype != TBIK_DTYPE_FP32)
    return set_error(TBIK_ERR_DTYPE, "tbik_route_topk: dtype must be bf16, fp16 or fp32");
  if (E < 1 || E > TBIK_MAX_GROUPS) return set_error(TBIK_ERR_SHAPE, "tbik_route_topk: E must be in 1 .. 1024");
  if (k < 1 || k > E || k > TBIK_MAX_TOPK) return set_error(TBIK_ERR_SHAPE, "tbik_route_topk: k must be in 1 .. min(E, 32)");
  if (T < 0 || T * k >= (int64_t(1) << 31)) return set_error(TBIK_ERR_SHAPE, "tbik_route_topk: T * k must be below 2^31");
  return TBIK_OK;
}

}  // namespace

int group_rows(const int32_t* ids, int64_t M, int groups, int32_t* order, int32_t* position, int32_t* offsets,
               cudaStream_t stream) {
  const int rc = check_group(M, groups, ids, order, position, offsets,
                             "tbik_group_rows: 1 .. 1024 groups, 0 .. 2^31 - 1 rows, no null pointers");
  if (rc != TBIK_OK) return rc;
  const GroupParams g{ids, M, groups, order, position, offsets};
  return launch_cluster(group_kernel, "group_kernel launch", cluster_size(M), group_smem_bytes(groups), false, stream, g);
}

int route_topk(const void* logits, int64_t ld, int64_t T, int E, int k, int dtype, int renormalize, float* weights,
               int32_t* ids, int32_t* order, int32_t* position, int32_t* offsets, cudaStream_t stream) {
  int rc = check_route(T, E, k, dtype);
  if (rc != TBIK_OK) return rc;
  rc = check_group(T * k, E, ids, order, position, offsets, "tbik_route_topk: null pointer");
  if (rc != TBIK_OK) return rc;
  if (T > 0 && (!logits || !weights)) return set_error(TBIK_ERR_ARG, "tbik_route_topk: null pointer");
  const RouteParams r{logits, ld, T, E, k, renormalize, weights, ids};
  const GroupParams g{ids, T * k, E, order, position, offsets};
  if (dtype == TBIK_DTYPE_BF16) return route_width<__nv_bfloat16>(r, g, stream);
  if (dtype == TBIK_DTYPE_FP16) return route_width<__half>(r, g, stream);
  return route_width<float>(r, g, stream);
}

int route_topk_backward(const void* logits, int64_t ld, int64_t T, int E, int k, int dtype, int renormalize,
                        const float* weights, const int32_t* ids, const float* dweights, void* dlogits, int64_t ldd,
                        cudaStream_t stream) {
  const int rc = check_route(T, E, k, dtype);
  if (rc != TBIK_OK || T == 0) return rc;
  if (!logits || !weights || !ids || !dweights || !dlogits) return set_error(TBIK_ERR_ARG, "tbik_route_topk_backward: null pointer");
  const RouteBackParams p{logits, ld, T, E, k, renormalize, weights, ids, dweights, dlogits, ldd};
  const unsigned grid = static_cast<unsigned>((T + kRouteWarps - 1) / kRouteWarps);
  if (dtype == TBIK_DTYPE_BF16) route_backward_kernel<__nv_bfloat16><<<grid, kRouteWarps * 32, 0, stream>>>(p);
  else if (dtype == TBIK_DTYPE_FP16) route_backward_kernel<__half><<<grid, kRouteWarps * 32, 0, stream>>>(p);
  else route_backward_kernel<float><<<grid, kRouteWarps * 32, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "route_backward_kernel launch");
}

}  // namespace tbik
