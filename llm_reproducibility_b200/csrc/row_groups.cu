// Rows grouped by id (a stable counting sort) and the router that produces the ids.
//
// Router.  A score's key is its bit pattern made monotone, with the expert's number below it, so keys are all different,
// larger score first, equal scores by lower number: one maximum gives value and expert, exact whatever the type.  16-bit
// scores make 32-bit keys, fp32 scores 64-bit ones.
//   k <= 8   up to 32 lanes per token, eight keys each at a time.  A lane sorts its eight in registers (a bitonic network),
//            then lists meet pairwise: of two descending lists a, b the larger of a[i], b[7-i] are the best eight, in bitonic
//            order.  No round depends on the one before.  The merges are a loop, not unrolled code: these are kernels of a
//            few microseconds, and fetching a large body costs more than it saves (16384 tokens, 128 experts, k = 8: k rounds
//            of a warp-wide maximum 18.6 us, sixteen keys per lane fully unrolled 12.1 us).
//   else     one warp per token, k rounds of two warp-wide integer reductions.
// Softmax statistics are fp32.
//
// Grouping: rows are dealt to warps in contiguous runs.  Every warp counts its rows per group, the counts are turned into
// first places -- over the warps of a block, over the blocks, over the groups with a scan -- and a second walk over the same
// rows hands out the places in row order: lanes with the same id find each other by ballots over the id's bits (a
// match.any takes some 300 cycles for 32 different ids, eight ballots a third of that).  No global atomics and no waiting
// between blocks: the order is the stable one whatever the timing.
//   few rows    one launch of ONE cluster of up to 8 CTAs; the blocks exchange their counts through distributed shared
//               memory.  What it takes is latency.
//   many rows   a counting launch (the router itself, which has the ids in registers) leaves one row of counts per block in
//               the workspace, and a second launch of as many blocks adds up the rows before its own.
// 131072 rows of 128 groups: one cluster took 41 us, its 8 SMs bound by match.any and by scattered 4-byte stores.
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

constexpr int kGroupThreads = 1024;  // of a CTA of the cluster form
constexpr int kManyThreads = 512;    // of a block of the many-rows form
constexpr int kMaxCluster = 8;
constexpr int kRouteWarps = 32;      // of a block of the router's own launch
constexpr int kBackWarps = 8;        // of a block of its gradient
constexpr int kMaxBlocks = 128;      // of the many-rows form
constexpr int kManyRows = 16384;     // rows from which it is taken

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T> struct Exponent { static constexpr bool kBf16 = false; };
template <> struct Exponent<__nv_bfloat16> { static constexpr bool kBf16 = true; };

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

// The same from a 16-bit score's own bits (u < 2^16), in 16 bits.
template <typename T> __device__ __forceinline__ uint32_t key16(uint32_t u) {
  constexpr uint32_t kInf = sizeof(T) == 2 && Exponent<T>::kBf16 ? 0x7F80u : 0x7C00u;
  const uint32_t size = u & 0x7FFFu;
  const uint32_t key = (u & 0x8000u) && size != 0u ? (~u & 0xFFFFu) : (size | 0x8000u);
  return size > kInf ? 0xFFFFu : key;
}
template <typename T> __device__ __forceinline__ float value16(uint32_t key) {
  if (key == 0xFFFFu) return __uint_as_float(0x7FC00000u);
  const uint16_t u = static_cast<uint16_t>((key & 0x8000u) ? (key & 0x7FFFu) : ~key);
  return to_float(*reinterpret_cast<const T*>(&u));
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
  int aligned;  // rows start on 16-byte boundaries and E is a multiple of 8
  int lanes;    // k <= 8: lanes per token, a power of two
};

// One token by one warp; V = ceil(E / 32) rounded up to a power of two.
// Returns the lane's id (-1 from lane k on).
template <typename T, int V>
__device__ __forceinline__ int route_token(const RouteParams& p, int64_t t, int lane) {
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
    return my_id;
  }
  return -1;
}

// ---- a few lanes per token
template <typename T> struct Key { using type = uint32_t; };
template <> struct Key<float> { using type = unsigned long long; };

// `raw`: the score's bits
template <typename T>
__device__ __forceinline__ typename Key<T>::type packed_key(uint32_t raw, int e) {
  if constexpr (sizeof(T) == 2) return (key16<T>(raw) << 16) | static_cast<uint32_t>(0xFFFF - e);
  else return (static_cast<unsigned long long>(key_of(__uint_as_float(raw))) << 32) | static_cast<uint32_t>(~e);
}
template <typename T>
__device__ __forceinline__ float raw_value(uint32_t raw) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(raw);
  else {
    const uint16_t u = static_cast<uint16_t>(raw);
    return to_float(*reinterpret_cast<const T*>(&u));
  }
}

template <typename K>
__device__ __forceinline__ void order2(K& a, K& b) {  // larger first
  const K hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi;
  b = lo;
}

// Bitonic list of N to descending order.
template <int N, typename K>
__device__ __forceinline__ void bitonic_merge(K* v) {
#pragma unroll
  for (int d = N / 2; d > 0; d /= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & d) == 0) order2(v[i], v[i + d]);
  }
}

// Eight keys in any order to descending order.
template <typename K>
__device__ __forceinline__ void sort8(K* v) {
#pragma unroll
  for (int size = 2; size <= 8; size *= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i ^ (size - 1)) > i) order2(v[i], v[i ^ (size - 1)]);
#pragma unroll
    for (int d = size / 4; d > 0; d /= 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((i & d) == 0) order2(v[i], v[i + d]);
    }
  }
}

// One token by p.lanes neighbouring lanes, k <= 8; live: the token exists (dead lanes shuffle along).  Lane l holds the
// experts 8 l .. 8 l + 7, and the same again 8 p.lanes further where there are more than 256.
template <typename T>
__device__ __forceinline__ void route_few(const RouteParams& p, int64_t t, bool live, int lane, int32_t* counts) {
  using K = typename Key<T>::type;
  const int l = lane & (p.lanes - 1), stride = 8 * p.lanes;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  auto load = [&](int e, uint32_t (&x)[8]) {  // the scores' bits, 0 where there is none
    if (p.aligned) {                          // pieces of eight are whole and on 16-byte boundaries
      uint4 v[sizeof(T) / 2];
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j)
        v[j] = live && e < p.E ? __ldg(reinterpret_cast<const uint4*>(row + e) + j) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4) {
          const uint4 q = v[j / 4];
          x[j] = j % 4 == 0 ? q.x : j % 4 == 1 ? q.y : j % 4 == 2 ? q.z : q.w;
        } else {
          const uint32_t w = j / 2 == 0 ? v[0].x : j / 2 == 1 ? v[0].y : j / 2 == 2 ? v[0].z : v[0].w;
          x[j] = j % 2 ? w >> 16 : w & 0xFFFFu;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = 0u;
        if (live && e + j < p.E) {
          if constexpr (sizeof(T) == 4) x[j] = __float_as_uint(row[e + j]);
          else x[j] = *reinterpret_cast<const uint16_t*>(row + e + j);
        }
      }
    }
  };
  // the best eight of two descending lists
  auto merge = [](K (&a)[8], const K (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = a[i] > b[7 - i] ? a[i] : b[7 - i];
    bitonic_merge<8>(a);
  };
  uint32_t x[8];
  K best[8];
#pragma unroll 1
  for (int e0 = 0; e0 < p.E; e0 += stride) {
    const int e = e0 + 8 * l;
    load(e, x);
    K key[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) key[j] = live && e + j < p.E ? packed_key<T>(x[j], e + j) : K(0);
    sort8(key);
    if (e0 == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) best[j] = key[j];
    } else {
      merge(best, key);
    }
  }
#pragma unroll 1
  for (int d = 1; d < p.lanes; d *= 2) {
    K other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(0xFFFFFFFFu, best[i], d);
    merge(best, other);
  }
  // every lane of the token holds the whole list
  auto value = [](K k) {
    if constexpr (sizeof(T) == 2) return value16<T>(k >> 16); else return value_of(static_cast<uint32_t>(k >> 32));
  };
  const float peak = value(best[0]);
  const bool empty = peak == -INFINITY;  // every expert masked
  // entry i of the list and its exponential: lane l's first is entry l, with fewer than eight lanes more follow
  auto entry = [&](int i) {
    K k = best[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) k = i == j ? best[j] : k;
    return k;
  };
  auto weight = [&](int i, K k) { return i < p.k && !empty ? expf(value(k) - peak) : 0.0f; };
  const K mine = entry(l & 7);
  const float w = weight(l, mine);
  float total = 0.0f;
  if (p.renormalize) {
    total = w;
    for (int i = l + p.lanes; i < p.k; i += p.lanes) total += weight(i, entry(i));
  } else {
#pragma unroll 1
    for (int e0 = 0; e0 < p.E; e0 += stride) {
      const int e = e0 + 8 * l;
      if (stride < p.E) load(e, x);  // else x still holds them
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < p.E) total += expf(raw_value<T>(x[j]) - peak);
    }
  }
  for (int d = 1; d < p.lanes; d *= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
  if (!live) return;
#pragma unroll 1
  for (int i = l; i < p.k; i += p.lanes) {  // the lanes share the writing
    const K k = i == l ? mine : entry(i);
    int e;
    if constexpr (sizeof(T) == 2) e = static_cast<int>(0xFFFFu - (k & 0xFFFFu)); else e = static_cast<int>(~static_cast<uint32_t>(k));
    p.weights[t * p.k + i] = empty ? 0.0f : (i == l ? w : weight(i, k)) / total;
    p.ids[t * p.k + i] = e;
    if (counts) atomicAdd(&counts[e], 1);
  }
}

// The tokens t0 .. t1 - 1 by `warps` warps.  V = 0: k <= 8; else one warp per token with V keys per lane.
template <typename T, int V>
__device__ __forceinline__ void route_run(const RouteParams& p, int64_t t0, int64_t t1, int warp, int warps, int lane, int32_t* counts) {
  if constexpr (V == 0) {
    const int tokens = 32 / p.lanes;
#pragma unroll 1
    for (int64_t t = t0 + warp * tokens; t < t1; t += warps * tokens) {
      const int64_t mine = t + lane / p.lanes;
      route_few<T>(p, mine, mine < t1, lane, counts);
    }
  } else {
#pragma unroll 1
    for (int64_t t = t0 + warp; t < t1; t += warps) {
      const int id = route_token<T, V>(p, t, lane);
      if (counts && id >= 0) atomicAdd(&counts[id], 1);
    }
  }
}

struct GroupParams {
  const int32_t* ids;
  int64_t M;
  int groups;
  int32_t *order, *position, *offsets;
  // many-rows form: counts[block][groups + 1] of runs of rows_per_block rows
  int32_t* counts;
  int64_t rows_per_block;
  int blocks;
};

// Many tokens: the block routes a run of tokens and counts their experts.
template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p, const GroupParams g) {
  __shared__ int32_t counts[TBIK_MAX_GROUPS];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = threadIdx.x; e < p.E; e += kRouteWarps * 32) counts[e] = 0;
  __syncthreads();
  const int64_t tokens = g.rows_per_block / p.k, t0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int64_t t1 = t0 + tokens < p.T ? t0 + tokens : p.T;
  route_run<T, V>(p, t0, t1, threadIdx.x >> 5, kRouteWarps, threadIdx.x & 31, counts);
  __syncthreads();
  for (int e = threadIdx.x; e <= p.E; e += kRouteWarps * 32)
    g.counts[static_cast<int64_t>(blockIdx.x) * (p.E + 1) + e] = e < p.E ? counts[e] : 0;
}

// The same counts for ids that are given.
__global__ void __launch_bounds__(kManyThreads) count_kernel(const GroupParams p) {
  __shared__ int32_t counts[TBIK_MAX_GROUPS + 1];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = threadIdx.x; e <= p.groups; e += kManyThreads) counts[e] = 0;
  __syncthreads();
  const int64_t r0 = blockIdx.x * p.rows_per_block, r1 = r0 + p.rows_per_block < p.M ? r0 + p.rows_per_block : p.M;
  for (int64_t i = r0 + threadIdx.x; i < r1; i += kManyThreads) {
    const int id = p.ids[i];
    atomicAdd(&counts[id < 0 || id >= p.groups ? p.groups : id], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= p.groups; e += kManyThreads) p.counts[static_cast<int64_t>(blockIdx.x) * (p.groups + 1) + e] = counts[e];
}

// Places of the rows of the batch.  smem: [warps][G + 1] counts, then [G + 1] totals of the block, [G + 1] rows before,
// [G + 1] first places, [32] warp sums of the scan.
template <bool MANY>
__device__ __forceinline__ void group_block(const GroupParams& p, int32_t* smem) {
  constexpr int THREADS = MANY ? kManyThreads : kGroupThreads, WARPS = THREADS / 32;
  cg::cluster_group cluster = cg::this_cluster();
  const int nb = MANY ? p.blocks : static_cast<int>(cluster.num_blocks());
  const int rank = MANY ? static_cast<int>(blockIdx.x) : static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.groups + 1;  // the last bucket: rows of no group
  int32_t* counts = smem;
  int32_t* totals = smem + WARPS * B;
  int32_t* earlier = totals + B;
  int32_t* first = earlier + B;
  int32_t* sums = first + B;
  for (int i = threadIdx.x; i < WARPS * B + 2 * B; i += THREADS) counts[i] = 0;
  __syncthreads();

  const int64_t per_block = MANY ? p.rows_per_block : (p.M + nb - 1) / nb;
  const int64_t per_warp = ((per_block + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int64_t run0 = MANY ? rank * per_block : rank * per_warp * WARPS;  // the block's run of rows
  const int64_t run1 = MANY ? (run0 + per_block < p.M ? run0 + per_block : p.M) : p.M;
  const int64_t row0 = run0 + warp * per_warp;
  const int64_t row1 = row0 + per_warp < run1 ? row0 + per_warp : run1;
  int32_t* mine = counts + warp * B;
  constexpr int U = 4;  // steps whose ids are requested together
  // walk(f): f(row, bucket, whether the lane has a row), 32 rows at a time, by all lanes
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
        if (r + u * 32 < row1) f(i, (id[u] < 0 || id[u] >= p.groups) ? p.groups : id[u], i < row1);
      }
    }
  };
  walk([&](int64_t, int b, bool live) {
    if (live) atomicAdd(&mine[b], 1);
  });
  if constexpr (MANY) {
    // Counts of the other blocks.  Eight neighbours share the reading: each adds up an eighth of the rows -- all of them, and
    // those before the cluster -- and leaves the sums to the others; what the neighbours before it have it reads itself.
    // (Every block reading all rows took 6.6k cycles, most of it waiting for the same lines as everyone else.)
    const int in_cluster = rank % kMaxCluster, first_block = rank - in_cluster;
    const int chunks = (B + 31) / 32;
    for (int c = warp; c < chunks; c += WARPS) {
      const int b = c * 32 + lane;
      if (b < B) {
        int all = 0, before = 0, near = 0;
        const int32_t* from = p.counts + b;
        int v[kMaxBlocks / kMaxCluster], u[kMaxCluster - 1];
#pragma unroll
        for (int i = 0; i < kMaxBlocks / kMaxCluster; ++i) {
          const int k = i * kMaxCluster + in_cluster;
          v[i] = k < nb ? __ldcg(from + static_cast<int64_t>(k) * B) : 0;
        }
#pragma unroll
        for (int i = 0; i < kMaxCluster - 1; ++i)
          u[i] = i < in_cluster && first_block + i < nb ? __ldcg(from + static_cast<int64_t>(first_block + i) * B) : 0;
#pragma unroll
        for (int i = 0; i < kMaxBlocks / kMaxCluster; ++i) {
          all += v[i];
          before += i * kMaxCluster + in_cluster < first_block ? v[i] : 0;
        }
#pragma unroll
        for (int i = 0; i < kMaxCluster - 1; ++i) near += u[i];
        totals[b] = all;
        earlier[b] = before;
        first[b] = near;
      }
    }
  }
  __syncthreads();
  const int64_t longest = min(MANY ? per_block : per_warp * WARPS, p.M);  // rows of a block at most
  const int used = per_warp > 0 ? static_cast<int>((longest + per_warp - 1) / per_warp) : 0;  // warps that can have rows
  for (int b = threadIdx.x; b < B; b += THREADS) {
    int32_t run = 0;
    for (int w = 0; w < used; ++w) {
      const int32_t c = counts[w * B + b];
      counts[w * B + b] = run;
      run += c;
    }
    if constexpr (!MANY) totals[b] = run;
  }
  if (MANY || nb > 1) cluster.sync(); else __syncthreads();
  // scan over the buckets, `width` neighbours per thread
  constexpr int PER = (TBIK_MAX_GROUPS + 1 + THREADS - 1) / THREADS;
  const int width = (B + THREADS - 1) / THREADS;
  int32_t all[PER], before[PER], run = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int b = width * static_cast<int>(threadIdx.x) + u;
    all[u] = before[u] = 0;
    if (u < width && b < B) {
      if constexpr (MANY) {
        before[u] = first[b];  // (this thread's alone)
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
          all[u] += cluster.map_shared_rank(totals, c)[b];
          before[u] += cluster.map_shared_rank(earlier, c)[b];
        }
      } else if (nb == 1) {
        all[u] = totals[b];
      } else {
        for (int c = 0; c < nb; ++c) {
          const int32_t v = cluster.map_shared_rank(totals, c)[b];
          all[u] += v;
          if (c < rank) before[u] += v;
        }
      }
    }
    run += all[u];
  }
  int32_t start = -run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(0xFFFFFFFFu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  start += run;
  for (int w = 0; w < warp; ++w) start += sums[w];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int b = width * static_cast<int>(threadIdx.x) + u;
    if (u < width && b < B) {
      first[b] = start + before[u];
      if (rank == 0) p.offsets[b] = start;
    }
    start += all[u];
  }
  if (MANY || nb > 1) cluster.sync(); else __syncthreads();  // nobody leaves while its totals may still be read
  const int bits = 32 - __clz(p.groups);  // of a bucket's number
  walk([&](int64_t i, int b, bool live) {
    unsigned peers = __ballot_sync(0xFFFFFFFFu, live);
    for (int k = 0; k < bits; ++k) {
      const unsigned set = __ballot_sync(0xFFFFFFFFu, (b >> k) & 1);
      peers &= (b >> k) & 1 ? set : ~set;
    }
    int at = 0;
    if (live) at = first[b] + mine[b] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();  // everyone has read the count before it moves on
    if (live && lane == __ffs(peers) - 1) mine[b] += __popc(peers);
    __syncwarp();
    if (live) {
      p.order[at] = static_cast<int32_t>(i);
      p.position[i] = at;
    }
  });
}

__global__ void __launch_bounds__(kGroupThreads) group_kernel(const GroupParams p) {
  extern __shared__ int32_t group_smem[];
  group_block<false>(p, group_smem);
}

__global__ void __launch_bounds__(kManyThreads) group_many_kernel(const GroupParams p) {
  extern __shared__ int32_t group_smem[];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the ids and counts of the launch before
  group_block<true>(p, group_smem);
}

// Few tokens: router and grouping in one launch of one cluster.
template <typename T, int V>
__global__ void __launch_bounds__(kGroupThreads) route_group_kernel(const RouteParams r, const GroupParams p) {
  extern __shared__ int32_t group_smem[];
  constexpr int WARPS = kGroupThreads / 32;
  route_run<T, V>(r, 0, r.T, blockIdx.x * WARPS + (threadIdx.x >> 5), gridDim.x * WARPS, threadIdx.x & 31, nullptr);
  __threadfence();
  if (gridDim.x > 1) cg::this_cluster().sync(); else __syncthreads();
  group_block<false>(p, group_smem);
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
__global__ void __launch_bounds__(kBackWarps * 32) route_backward_kernel(const RouteBackParams p) {
  __shared__ float rows[kBackWarps][TBIK_MAX_GROUPS];
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kBackWarps + (threadIdx.x >> 5);
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
size_t group_smem_bytes(int groups, int threads) { return (static_cast<size_t>(threads / 32 + 3) * (groups + 1) + 32) * sizeof(int32_t); }

// CTAs of the cluster: one per 1024 rows, at most 8.  Few rows are done sooner without the cluster's barriers.
int cluster_size(int64_t M) {
  int c = 1;
  while (c < kMaxCluster && M > 1024 * c) c *= 2;
  return c;
}

// Launches `kernel` on `blocks` blocks: as one cluster, or (after) in clusters of eight that may start while the launch
// before them still runs and wait for it themselves.
template <typename... Params>
int launch_groups(void (*kernel)(Params...), const char* what, int blocks, int threads, size_t smem, bool after, cudaStream_t stream,
                  const Params&... params) {
  if (smem > 48 * 1024) {
    // belongs to (kernel, device); setting it again is cheap and idempotent
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return set_cuda_error(e, what);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(after ? kMaxCluster : blocks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params...);
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, what);
}

// Blocks of the many-rows form: runs of whole multiples of `unit` rows, at least 64, at most kMaxBlocks of them.
void many_blocks(GroupParams* g, int64_t unit) {
  int64_t per = (g->M + kMaxBlocks - 1) / kMaxBlocks;
  if (per < 64) per = 64;
  g->rows_per_block = (per + unit - 1) / unit * unit;
  g->blocks = static_cast<int>((g->M + g->rows_per_block - 1) / g->rows_per_block);
}

int check_group(int64_t M, int groups, const void* ids, const void* order, const void* position, const void* offsets,
                const char* what) {
  if (groups < 1 || groups > TBIK_MAX_GROUPS) return set_error(TBIK_ERR_SHAPE, what);
  if (M < 0 || M >= (int64_t(1) << 31)) return set_error(TBIK_ERR_SHAPE, what);
  if (!offsets || (M > 0 && (!ids || !order || !position))) return set_error(TBIK_ERR_ARG, what);
  return TBIK_OK;
}

template <typename T, int V>
int route_launch(const RouteParams& r, GroupParams g, cudaStream_t stream) {
  constexpr int WARPS = kGroupThreads / 32;
  const int tokens = V == 0 ? 32 / r.lanes : 1;  // of a warp at a time
  if (g.M < kManyRows && r.T <= 4 * kMaxCluster * WARPS * tokens) {
    // one launch: the cluster's warps go round four times at most
    int ctas = cluster_size(g.M);
    while (ctas < kMaxCluster && r.T > ctas * WARPS * tokens) ctas *= 2;
    return launch_groups(route_group_kernel<T, V>, "route_group_kernel launch", ctas, kGroupThreads,
                         group_smem_bytes(g.groups, kGroupThreads), false, stream, r, g);
  }
  many_blocks(&g, r.k);
  route_kernel<T, V><<<static_cast<unsigned>(g.blocks), kRouteWarps * 32, 0, stream>>>(r, g);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "route_kernel launch");
  return launch_groups(group_many_kernel, "group_many_kernel launch", (g.blocks + kMaxCluster - 1) / kMaxCluster * kMaxCluster, kManyThreads, group_smem_bytes(g.groups, kManyThreads),
                       true, stream, g);
}

template <typename T>
int route_width(const RouteParams& r, const GroupParams& g, cudaStream_t stream) {
  if (r.k <= 8) return route_launch<T, 0>(r, g, stream);
  if (r.E <= 128) return route_launch<T, 4>(r, g, stream);
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

int check_workspace(int64_t M, int groups, const void* workspace, size_t bytes) {
  if (!workspace || bytes < group_workspace_bytes(M, groups) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
    return set_error(TBIK_ERR_ARG, "tbik_group_rows / tbik_route_topk: workspace of tbik_group_workspace_bytes() bytes needed");
  return TBIK_OK;
}

}  // namespace

size_t group_workspace_bytes(int64_t M, int groups) {
  // the router's runs are whole tokens and no shorter than these
  if (M < 1 || groups < 1 || groups > TBIK_MAX_GROUPS) return 0;
  GroupParams g{};
  g.M = M;
  many_blocks(&g, 1);
  return static_cast<size_t>(g.blocks) * (groups + 1) * sizeof(int32_t);
}

int group_rows(const int32_t* ids, int64_t M, int groups, int32_t* order, int32_t* position, int32_t* offsets, void* workspace,
               size_t workspace_bytes, cudaStream_t stream) {
  const int rc = check_group(M, groups, ids, order, position, offsets,
                             "tbik_group_rows: 1 .. 1024 groups, 0 .. 2^31 - 1 rows, no null pointers");
  if (rc != TBIK_OK) return rc;
  GroupParams g{ids, M, groups, order, position, offsets, static_cast<int32_t*>(workspace), 0, 0};
  if (M < kManyRows)
    return launch_groups(group_kernel, "group_kernel launch", cluster_size(M), kGroupThreads, group_smem_bytes(groups, kGroupThreads),
                         false, stream, g);
  const int rc2 = check_workspace(M, groups, workspace, workspace_bytes);
  if (rc2 != TBIK_OK) return rc2;
  many_blocks(&g, 1);
  count_kernel<<<static_cast<unsigned>(g.blocks), kManyThreads, 0, stream>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "count_kernel launch");
  return launch_groups(group_many_kernel, "group_many_kernel launch", (g.blocks + kMaxCluster - 1) / kMaxCluster * kMaxCluster, kManyThreads, group_smem_bytes(groups, kManyThreads),
                       true, stream, g);
}

int route_topk(const void* logits, int64_t ld, int64_t T, int E, int k, int dtype, int renormalize, float* weights,
               int32_t* ids, int32_t* order, int32_t* position, int32_t* offsets, void* workspace, size_t workspace_bytes,
               cudaStream_t stream) {
  int rc = check_route(T, E, k, dtype);
  if (rc != TBIK_OK) return rc;
  rc = check_group(T * k, E, ids, order, position, offsets, "tbik_route_topk: null pointer");
  if (rc != TBIK_OK) return rc;
  if (T > 0 && (!logits || !weights)) return set_error(TBIK_ERR_ARG, "tbik_route_topk: null pointer");
  if (T > 0) {
    rc = check_workspace(T * k, E, workspace, workspace_bytes);
    if (rc != TBIK_OK) return rc;
  }
  const int es = dtype == TBIK_DTYPE_FP32 ? 4 : 2;
  const int aligned = E % 8 == 0 && ld * es % 16 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
  int lanes = 1;
  while (lanes < 32 && lanes * 8 < E) lanes *= 2;
  const RouteParams r{logits, ld, T, E, k, renormalize, weights, ids, aligned, lanes};
  const GroupParams g{ids, T * k, E, order, position, offsets, static_cast<int32_t*>(workspace), 0, 0};
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
  const unsigned grid = static_cast<unsigned>((T + kBackWarps - 1) / kBackWarps);
  if (dtype == TBIK_DTYPE_BF16) route_backward_kernel<__nv_bfloat16><<<grid, kBackWarps * 32, 0, stream>>>(p);
  else if (dtype == TBIK_DTYPE_FP16) route_backward_kernel<__half><<<grid, kBackWarps * 32, 0, stream>>>(p);
  else route_backward_kernel<float><<<grid, kBackWarps * 32, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "route_backward_kernel launch");
}

}  // namespace tbik
