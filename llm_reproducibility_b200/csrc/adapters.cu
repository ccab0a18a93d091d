// Low-rank adapters of many requests: out[t] = round(y[t] + s_a B_a h[t]), h[t] = A_a x[t] in fp32, a = adapter of row t.
//
// First form: one block per row, every dot product by one warp, nothing shared between rows.  K is summed leaf by leaf,
// the leaves' sums are added pairwise.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tbik_internal.h"

namespace tbik {
namespace {

constexpr int kThreads = 256;
constexpr int kLeaves = 8;

__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }

struct Params {
  const void *x, *y, *A, *B;
  void* out;
  const float* scales;
  float* h;
  const int32_t *order, *offsets;
  int64_t T, ldx, ldy, ldo;
  int N, K, R, adapters, leaf;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) adapters_kernel(const Params p) {
  __shared__ float hs[TBIK_MAX_RANK];
  __shared__ int adapter;
  const int64_t place = blockIdx.x;
  const int64_t t = p.order[place];
  if (t < 0 || t >= p.T) return;
  if (threadIdx.x == 0) {
    int a = -1;
    for (int g = 0; g < p.adapters; ++g)
      if (place >= p.offsets[g] && place < p.offsets[g + 1]) a = g;
    adapter = a;
  }
  __syncthreads();
  const int a = adapter, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (p.x && a >= 0) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    for (int r = warp; r < p.R; r += kThreads / 32) {
      const T* w = static_cast<const T*>(p.A) + (static_cast<int64_t>(a) * p.R + r) * p.K;
      float sum[kLeaves];
#pragma unroll
      for (int l = 0; l < kLeaves; ++l) {
        sum[l] = 0.0f;
        for (int64_t k = static_cast<int64_t>(l) * p.leaf + lane; k < min(static_cast<int64_t>(l + 1) * p.leaf, static_cast<int64_t>(p.K)); k += 32)
          sum[l] = fmaf(f32(x[k]), f32(w[k]), sum[l]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum[l] += __shfl_xor_sync(0xFFFFFFFFu, sum[l], o);
      }
      if (lane == 0) hs[r] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
    }
  } else {
    for (int r = threadIdx.x; r < p.R; r += kThreads) hs[r] = (p.x || a < 0) ? 0.0f : p.h[t * p.R + r];
  }
  __syncthreads();
  if (!p.y) {
    for (int r = threadIdx.x; r < p.R; r += kThreads) p.h[t * p.R + r] = hs[r];
    return;
  }
  const T* y = static_cast<const T*>(p.y) + t * p.ldy;
  T* out = static_cast<T*>(p.out) + t * p.ldo;
  for (int n = threadIdx.x; n < p.N; n += kThreads) {
    if (a < 0) {
      out[n] = y[n];
      continue;
    }
    const T* b = static_cast<const T*>(p.B) + (static_cast<int64_t>(a) * p.N + n) * p.R;
    float d = 0.0f;
    for (int r = 0; r < p.R; ++r) d = fmaf(hs[r], f32(b[r]), d);
    out[n] = rounded<T>(f32(y[n]) + p.scales[a] * d);
  }
}

bool bad_align(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

int adapters(const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo, const void* A, const void* B,
             const float* scales, float* h, const int32_t* order, const int32_t* offsets, int64_t T, int N, int K, int R,
             int adapters, int dtype, int leaf, cudaStream_t stream) {
  if (dtype != TBIK_DTYPE_BF16 && dtype != TBIK_DTYPE_FP16) return set_error(TBIK_ERR_DTYPE, "tbik_adapters supports bf16 and fp16");
  if (T < 0 || T >= (int64_t(1) << 31) || N < 8 || N % 8 || K < 8 || K % 8)
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: T in 0 .. 2^31 - 1, N and K positive multiples of 8");
  if (R < 8 || R % 8 || R > TBIK_MAX_RANK) return set_error(TBIK_ERR_SHAPE, "tbik_adapters: R must be a multiple of 8 up to 128");
  if (adapters < 1 || adapters > TBIK_MAX_GROUPS) return set_error(TBIK_ERR_SHAPE, "tbik_adapters: 1 .. 1024 adapters");
  if (leaf == 0) leaf = (K + 255) / 256 * 32;
  if (leaf < 0 || leaf % 32 || (static_cast<int64_t>(K) + leaf - 1) / leaf > kLeaves)
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: leaf must be a multiple of 32 with at most 8 leaves covering K");
  if (T == 0) return TBIK_OK;
  const bool shrink = x != nullptr, expand = y != nullptr;
  if (!order || !offsets || (!shrink && !expand) || (shrink && !A) || (expand && (!out || !B || !scales)) || (shrink != expand && !h))
    return set_error(TBIK_ERR_ARG, "tbik_adapters: null pointer");
  if ((shrink && ldx < K) || (expand && (ldy < N || ldo < N)))
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: row stride smaller than the row");
  if (bad_align(x) || bad_align(y) || bad_align(out) || bad_align(A) || bad_align(B) || bad_align(h) || ldx % 8 || ldy % 8 || ldo % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_adapters: pointers must be 16-byte aligned, row strides multiples of 8 elements");
  const Params p{x, y, A, B, out, scales, h, order, offsets, T, ldx, ldy, ldo, N, K, R, adapters, leaf};
  if (dtype == TBIK_DTYPE_BF16) adapters_kernel<__nv_bfloat16><<<static_cast<unsigned>(T), kThreads, 0, stream>>>(p);
  else adapters_kernel<__half><<<static_cast<unsigned>(T), kThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "adapters_kernel launch");
}

}  // namespace tbik
