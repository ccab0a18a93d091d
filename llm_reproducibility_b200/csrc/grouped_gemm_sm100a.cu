// Products of rows grouped by expert, ragged sizes: C[i] = A[i] W[g(i)]^T and the weight gradient.
//
// First form: 64x64 tiles of fp32 fused multiply-adds from shared memory, one block per column tile and group.  Right for
// every layout, type and size; bound by the fp32 pipe.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "tbik_internal.h"

namespace tbik {
namespace {

constexpr int TM = 64, TN = 64, TK = 16;
constexpr int kMaxLevels = 16;

__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

struct Params {
  const void *A, *W;
  void* C;
  const int32_t* offsets;
  int64_t M;
  int N, K, groups;
  int64_t lda, ldw, stride_w, ldc;
  int w_n_contiguous, leaf, T, F, L, outside;
};

// The group's rows, clamped to the operands whatever the table holds.
__device__ __forceinline__ void group_rows_of(const int32_t* offsets, int g, int64_t M, int64_t& r0, int64_t& r1) {
  r0 = min(max(static_cast<int64_t>(offsets[g]), int64_t(0)), M);
  r1 = min(max(static_cast<int64_t>(offsets[g + 1]), r0), M);
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) grouped_kernel(const Params p) {
  __shared__ float sa[TK][TM + 4], sw[TK][TN + 4];
  const int g = blockIdx.y, n0 = blockIdx.x * TN;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  O* C = static_cast<O*>(p.C);
  if (g == p.groups) {  // rows of no group
    const int64_t lo = min(max(static_cast<int64_t>(p.offsets[0]), int64_t(0)), p.M);
    const int64_t hi = min(max(static_cast<int64_t>(p.offsets[p.groups]), int64_t(0)), p.M);
    for (int64_t i = threadIdx.x; i < p.M * TN; i += 256) {
      const int64_t r = i / TN;
      const int n = n0 + static_cast<int>(i % TN);
      if ((r < lo || r >= hi) && n < p.N) put(C + r * p.ldc + n, 0.0f);
    }
    return;
  }
  int64_t r0, r1;
  group_rows_of(p.offsets, g, p.M, r0, r1);
  const T* A = static_cast<const T*>(p.A);
  const T* W = static_cast<const T*>(p.W) + static_cast<int64_t>(g) * p.stride_w;
  for (int64_t m0 = r0; m0 < r1; m0 += TM) {
    float level[kMaxLevels][4][4], node[4][4] = {};
    int in_group = 0;
    unsigned closed = 0;
    for (int l = 0; l < p.T; ++l) {
      float acc[4][4] = {};
      const int k1 = min((l + 1) * p.leaf, p.K);
      for (int k0 = l * p.leaf; k0 < k1; k0 += TK) {
        for (int i = threadIdx.x; i < TM * TK; i += 256) {
          const int m = i / TK, k = i % TK;
          sa[k][m] = (m0 + m < r1 && k0 + k < k1) ? f32(A[(m0 + m) * p.lda + k0 + k]) : 0.0f;
          sw[k][m] = (n0 + m < p.N && k0 + k < k1)
                         ? f32(p.w_n_contiguous ? W[static_cast<int64_t>(k0 + k) * p.ldw + n0 + m]
                                                : W[static_cast<int64_t>(n0 + m) * p.ldw + k0 + k]) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < TK; ++k)
          for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sw[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
      }
      // level 0: F leaves left to right; above it a binary tree
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) node[i][j] = in_group ? node[i][j] + acc[i][j] : acc[i][j];
      if (++in_group < p.F) continue;
      in_group = 0;
      int lvl = 0;
      for (unsigned c = closed++; c & 1u; c >>= 1, ++lvl)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) node[i][j] = level[lvl][i][j] + node[i][j];
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) level[lvl][i][j] = node[i][j];
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j)
        if (m0 + ty * 4 + i < r1 && n0 + tx * 4 + j < p.N) put(C + (m0 + ty * 4 + i) * p.ldc + n0 + tx * 4 + j, node[i][j]);
  }
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) wgrad_kernel(const T* dC, const T* A, O* dW, const int32_t* offsets, int64_t M, int N,
                                                    int K, int64_t lddc, int64_t lda) {
  __shared__ float sd[TK][TN + 4], sa[TK][TM + 4];
  const int k0 = blockIdx.x * TM, n0 = blockIdx.y * TN, g = blockIdx.z;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int64_t r0, r1;
  group_rows_of(offsets, g, M, r0, r1);
  float acc[4][4] = {};
  for (int64_t r = r0; r < r1; r += TK) {
    for (int i = threadIdx.x; i < TM * TK; i += 256) {
      const int c = i % TM, m = i / TM;
      sd[m][c] = (r + m < r1 && n0 + c < N) ? f32(dC[(r + m) * lddc + n0 + c]) : 0.0f;
      sa[m][c] = (r + m < r1 && k0 + c < K) ? f32(A[(r + m) * lda + k0 + c]) : 0.0f;
    }
    __syncthreads();
    for (int m = 0; m < TK; ++m)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sd[m][ty * 4 + i], sa[m][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (n0 + ty * 4 + i < N && k0 + tx * 4 + j < K)
        put(dW + (static_cast<int64_t>(g) * N + n0 + ty * 4 + i) * K + k0 + tx * 4 + j, acc[i][j]);
}

template <typename T, typename O>
int launch(const Params& p, cudaStream_t stream) {
  const dim3 grid((p.N + TN - 1) / TN, p.groups + (p.outside ? 1 : 0));
  grouped_kernel<T, O><<<grid, 256, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "grouped_kernel launch");
}

template <typename T, typename O>
int launch_wgrad(const void* dC, const void* A, void* dW, const int32_t* offsets, int64_t M, int N, int K, int groups,
                 int64_t lddc, int64_t lda, cudaStream_t stream) {
  const dim3 grid((K + TM - 1) / TM, (N + TN - 1) / TN, groups);
  wgrad_kernel<T, O><<<grid, 256, 0, stream>>>(static_cast<const T*>(dC), static_cast<const T*>(A), static_cast<O*>(dW), offsets,
                                               M, N, K, lddc, lda);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "wgrad_kernel launch");
}

bool bad_align(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_common(const char* what, int64_t M, int N, int K, int groups, int dtype, int out_dtype) {
  char msg[160];
  if (dtype != TBIK_DTYPE_BF16 && dtype != TBIK_DTYPE_FP16) {
    snprintf(msg, sizeof(msg), "%s supports bf16 and fp16 operands", what);
    return set_error(TBIK_ERR_DTYPE, msg);
  }
  if (out_dtype != dtype && out_dtype != TBIK_DTYPE_FP32) {
    snprintf(msg, sizeof(msg), "%s: the result has the operand type or fp32", what);
    return set_error(TBIK_ERR_DTYPE, msg);
  }
  if (M < 0 || M >= (int64_t(1) << 31) || N < 0 || K <= 0) {
    snprintf(msg, sizeof(msg), "%s: M in 0 .. 2^31 - 1, N >= 0, K > 0", what);
    return set_error(TBIK_ERR_SHAPE, msg);
  }
  if (groups < 1 || groups > TBIK_MAX_GROUPS) {
    snprintf(msg, sizeof(msg), "%s: 1 .. %d groups", what, TBIK_MAX_GROUPS);
    return set_error(TBIK_ERR_SHAPE, msg);
  }
  return TBIK_OK;
}

}  // namespace

int grouped_gemm(const void* A, const void* W, void* C, const int32_t* offsets, int64_t M, int N, int K, int groups,
                 int64_t lda, int64_t ldw, int64_t stride_w, int64_t ldc, int w_layout, int dtype, int out_dtype, int leaf,
                 int outside, int max_ctas, cudaStream_t stream) {
  int rc = check_common("tbik_grouped_gemm", M, N, K, groups, dtype, out_dtype);
  if (rc != TBIK_OK) return rc;
  if (w_layout != TBIK_W_K_CONTIGUOUS && w_layout != TBIK_W_N_CONTIGUOUS)
    return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm: unknown layout of W");
  if (leaf < 0 || leaf % 64 != 0 || (leaf > 0 && K % leaf != 0))
    return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: leaf must be 0 or a multiple of 64 that divides K");
  int T = 1, F = 1, L = 1;
  if (leaf > 0) (void)tree_shape(K, leaf, &T, &F, &L);
  if (L > 15) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: at most 15 tree levels: use a wider leaf");
  if (M == 0 || N == 0) return TBIK_OK;
  if (!A || !W || !C || !offsets) return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm: null pointer");
  const int64_t w_row = w_layout == TBIK_W_K_CONTIGUOUS ? K : N, w_rows = w_layout == TBIK_W_K_CONTIGUOUS ? N : K;
  if (lda < K || ldw < w_row || ldc < N || (groups > 1 && stride_w < (w_rows - 1) * ldw + w_row))
    return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: stride smaller than what it steps over");
  if (bad_align(A) || bad_align(W) || lda % 8 || ldw % 8 || stride_w % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm: A and W must be 16-byte aligned with strides that are multiples of 8 elements");
  const Params p{A, W, C, offsets, M, N, K, groups, lda, ldw, stride_w, ldc, w_layout, leaf > 0 ? leaf : K, T, F, L, outside};
  (void)max_ctas;
  if (dtype == TBIK_DTYPE_BF16)
    return out_dtype == TBIK_DTYPE_FP32 ? launch<__nv_bfloat16, float>(p, stream) : launch<__nv_bfloat16, __nv_bfloat16>(p, stream);
  return out_dtype == TBIK_DTYPE_FP32 ? launch<__half, float>(p, stream) : launch<__half, __half>(p, stream);
}

int grouped_gemm_wgrad(const void* dC, const void* A, void* dW, const int32_t* offsets, int64_t M, int N, int K, int groups,
                       int64_t lddc, int64_t lda, int dtype, int out_dtype, int max_ctas, cudaStream_t stream) {
  int rc = check_common("tbik_grouped_gemm_wgrad", M, N, K, groups, dtype, out_dtype);
  if (rc != TBIK_OK || N == 0) return rc;
  if (!dC || !A || !dW || !offsets) return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm_wgrad: null pointer");
  if (lddc < N || lda < K) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm_wgrad: leading dimension smaller than the row");
  if (bad_align(A) || bad_align(dC) || lda % 8 || lddc % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm_wgrad: operands must be 16-byte aligned with row strides that are multiples of 8 elements");
  (void)max_ctas;
  if (dtype == TBIK_DTYPE_BF16)
    return out_dtype == TBIK_DTYPE_FP32
               ? launch_wgrad<__nv_bfloat16, float>(dC, A, dW, offsets, M, N, K, groups, lddc, lda, stream)
               : launch_wgrad<__nv_bfloat16, __nv_bfloat16>(dC, A, dW, offsets, M, N, K, groups, lddc, lda, stream);
  return out_dtype == TBIK_DTYPE_FP32 ? launch_wgrad<__half, float>(dC, A, dW, offsets, M, N, K, groups, lddc, lda, stream)
                                      : launch_wgrad<__half, __half>(dC, A, dW, offsets, M, N, K, groups, lddc, lda, stream);
}

}  // namespace tbik
