// ops.cuh - what the operator kernels (loss.cu, blocks.cu) share: operand
// types, conversions, argument checks' statuses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/annb200.h"
#include "internal.cuh"

namespace annb200 {

enum OpStatus { OP_OK = 0, OP_INVALID = 1, OP_UNSUPPORTED = 2, OP_NOMEM = 4, OP_BACKEND_ERROR = 5 };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline bool op_dtype(uint32_t dtype) { return dtype == ANNB200_F32 || dtype == ANNB200_F16 || dtype == ANNB200_BF16; }
inline uint32_t op_bytes(uint32_t dtype) { return dtype == ANNB200_F32 ? 4 : 2; }

inline int op_launched(const char *what, unsigned long long kernels) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return report_error(e == cudaErrorMemoryAllocation ? OP_NOMEM : OP_BACKEND_ERROR, "%s: %s", what,
                        cudaGetErrorString(e));
  count_launches(kernels);
  return OP_OK;
}

// C[m][n] = sum_k A(m, k) B(n, k) in FP32 on CUDA cores: 64 x 64 tiles, 256
// threads of 4 x 4 sums. A, B: float (row, k); out(m, n, sum) for m < M, n < N.
constexpr int kSimtTile = 64, kSimtK = 16;
template <typename LA, typename LB, typename E>
__global__ void __launch_bounds__(256) simt_gemm(LA a, LB b, int64_t M, int64_t N, int64_t K, E out) {
  __shared__ float as[kSimtK][kSimtTile + 4], bs[kSimtK][kSimtTile + 4];
  const int64_t m0 = (int64_t)blockIdx.y * kSimtTile, n0 = (int64_t)blockIdx.x * kSimtTile;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += kSimtK) {
    for (int i = threadIdx.x; i < kSimtTile * kSimtK; i += 256) {
      const int r = i / kSimtK, k = i % kSimtK;
      as[k][r] = m0 + r < M && k0 + k < K ? a(m0 + r, k0 + k) : 0.0f;
      bs[k][r] = n0 + r < N && k0 + k < K ? b(n0 + r, k0 + k) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSimtK; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(as[k][tm * 4 + i], bs[k][tn * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++)
      if (m0 + tm * 4 + i < M && n0 + tn * 4 + j < N) out(m0 + tm * 4 + i, n0 + tn * 4 + j, acc[i][j]);
}
template <typename LA, typename LB, typename E>
void launch_simt_gemm(LA a, LB b, int64_t M, int64_t N, int64_t K, E out, cudaStream_t st) {
  const dim3 grid((unsigned)((N + kSimtTile - 1) / kSimtTile), (unsigned)((M + kSimtTile - 1) / kSimtTile));
  simt_gemm<<<grid, 256, 0, st>>>(a, b, M, N, K, out);
}

}  // namespace annb200
