// ops.cuh - what the operator kernels (loss.cu, blocks.cu) share: operand
// types, conversions, argument checks' statuses.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

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

// Two values rounded to a 16-bit type, packed.
template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 16 bytes of T from FP32.
__device__ __forceinline__ uint4 pack_chunk(const float *v, float *) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <typename T> __device__ __forceinline__ uint4 pack_chunk(const float *v, T *) {
  return make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]), pack16<T>(v[6], v[7]));
}

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

// A call's kernels after its first start while the one before still runs, get
// their setup done, and wait for its end before they touch memory: of a product
// of a few tiles (5.7 us) 1.2 us are setup, and each launch adds a few more (loss
// and gradients of one query and 1,000 rows, 10 kernels: 70 -> 62 us). Every
// kernel of a chain waits, so each starts its work after all before it.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... Params, typename... Args>
cudaError_t launch_chained(bool after, void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem,
                           cudaStream_t st, Args... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// The limit of a pipeline wait (scan_tc.cu).
uint64_t pipeline_wait_ns();

// A tensor map of an operand (shard.cu): boxes of 128 bytes x box_rows rows, 128-byte swizzle.
bool encode_operand_map(CUtensorMap *map, uint32_t bytes, const void *base, uint64_t inner, uint64_t outer,
                        uint64_t pitch, uint32_t box_rows);

// FP32 sums [planes][outer][inner] in boxes of 32 values x 32 rows (shard.cu).
bool encode_sums_map(CUtensorMap *map, void *base, uint64_t inner, uint64_t outer, uint64_t planes, uint64_t pitch);

// SMs of the current device (a device's number never changes: asked once each).
inline int op_sms() {
  static std::atomic<int> known[64];   // (calls come from any thread)
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 0;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace annb200
