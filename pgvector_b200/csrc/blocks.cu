// blocks.cu - E4M3 with one FP32 scale per block of 128: the quantizer and the
// product of two operands in that form (AnnB200QuantizeBlocks,
// AnnB200MatmulBlocks).
#include <cuda_fp8.h>

#include <algorithm>

#include "ops.cuh"

namespace annb200 {
namespace {

constexpr uint32_t kBlock = 128;

// A block's scale and its inverse from absmax's bits (integer order keeps a
// NaN above everything): 448 / a, a at least 2^-100; 0 gives scale 1.
__device__ __forceinline__ float block_scale(uint32_t bits, float &inverse) {
  const float a = bits == 0 ? 448.0f : (bits < 0x0d800000u ? __uint_as_float(0x0d800000u) : __uint_as_float(bits));
  inverse = __fdiv_rn(448.0f, a);
  return __fdiv_rn(a, 448.0f);
}

__device__ __forceinline__ uint8_t e4m3_code(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// One block of the output grid a 1 x 128 or 128 x 128 block, 128 threads.
template <typename T>
__global__ void __launch_bounds__(128) quantize(const T *x, uint64_t stride, uint64_t m, uint32_t k, uint32_t height,
                                                uint8_t *codes, uint64_t code_stride, float *scales) {
  const uint32_t kb = (k + kBlock - 1) / kBlock;
  const uint64_t rb = blockIdx.x / kb;
  const uint32_t b = (uint32_t)(blockIdx.x % kb);
  const uint64_t r0 = rb * height, r1 = min(m, r0 + height);
  const uint32_t c = b * kBlock + threadIdx.x;
  const uint32_t k16 = (k + 15) / 16 * 16;
  __shared__ uint32_t top[4];
  uint32_t bits = 0;
  if (c < k)
    for (uint64_t r = r0; r < r1; r++) bits = max(bits, __float_as_uint(to_float(x[r * stride + c])) & 0x7fffffffu);
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = bits;
  __syncthreads();
  bits = max(max(top[0], top[1]), max(top[2], top[3]));
  float inverse;
  const float scale = block_scale(bits, inverse);
  if (threadIdx.x == 0) scales[rb * kb + b] = scale;
  if (c < k16)
    for (uint64_t r = r0; r < r1; r++)
      codes[r * code_stride + c] = c < k ? e4m3_code(__fmul_rn(to_float(x[r * stride + c]), inverse)) : 0;
}

template <typename T>
__global__ void __launch_bounds__(256)
    matmul(const uint8_t *a, uint64_t a_stride, const float *a_scales, uint32_t a_shift, const uint8_t *b,
           uint64_t b_stride, const float *b_scales, uint32_t b_shift, uint64_t m, uint64_t n, uint32_t k, T *out,
           uint64_t out_stride) {
  __shared__ float as[16][68], bs[16][68];
  const uint64_t m0 = (uint64_t)blockIdx.y * 64, n0 = (uint64_t)blockIdx.x * 64;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  const uint32_t kb = (k + kBlock - 1) / kBlock;
  float sum[4][4] = {};
  for (uint32_t blk = 0; blk < kb; blk++) {
    float acc[4][4] = {};
    const uint32_t kend = min(k, (blk + 1) * kBlock);
    for (uint32_t k0 = blk * kBlock; k0 < kend; k0 += 16) {
      for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i / 16, c = i % 16;
        as[c][r] = m0 + r < m && k0 + c < kend ? e4m3_value(a[(m0 + r) * a_stride + k0 + c]) : 0.0f;
        bs[c][r] = n0 + r < n && k0 + c < kend ? e4m3_value(b[(n0 + r) * b_stride + k0 + c]) : 0.0f;
      }
      __syncthreads();
      for (int c = 0; c < 16; c++)
        for (int i = 0; i < 4; i++)
          for (int j = 0; j < 4; j++) acc[i][j] = fmaf(as[c][tm * 4 + i], bs[c][tn * 4 + j], acc[i][j]);
      __syncthreads();
    }
    for (int i = 0; i < 4; i++)
      for (int j = 0; j < 4; j++) {
        const uint64_t r = m0 + tm * 4 + i, c = n0 + tn * 4 + j;
        if (r < m && c < n)
          sum[i][j] += acc[i][j] * (a_scales[(r >> a_shift) * kb + blk] * b_scales[(c >> b_shift) * kb + blk]);
      }
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const uint64_t r = m0 + tm * 4 + i, c = n0 + tn * 4 + j;
      if (r < m && c < n) out[r * out_stride + c] = from_float<T>(sum[i][j]);
    }
}

}  // namespace
}  // namespace annb200

using namespace annb200;

extern "C" int AnnB200QuantizeBlocks(uint32_t dtype, const void *x, uint64_t stride, uint64_t m, uint32_t k,
                                     uint32_t square, uint8_t *codes, uint64_t code_stride, float *scales,
                                     void *stream) {
  if (!op_dtype(dtype)) return report_error(OP_INVALID, "type %u", dtype);
  if (m > 0x7fffffffull || k > (1u << 20)) return report_error(OP_INVALID, "more than 2^31 rows or 2^20 columns");
  if (m == 0 || k == 0) return OP_OK;
  if (!x || !codes || !scales) return report_error(OP_INVALID, "NULL pointer");
  if (stride < k || code_stride < k || code_stride % 16 || reinterpret_cast<uintptr_t>(codes) % 16)
    return report_error(OP_INVALID, "rows overlap, or code rows are not 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint32_t kb = (k + kBlock - 1) / kBlock, height = square ? kBlock : 1;
  const uint64_t blocks = (m + height - 1) / height * kb;
  if (blocks > 0x7fffffffull) return report_error(OP_INVALID, "more than 2^31 blocks");
  switch (dtype) {
    case ANNB200_F32:
      quantize<<<(unsigned)blocks, 128, 0, st>>>(static_cast<const float *>(x), stride, m, k, height, codes,
                                                 code_stride, scales);
      break;
    case ANNB200_F16:
      quantize<<<(unsigned)blocks, 128, 0, st>>>(static_cast<const __half *>(x), stride, m, k, height, codes,
                                                 code_stride, scales);
      break;
    default:
      quantize<<<(unsigned)blocks, 128, 0, st>>>(static_cast<const __nv_bfloat16 *>(x), stride, m, k, height, codes,
                                                 code_stride, scales);
  }
  return op_launched("quantize blocks", 1);
}

extern "C" int AnnB200MatmulBlocks(const uint8_t *a, uint64_t a_stride, const float *a_scales, uint32_t a_square,
                                   const uint8_t *b, uint64_t b_stride, const float *b_scales, uint32_t b_square,
                                   uint64_t m, uint64_t n, uint32_t k, uint32_t out_dtype, void *out,
                                   uint64_t out_stride, void *stream) {
  if (!op_dtype(out_dtype)) return report_error(OP_INVALID, "output type %u", out_dtype);
  if (m > 0x7fffffffull || n > 0x7fffffffull || k > (1u << 20))
    return report_error(OP_INVALID, "more than 2^31 rows or 2^20 columns");
  if (m == 0 || n == 0) return OP_OK;
  if (!out || out_stride < n) return report_error(OP_INVALID, "NULL output, or its rows overlap");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k == 0) {
    const cudaError_t e = cudaMemset2DAsync(out, out_stride * op_bytes(out_dtype), 0, n * op_bytes(out_dtype), m, st);
    return e == cudaSuccess ? OP_OK : report_error(OP_BACKEND_ERROR, "matmul blocks: %s", cudaGetErrorString(e));
  }
  if (!a || !a_scales || !b || !b_scales) return report_error(OP_INVALID, "NULL pointer");
  if (a_stride < k || b_stride < k || a_stride % 16 || b_stride % 16 || reinterpret_cast<uintptr_t>(a) % 16 ||
      reinterpret_cast<uintptr_t>(b) % 16)
    return report_error(OP_INVALID, "rows of codes overlap, or are not 16-byte aligned");
  const uint32_t sa = a_square ? 7 : 0, sb = b_square ? 7 : 0;
  // the grid's y dimension takes 65,535 tiles: more rows go in several launches
  const uint64_t rows = 65535ull * 64;
  unsigned long long launches = 0;
  for (uint64_t r = 0; r < m; r += rows) {
    const uint64_t mm = std::min(rows, m - r);
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((mm + 63) / 64));
    const uint8_t *ar = a + r * a_stride;
    const float *as = a_scales + (r >> sa) * ((k + kBlock - 1) / kBlock);
    const uint64_t o = r * out_stride;
    switch (out_dtype) {
      case ANNB200_F32:
        matmul<<<grid, 256, 0, st>>>(ar, a_stride, as, sa, b, b_stride, b_scales, sb, mm, n, k,
                                     static_cast<float *>(out) + o, out_stride);
        break;
      case ANNB200_F16:
        matmul<<<grid, 256, 0, st>>>(ar, a_stride, as, sa, b, b_stride, b_scales, sb, mm, n, k,
                                     static_cast<__half *>(out) + o, out_stride);
        break;
      default:
        matmul<<<grid, 256, 0, st>>>(ar, a_stride, as, sa, b, b_stride, b_scales, sb, mm, n, k,
                                     static_cast<__nv_bfloat16 *>(out) + o, out_stride);
    }
    launches++;
  }
  return op_launched("matmul blocks", launches);
}
