// blocks.cu - E4M3 with one FP32 scale per block of 128: the quantizer and the
// product of two operands in that form (AnnB200QuantizeBlocks,
// AnnB200MatmulBlocks).
//
// The product has two kernels. With up to 8 rows in a (single queries) it is
// bound by reading b once: a warp 16 rows of b, straight into registers. Above
// that the pairs of SMs of pair_gemm.cuh: a K block of 128 is one sum in tensor memory,
// which the epilogue takes out, scales and adds up in FP32 registers while the
// next block's products run.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "pair_gemm.cuh"

namespace annb200 {
namespace {

constexpr uint32_t kBlock = 128;

// ---------------------------------------------------------------- quantizer

// A block's scale and its inverse from absmax's bits (integer order keeps a
// NaN above everything): 448 / a, a at least 2^-100; 0 gives scale 1.
__device__ __forceinline__ float block_scale(uint32_t bits, float &inverse) {
  const float a = bits == 0 ? 448.0f : (bits < 0x0d800000u ? __uint_as_float(0x0d800000u) : __uint_as_float(bits));
  inverse = __fdiv_rn(448.0f, a);
  return __fdiv_rn(a, 448.0f);
}

// 8 values of a row from column c on (c % 8 == 0), zero past k. vec: rows are 16-byte aligned.
template <typename T> struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *row, uint32_t c, uint32_t k, bool vec) {
    if (vec && c + 8 <= k) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; j++) w[j] = __ldcs(reinterpret_cast<const uint4 *>(row + c) + j);
    } else {
      alignas(16) T t[8];   // (read back 16 bytes at a time)
#pragma unroll
      for (int j = 0; j < 8; j++) t[j] = c + j < k ? row[c + j] : from_float<T>(0.0f);
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; j++) w[j] = reinterpret_cast<const uint4 *>(t)[j];
    }
  }
};
// The largest magnitude by its bits, whose integer order keeps a NaN above
// everything; 16-bit types two at a time until the end.
template <typename T> __device__ __forceinline__ uint32_t join_bits(uint32_t a, uint32_t b) {
  return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b);
}
template <typename T> __device__ __forceinline__ uint32_t largest_bits(const Eight<T> &e) {
  constexpr uint32_t MASK = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  uint32_t b = 0;
#pragma unroll
  for (int j = 0; j < (int)sizeof(T) / 2; j++)
    b = join_bits<T>(b, join_bits<T>(join_bits<T>(e.w[j].x & MASK, e.w[j].y & MASK),
                                     join_bits<T>(e.w[j].z & MASK, e.w[j].w & MASK)));
  return b;
}
// The bits of the FP32 value of that magnitude.
__device__ __forceinline__ uint32_t float_bits(uint32_t b, const float *) { return b; }
__device__ __forceinline__ uint32_t float_bits(uint32_t b, const __half *) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(b & 0xffffu, b >> 16))));
}
__device__ __forceinline__ uint32_t float_bits(uint32_t b, const __nv_bfloat16 *) { return max(b & 0xffffu, b >> 16) << 16; }

__device__ __forceinline__ float2 two_floats(uint32_t w, const __half *) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 two_floats(uint32_t w, const __nv_bfloat16 *) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// The codes of two values, rounded to nearest (ties to even) by the hardware's conversion.
__device__ __forceinline__ uint32_t codes2(float2 v, float inverse) {
  return __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(v.x, inverse), __fmul_rn(v.y, inverse)), __NV_SATFINITE,
                                  __NV_E4M3);
}
__device__ __forceinline__ uint2 codes8(const Eight<float> &e, float inverse) {
  auto four = [&](const uint4 &w) {
    return codes2(make_float2(__uint_as_float(w.x), __uint_as_float(w.y)), inverse) |
           (codes2(make_float2(__uint_as_float(w.z), __uint_as_float(w.w)), inverse) << 16);
  };
  return make_uint2(four(e.w[0]), four(e.w[1]));
}
template <typename T> __device__ __forceinline__ uint2 codes8(const Eight<T> &e, float inverse) {
  auto four = [&](uint32_t a, uint32_t b) {
    return codes2(two_floats(a, static_cast<T *>(nullptr)), inverse) |
           (codes2(two_floats(b, static_cast<T *>(nullptr)), inverse) << 16);
  };
  return make_uint2(four(e.w[0].x, e.w[0].y), four(e.w[0].z, e.w[0].w));
}

// Blocks of 1 x 128: 16 lanes a block, 8 values a lane, read once and kept in
// registers; a warp 8 blocks, their loads all in flight. Bound by memory if the
// instructions are few: lane l of a half works out the scale of the half's
// block l % 4, so the two divisions are done once for the 8. 1,000,000 x 768
// FP16: 417 us, 5.6 TB/s (85 % of a copy's rate); 500,000 x 768 FP32 288 us,
// 6.7 TB/s; with the divisions in every lane and FP32 compares 901 us.
constexpr int kQuantUnits = 4;
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows(const T *x, uint64_t stride, uint64_t blocks, uint32_t k,
                                                     uint32_t kb, uint32_t rows2, uint32_t blocks2, uint8_t *codes,
                                                     uint64_t code_stride, float *scales) {
  const uint32_t lane = threadIdx.x & 15, half = (threadIdx.x >> 4) & 1;
  const bool vec = stride % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const uint32_t k16 = (k + 15) / 16 * 16;
  // this half's blocks: u0, u0 + 2, u0 + 4, u0 + 6
  const uint64_t u0 = ((uint64_t)blockIdx.x * 8 + threadIdx.x / 32) * (2 * kQuantUnits) + half;
  Eight<T> e[kQuantUnits];
  uint32_t col[kQuantUnits];
  uint64_t row = blocks < 0x80000000ull ? (uint32_t)u0 / kb : u0 / kb;
  uint32_t b = (uint32_t)(u0 - row * kb);
  uint8_t *to[kQuantUnits];
#pragma unroll
  for (int u = 0; u < kQuantUnits; u++) {
    col[u] = b * kBlock + lane * 8;
    to[u] = codes + row * code_stride + col[u];
    if (u0 + 2 * u < blocks) e[u].load(x + row * stride, col[u], k, vec);
    // two blocks on: rows2 whole rows and blocks2 blocks
    row += rows2;
    b += blocks2;
    if (b >= kb) {
      b -= kb;
      row++;
    }
  }
  uint32_t bits[kQuantUnits];
#pragma unroll
  for (int u = 0; u < kQuantUnits; u++) {
    bits[u] = u0 + 2 * u < blocks ? largest_bits(e[u]) : 0;
#pragma unroll
    for (int d = 8; d; d >>= 1) bits[u] = join_bits<T>(bits[u], __shfl_xor_sync(0xffffffffu, bits[u], d));
  }
  const uint32_t mine = (lane & 2) ? ((lane & 1) ? bits[3] : bits[2]) : ((lane & 1) ? bits[1] : bits[0]);
  float inverse;
  const float scale = block_scale(float_bits(mine, static_cast<T *>(nullptr)), inverse);
  if (lane < kQuantUnits && u0 + 2 * lane < blocks) scales[u0 + 2 * lane] = scale;
#pragma unroll
  for (int u = 0; u < kQuantUnits; u++) {
    const float inv = __shfl_sync(0xffffffffu, inverse, u, 16);
    if (u0 + 2 * u < blocks && col[u] < k16) *reinterpret_cast<uint2 *>(to[u]) = codes8(e[u], inv);
  }
}

// Blocks of 128 x 128: a CTA a block, 8 rows x 8 values a thread in registers.
// 65,537 x 1,000 bf16: 34 us, 5.8 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) quantize_square(const T *x, uint64_t stride, uint64_t m, uint32_t k, uint32_t kb,
                                                       uint8_t *codes, uint64_t code_stride, float *scales) {
  const uint32_t lane = threadIdx.x & 15;
  const bool vec = stride % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const uint32_t k16 = (k + 15) / 16 * 16;
  const uint64_t r0 = (uint64_t)(blockIdx.x / kb) * kBlock + threadIdx.x / 16;
  const uint32_t c = blockIdx.x % kb * kBlock + lane * 8;
  Eight<T> e[8];
#pragma unroll
  for (int u = 0; u < 8; u++)
    if (r0 + 16 * u < m) e[u].load(x + (r0 + 16 * u) * stride, c, k, vec);
  uint32_t bits = 0;
#pragma unroll
  for (int u = 0; u < 8; u++)
    if (r0 + 16 * u < m) bits = join_bits<T>(bits, largest_bits(e[u]));
  __shared__ uint32_t top[8];
  bits = __reduce_max_sync(0xffffffffu, float_bits(bits, static_cast<T *>(nullptr)));
  if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = bits;
  __syncthreads();
  bits = 0;
#pragma unroll
  for (int u = 0; u < 8; u++) bits = max(bits, top[u]);
  float inverse;
  const float scale = block_scale(bits, inverse);
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
  if (c >= k16) return;
#pragma unroll
  for (int u = 0; u < 8; u++)
    if (r0 + 16 * u < m) *reinterpret_cast<uint2 *>(codes + (r0 + 16 * u) * code_stride + c) = codes8(e[u], inverse);
}

template <typename T>
void launch_quantize(const T *x, uint64_t stride, uint64_t m, uint32_t k, bool square, uint8_t *codes,
                     uint64_t code_stride, float *scales, cudaStream_t st) {
  const uint32_t kb = (k + kBlock - 1) / kBlock;
  if (square) {
    quantize_square<<<(unsigned)((m + kBlock - 1) / kBlock * kb), 256, 0, st>>>(x, stride, m, k, kb, codes,
                                                                               code_stride, scales);
  } else {
    const uint64_t blocks = m * kb;
    quantize_rows<<<(unsigned)((blocks + 16 * kQuantUnits - 1) / (16 * kQuantUnits)), 256, 0, st>>>(
        x, stride, blocks, k, kb, 2 / kb, 2 % kb, codes, code_stride, scales);
  }
}

// ---------------------------------------------------------------- product, few rows of a

struct Operands {
  const uint8_t *a, *b;
  uint64_t a_stride, b_stride;
  const float *a_scales, *b_scales;
  uint32_t a_shift, b_shift;   // 7 for square blocks: rows / 128
  uint64_t m, n;
  uint32_t k, kb;
  uint64_t out_stride;
};

// 16 codes of a row from column c on; those past k are zero.
__device__ __forceinline__ uint4 load16(const uint8_t *row, uint32_t c, uint32_t k) {
  if (c >= k) return make_uint4(0, 0, 0, 0);
  uint4 w = __ldg(reinterpret_cast<const uint4 *>(row + c));
  if (c + 16 > k) {
    uint32_t *p = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int left = (int)(k - c) - 4 * j;
      if (left < 4) p[j] = left <= 0 ? 0u : p[j] & ((1u << (8 * left)) - 1u);
    }
  }
  return w;
}
// 16 x 8 sums of 32 codes each: the warp-level instruction, whose operands come
// straight from registers (bound by reading b, nothing is gained by staging).
__device__ __forceinline__ void mma_16x8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Up to 8 rows in a: a warp 16 rows of b against all of them, a block of 128 at
// a time. A thread (row l / 4, quarter l % 4) reads 32 codes of rows l / 4 and
// + 8 of b and of row l / 4 of a; which of the 128 a register stands for does
// not matter as long as both operands agree. The block's sums are scaled and
// added up in FP32. SPLIT warps share 16 rows, each every SPLIT-th block, and
// join their sums in shared memory: for few rows of b. 1 x 100,000 x 1024: 24.5
// us, 1 x 1,000,000 x 1024: 195 us (5.3 TB/s, 81 % of a copy's rate); on CUDA
// cores alone, decoding to FP32, 28 us for the first.
constexpr int kFewWarps = 8;
template <int SPLIT, typename T>
__global__ void __launch_bounds__(32 * kFewWarps) matmul_few(const Operands p, T *out) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const uint32_t part = warp % SPLIT;
  const uint64_t n0 = ((uint64_t)blockIdx.x * (kFewWarps / SPLIT) + warp / SPLIT) * 16;
  // rows past the ends read the last one's codes; their results are not stored
  const uint64_t na = min(n0 + r, p.n - 1), nb = min(n0 + r + 8, p.n - 1), m = min((uint64_t)r, p.m - 1);
  const uint8_t *ba = p.b + na * p.b_stride, *bb = p.b + nb * p.b_stride, *a = p.a + m * p.a_stride;
  const float *sba = p.b_scales + (na >> p.b_shift) * p.kb, *sbb = p.b_scales + (nb >> p.b_shift) * p.kb;
  const float *sa0 = p.a_scales + (min((uint64_t)(2 * q), p.m - 1) >> p.a_shift) * p.kb;
  const float *sa1 = p.a_scales + (min((uint64_t)(2 * q + 1), p.m - 1) >> p.a_shift) * p.kb;
  float sum[4] = {};
#pragma unroll 4
  for (uint32_t b = part; b < p.kb; b += SPLIT) {
    const uint32_t c = b * kBlock + q * 32;
    const uint4 xa = load16(ba, c, p.k), ya = load16(ba, c + 16, p.k), xb = load16(bb, c, p.k),
                yb = load16(bb, c + 16, p.k), xm = load16(a, c, p.k), ym = load16(a, c + 16, p.k);
    const float s0 = __ldg(sa0 + b), s1 = __ldg(sa1 + b), ra = __ldg(sba + b), rb = __ldg(sbb + b);
    float d[4] = {};
    mma_16x8(d, xa.x, xb.x, xa.y, xb.y, xm.x, xm.y);
    mma_16x8(d, xa.z, xb.z, xa.w, xb.w, xm.z, xm.w);
    mma_16x8(d, ya.x, yb.x, ya.y, yb.y, ym.x, ym.y);
    mma_16x8(d, ya.z, yb.z, ya.w, yb.w, ym.z, ym.w);
    sum[0] = fmaf(d[0], ra * s0, sum[0]);
    sum[1] = fmaf(d[1], ra * s1, sum[1]);
    sum[2] = fmaf(d[2], rb * s0, sum[2]);
    sum[3] = fmaf(d[3], rb * s1, sum[3]);
  }
  if (SPLIT > 1) {
    __shared__ float4 joined[kFewWarps][32];
    joined[warp][lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (part != 0) return;
    for (int w = 1; w < SPLIT; w++) {
      const float4 v = joined[warp + w][lane];
      sum[0] += v.x;
      sum[1] += v.y;
      sum[2] += v.z;
      sum[3] += v.w;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint64_t n = n0 + r + 8 * (j >> 1);
    const uint32_t i = 2 * q + (j & 1);
    if (n < p.n && i < p.m) out[(uint64_t)i * p.out_stride + n] = from_float<T>(sum[j]);
  }
}

template <int SPLIT, typename T>
cudaError_t launch_few(const Operands &o, T *out, cudaStream_t st) {
  const uint64_t rows = 16 * (kFewWarps / SPLIT);
  matmul_few<SPLIT><<<(unsigned)((o.n + rows - 1) / rows), 32 * kFewWarps, 0, st>>>(o, out);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- product, tensor cores

// The scales of a K block, one a lane and one a column of the tile, for the
// epilogues below: two helper warps bring AHEAD blocks at a time (16 bytes of
// each scale row) into one of two buffers, transposed, so that lanes read
// theirs side by side and columns' can be read several at once.
//   LANES, COLS: scales a block (COLS 2: one for each half of the columns)
//   Order: where scale c of a block is kept, of ROW floats
struct InOrder {
  static constexpr int room(int n) { return n; }
  static __device__ __forceinline__ uint32_t place(uint32_t c) { return c; }
};
template <int LANES_, int COLS_, typename Order = InOrder>
struct ScaleStage {
  static constexpr int LANES = LANES_, COLS = COLS_, ROW = Order::room(LANES + (COLS < 4 ? 4 : COLS)), AHEAD = 4;
  static constexpr int BUFFER = AHEAD * ROW * 4;
  static constexpr int BYTES = 2 * BUFFER + 64;
  uint8_t *scratch;
  uint32_t group = 0;
  __device__ __forceinline__ uint64_t *bars() const { return reinterpret_cast<uint64_t *>(scratch + 2 * BUFFER); }
  __device__ __forceinline__ void init() const {   // full[2], empty[2]
    for (int i = 0; i < 2; i++) {
      mbar_init(bars() + i, 2);
      mbar_init(bars() + 2 + i, kPairEpi);
    }
  }
  // The helpers' part for one item: t = 0 .. 63; row(c): scale c's row of kb blocks.
  template <typename Rows>
  __device__ __forceinline__ bool fill(uint32_t t, const Rows &row_of, uint32_t kb, bool vec, volatile PairBounds *bounds) {
    constexpr int EACH = (LANES + COLS + 63) / 64;
    const float *row[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) row[e] = row_of(min(t + 64 * e, (uint32_t)(LANES + COLS - 1)));
    float4 v[EACH];
    // blocks b0 .. b0 + 3 of each row (past the last: not used), all loads before any use
    auto load = [&](uint32_t b0) {
      if (vec) {
#pragma unroll
        for (int e = 0; e < EACH; e++) v[e] = __ldg(reinterpret_cast<const float4 *>(row[e] + b0));
      } else {
        const uint32_t last = kb - 1;
#pragma unroll
        for (int e = 0; e < EACH; e++)
          v[e] = make_float4(__ldg(row[e] + b0), __ldg(row[e] + min(b0 + 1, last)), __ldg(row[e] + min(b0 + 2, last)),
                             __ldg(row[e] + min(b0 + 3, last)));
      }
    };
    load(0);
    for (uint32_t b0 = 0; b0 < kb; b0 += AHEAD, group++) {
      uint64_t *bar = bars() + (group & 1);
      // (the warp leaves together: a lane that goes on alone would wait for the others below)
      if (!__all_sync(0xffffffffu, pair_wait(bar + 2, ((group >> 1) & 1) ^ 1, bounds))) return false;
      float *at = reinterpret_cast<float *>(scratch + (group & 1) * BUFFER);
#pragma unroll
      for (int e = 0; e < EACH; e++) {
        const uint32_t c = t + 64 * e, to = Order::place(c);
        if (c < LANES + COLS) {
          at[to] = v[e].x;
          at[ROW + to] = v[e].y;
          at[2 * ROW + to] = v[e].z;
          at[3 * ROW + to] = v[e].w;
        }
      }
      __syncwarp();
      if ((t & 31) == 0) mbar_arrive(bar);
      if (b0 + AHEAD < kb) load(b0 + AHEAD);   // under the products of this group
    }
    return true;
  }
  // The epilogue's: shared address of block b's scales, and the end of its use.
  template <typename Sums>
  __device__ __forceinline__ uint32_t take(uint32_t b, Sums &sums) const {
    if (b % AHEAD == 0 && sums.ok)
      sums.ok = __all_sync(0xffffffffu, pair_wait(bars() + (group & 1), (group >> 1) & 1, sums.bounds));
    return smem_u32(scratch) + (group & 1) * BUFFER + (b % AHEAD) * (ROW * 4);
  }
  // (A warp whose waits have run out no longer keeps step with the others: it does not arrive for them.)
  __device__ __forceinline__ void done(uint32_t b, uint32_t kb, bool ok) {
    if (b % AHEAD == AHEAD - 1 || b + 1 == kb) {
      __syncwarp();
      if ((threadIdx.x & 31) == 0 && ok) mbar_arrive(bars() + 2 + (group & 1));
      group++;
    }
  }
};
__device__ __forceinline__ float shared_float(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <typename T>
struct BlocksArgs {
  CUtensorMap a[1], b[1];   // the tile's rows and columns
  uint32_t bn;
  uint32_t mt, nt;          // tiles of a's rows, of b's
  Operands o;
  T *out;
  int boxes;                // out's rows start on 16-byte boundaries: `map` stores boxes
  int ragged;               // and do not end on one: not the last box, which would write past n
  CUtensorMap map;
};
// Scales a and b both 16-byte aligned, and their rows: loads of four blocks.
__device__ __forceinline__ bool scales_vec(const Operands &o) {
  return (o.kb & 3) == 0 &&
         ((reinterpret_cast<uintptr_t>(o.a_scales) | reinterpret_cast<uintptr_t>(o.b_scales)) & 15) == 0;
}

// Up to 128 rows in a: tiles of 256 of b's rows (lanes) x 2 COLS of a's (COLS a
// thread), bound by reading b. A store of a column is 32 of b's rows side by side.
// 16 x 1,000,000 x 1000: 195 us, 5.4 TB/s; 33 x 65,536 x 768: 20 us, where 256
// tiles for 74 clusters and the start show.
template <int COLS, typename T>
struct NarrowOp {
  static constexpr PairKind KIND = PAIR_E4M3;
  static constexpr bool A_MN = false, B_MN = false, A_SAME = false;
  static constexpr int PLANES = 1, MAX_STAGES = 12, CHUNK = 1, HELPERS = 2;
  // a block's sum passes from role to role in about 1,000 clocks, in which b's next blocks arrive
  static constexpr int ACCS = 2 * COLS >= 128 ? 4 : 8;
  using Scales = ScaleStage<128, 2 * COLS>;
  static constexpr int SCRATCH = Scales::BYTES;
  using Args = BlocksArgs<T>;
  static __device__ __forceinline__ uint32_t items(const Args &p) { return p.mt * p.nt; }
  static __device__ __forceinline__ PairItem item(const Args &p, uint32_t i) {
    return {(int32_t)((i / p.mt) * 256), (int32_t)((i % p.mt) * p.bn), 0, p.o.kb, 0};
  }
  static __device__ __forceinline__ void init(uint8_t *scratch) { Scales{scratch}.init(); }
  static __device__ __forceinline__ void help(const Args &p, uint8_t *scratch, uint32_t rank, uint32_t cluster,
                                              uint32_t clusters, volatile PairBounds *bounds) {
    const Operands &o = p.o;
    Scales scales{scratch};
    const bool vec = scales_vec(o);
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      const PairItem w = item(p, i);
      const uint64_t n0 = (uint64_t)w.a_row + rank * 128, m0 = (uint64_t)w.b_row;
      if (!scales.fill(threadIdx.x - 32 * (kPairEpi + 2),
                       [&](uint32_t c) {
                         return c < 128 ? o.b_scales + (min(n0 + c, o.n - 1) >> o.b_shift) * o.kb
                                        : o.a_scales + (min(m0 + c - 128, o.m - 1) >> o.a_shift) * o.kb;
                       },
                       o.kb, vec, bounds))
        return;
    }
  }
  static __device__ __forceinline__ void epilogue(const Args &p, PairSumsOf<ACCS> &sums, uint8_t *scratch, uint32_t rank,
                                                  uint32_t cluster, uint32_t clusters) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2, quad = warp & 3;
    const Operands &o = p.o;
    Scales scales{scratch};
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      float v[COLS];
#pragma unroll
      for (int j = 0; j < COLS; j++) v[j] = 0.0f;
#pragma unroll 1
      for (uint32_t b = 0; b < o.kb; b++) {
        const uint32_t scale = scales.take(b, sums);
        const uint32_t addr = sums.acquire() + half * COLS, cols = scale + (128 + half * COLS) * 4;
        const float ls = shared_float(scale + (quad * 32 + lane) * 4);
        constexpr int STEP = COLS < 32 ? COLS : 32;
#pragma unroll
        for (int c = 0; c < COLS; c += STEP) {
          uint32_t r[STEP];
          if (sums.ok) {
            if constexpr (STEP == 32) TMEM_LD32(addr + c, r);
            else TMEM_LD16(addr + c, r);
            tmem_ld_wait();
            if constexpr (STEP == 32) TMEM_KEEP32(r);
            else TMEM_KEEP16(r);
          }
#pragma unroll
          for (int j = 0; j < STEP; j += 4) {
            float s[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(s[0]), "=f"(s[1]), "=f"(s[2]), "=f"(s[3])
                         : "r"(cols + (c + j) * 4));
#pragma unroll
            for (int u = 0; u < 4; u++) v[c + j + u] = fmaf(__uint_as_float(r[j + u]), s[u] * ls, v[c + j + u]);
          }
        }
        sums.release();
        scales.done(b, o.kb, sums.ok);
      }
      const PairItem w = item(p, i);
      const uint64_t n = (uint64_t)w.a_row + rank * 128 + quad * 32 + lane;   // b's row
      const uint64_t m0 = (uint64_t)w.b_row + half * COLS;                    // a's first row
      if (n >= o.n) continue;
      const float poison = sums.ok ? 0.0f : __uint_as_float(0x7fc00000u);
      T *col = p.out + m0 * o.out_stride + n;
      const int rows = m0 < o.m ? (int)min((uint64_t)COLS, o.m - m0) : 0;
#pragma unroll
      for (int j = 0; j < COLS; j++) {
        if (j < rows) *col = from_float<T>(v[j] + poison);
        col += o.out_stride;
      }
    }
  }
};

// Scales for lanes that hold 8 x 4 patches (below): a thread's 4 rows side by
// side, then each half's columns, a thread's 32 side by side (4 threads of a row
// 36 floats apart: different banks).
struct PatchOrder {
  static constexpr int room(int) { return 128 + 2 * 4 * 36; }
  static __device__ __forceinline__ uint32_t place(uint32_t c) {
    if (c < 128) return (c & ~31u) + (c & 7) * 4 + ((c >> 3) & 3);
    c -= 128;
    return 128 + (c >> 7) * 144 + ((c >> 1) & 3) * 36 + ((c & 127) >> 3) * 2 + (c & 1);
  }
};
__device__ __forceinline__ void shared_float4(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr));
}

// More rows: tiles of 256 of a's rows x 256 of b's, 128 columns a thread's warp.
// b's scales square (UNIFORM): a lane is one of a's rows and has one scale a
// block. Else each value has a scale of its own; columns' scales read by every
// lane would fill the shared-memory port, so the lanes read tensor memory in 8 x
// 4 patches, where a thread has 4 rows and 32 columns: 9 reads of shared memory
// a block. Bound by the epilogue: a block's products and loads alone take 720
// clocks, with the scaling 1,260 (8,191 x 5,000 x 4,096, square: 212 us, 1.58
// PFLOP/s; 219 us a call among calls) and 1,800 (1,024 x 1,000,000 x 1,024: 1,735
// us, 1.21 PFLOP/s, where 2 GB of results go out under it; 1,895 us among calls,
// under the power cap). 16 epilogue warps were no faster.
template <bool UNIFORM, typename T>
struct WideOp {
  static constexpr PairKind KIND = PAIR_E4M3;
  static constexpr bool A_MN = false, B_MN = false, A_SAME = false;
  static constexpr int PLANES = 1, MAX_STAGES = 12, CHUNK = 1, HELPERS = 2, ACCS = 2;
  using Scales = ScaleStage<128, UNIFORM ? 2 : 256, std::conditional_t<UNIFORM, InOrder, PatchOrder>>;
  static constexpr int SCALE_BYTES = (Scales::BYTES + 1023) / 1024 * 1024;
  static constexpr int SCRATCH = SCALE_BYTES + kPairEpi * kBoxBytes;   // (a second box a warp costs a stage: slower)
  using Args = BlocksArgs<T>;
  static __device__ __forceinline__ uint32_t items(const Args &p) { return p.mt * p.nt; }
  static __device__ __forceinline__ PairItem item(const Args &p, uint32_t i) {
    return {(int32_t)((i % p.mt) * 256), (int32_t)((i / p.mt) * 256), 0, p.o.kb, 0};
  }
  static __device__ __forceinline__ void init(uint8_t *scratch) { Scales{scratch}.init(); }
  static __device__ __forceinline__ void help(const Args &p, uint8_t *scratch, uint32_t rank, uint32_t cluster,
                                              uint32_t clusters, volatile PairBounds *bounds) {
    const Operands &o = p.o;
    Scales scales{scratch};
    const bool vec = scales_vec(o);
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      const PairItem w = item(p, i);
      const uint64_t m0 = (uint64_t)w.a_row + rank * 128, n0 = (uint64_t)w.b_row;
      if (!scales.fill(threadIdx.x - 32 * (kPairEpi + 2),
                       [&](uint32_t c) {
                         if (c < 128) return o.a_scales + (min(m0 + c, o.m - 1) >> o.a_shift) * o.kb;
                         const uint64_t n = n0 + (UNIFORM ? (c - 128) * 128 : c - 128);
                         return o.b_scales + (min(n, o.n - 1) >> o.b_shift) * o.kb;
                       },
                       o.kb, vec, bounds))
        return;
    }
  }
  static __device__ __forceinline__ void epilogue(const Args &p, PairSums &sums, uint8_t *scratch, uint32_t rank,
                                                  uint32_t cluster, uint32_t clusters) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2, quad = warp & 3;
    const Operands &o = p.o;
    Scales scales{scratch};
    BoxStore box{scratch + SCALE_BYTES + warp * kBoxBytes};
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      // UNIFORM: v[c] column c of the lane's row. Else v[16 c + 4 g + u], c = 2 h + l: rows 16 l + lane / 4 (u < 2)
      // and + 8, columns 32 h + 8 g + 2 (lane % 4) + u % 2
      float v[128];
#pragma unroll
      for (int j = 0; j < 128; j++) v[j] = 0.0f;
#pragma unroll 1
      for (uint32_t b = 0; b < o.kb; b++) {
        const uint32_t scale = scales.take(b, sums);
        const uint32_t addr = sums.acquire() + half * 128;
        if (sums.ok) {
          // eight (UNIFORM: four) reads of tensor memory, one ahead of what uses it
          constexpr int STEP = UNIFORM ? 32 : 16, STEPS = 128 / STEP;
          uint32_t r[2][STEP];
          auto read = [&](int c, uint32_t(&to)[STEP]) {
            if constexpr (UNIFORM) TMEM_LD32(addr + c * 32, to);
            else TMEM_LD_16X32(addr + (c >> 1) * 32 + ((uint32_t)(c & 1) << 20), to);
          };
          auto wait = [&](uint32_t(&to)[STEP]) {
            tmem_ld_wait();
            if constexpr (UNIFORM) TMEM_KEEP32(to);
            else TMEM_KEEP16(to);
          };
          read(0, r[0]);
          float rows[4];
          f32x2 cols[16];
          if constexpr (UNIFORM) {
            rows[0] = shared_float(scale + (quad * 32 + lane) * 4) * shared_float(scale + (128 + half) * 4);
          } else {
            shared_float4(scale + (quad * 32 + (lane >> 2) * 4) * 4, rows);
#pragma unroll
            for (int k = 0; k < 8; k++)
              asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];"
                           : "=l"(cols[2 * k]), "=l"(cols[2 * k + 1])
                           : "r"(scale + (128 + half * 144 + (lane & 3) * 36 + 4 * k) * 4));
          }
          wait(r[0]);
#pragma unroll
          for (int c = 0; c < STEPS; c++) {
            if (c + 1 < STEPS) read(c + 1, r[(c + 1) & 1]);
            const uint32_t(&t)[STEP] = r[c & 1];
            if constexpr (UNIFORM) {
#pragma unroll
              for (int j = 0; j < 32; j++) v[c * 32 + j] = fmaf(__uint_as_float(t[j]), rows[0], v[c * 32 + j]);
            } else {
              const f32x2 ra = pack2(rows[2 * (c & 1)], rows[2 * (c & 1)]);
              const f32x2 rb = pack2(rows[2 * (c & 1) + 1], rows[2 * (c & 1) + 1]);
#pragma unroll
              for (int g = 0; g < 4; g++) {
                float *o4 = v + c * 16 + g * 4;
                float a0, a1, b0, b1;
                unpack2(mul2(cols[(c >> 1) * 4 + g], ra), a0, a1);
                unpack2(mul2(cols[(c >> 1) * 4 + g], rb), b0, b1);
                o4[0] = fmaf(__uint_as_float(t[4 * g]), a0, o4[0]);
                o4[1] = fmaf(__uint_as_float(t[4 * g + 1]), a1, o4[1]);
                o4[2] = fmaf(__uint_as_float(t[4 * g + 2]), b0, o4[2]);
                o4[3] = fmaf(__uint_as_float(t[4 * g + 3]), b1, o4[3]);
              }
            }
            if (c + 1 < STEPS) wait(r[(c + 1) & 1]);
          }
        }
        sums.release();
        scales.done(b, o.kb, sums.ok);
      }
      const PairItem w = item(p, i);
      const uint32_t m0 = (uint32_t)w.a_row + rank * 128 + quad * 32, n0 = (uint32_t)w.b_row + half * 128;
      if (m0 >= o.m || n0 >= o.n) continue;
      if (!sums.ok) {
#pragma unroll
        for (int j = 0; j < 128; j++) v[j] = __uint_as_float(0x7fc00000u);
      }
      constexpr int BOX = 128 / sizeof(T);   // columns of a box
#pragma unroll
      for (int x = 0; x < 128 / BOX; x++) {
        if (n0 + x * BOX >= o.n) break;
        box.reuse();
        if constexpr (UNIFORM) {
          constexpr int V = 16 / sizeof(T);
#pragma unroll
          for (int c = 0; c < 8; c++) {
            box.put(c, pack_chunk(v + x * BOX + c * V, static_cast<T *>(nullptr)));
          }
        } else {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
              for (int u = 0; u < 4; u++) {
                const float *q = v + (2 * x + u / 2) * 16 + g * 4 + 2 * (u & 1);
                const uint32_t at = (g * 8 + 2 * (lane & 3)) * 4;
                *reinterpret_cast<float2 *>(box.at(8 * u + lane / 4, at >> 4) + (at & 15)) = make_float2(q[0], q[1]);
              }
          } else {
            // 8 x 8 patches, four (a column of the box's 32 rows) at a time: lane l gives the address of row l
#pragma unroll
            for (int g = 0; g < 8; g++) {
              uint32_t q[4];
#pragma unroll
              for (int u = 0; u < 4; u++) {
                const float *w2 = v + (2 * (2 * x + g / 4) + u / 2) * 16 + (g & 3) * 4 + 2 * (u & 1);
                q[u] = pack16<T>(w2[0], w2[1]);
              }
              asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                               smem_u32(box.at(lane, g))),
                           "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                           : "memory");
            }
          }
        }
        if (p.boxes && !(p.ragged && n0 + (x + 1) * BOX > o.n)) {   // (in 16-bit values)
          box.store(&p.map, (int32_t)((n0 + x * BOX) * (sizeof(T) / 2)), (int32_t)m0);
        } else {
          box.copy(p.out + (uint64_t)m0 * o.out_stride + n0 + x * BOX, o.out_stride,
                   (uint32_t)min((uint64_t)32, o.m - m0), (uint32_t)min((uint64_t)BOX, o.n - n0 - x * BOX));
        }
      }
    }
  }
};

template <class Op, typename T>
cudaError_t launch_tiles(const Operands &o, T *out, bool wide, uint32_t bn, int sms, cudaStream_t st) {
  BlocksArgs<T> args = {};
  args.bn = bn;
  args.o = o;
  args.out = out;
  // the tile's 256 rows: a's (wide) or b's; its bn columns: the other's
  args.mt = (uint32_t)((o.m + (wide ? 256 : bn) - 1) / (wide ? 256 : bn));
  args.nt = (uint32_t)((o.n + 255) / 256);
  args.boxes = wide && o.out_stride * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 &&
               o.n * sizeof(T) / 2 <= 0x7fffffffull;
  args.ragged = o.n * sizeof(T) % 16 != 0;
  const bool maps =
      encode_operand_map(args.a, 1, wide ? o.a : o.b, o.k, wide ? o.m : o.n, wide ? o.a_stride : o.b_stride, 128) &&
      encode_operand_map(args.b, 1, wide ? o.b : o.a, o.k, wide ? o.n : o.m, wide ? o.b_stride : o.a_stride, bn / 2) &&
      (!args.boxes ||
       encode_operand_map(&args.map, 2, out, o.n * sizeof(T) / 2, o.m, o.out_stride * sizeof(T), 32));
  if (!maps) return cudaErrorInvalidValue;
  return launch_pair<Op>(args, args.mt * args.nt, sms, st, false);
}

template <typename T>
cudaError_t launch_matmul(const Operands &o, T *out, cudaStream_t st) {
  if (o.m <= 8) {
    // enough warps for every SM, as long as each has blocks of its own
    const uint64_t warps = (o.n + 15) / 16, want = 148 * 16;
    if (warps >= want || o.kb < 2) return launch_few<1>(o, out, st);
    if (warps * 2 >= want || o.kb < 4) return launch_few<2>(o, out, st);
    if (warps * 4 >= want || o.kb < 8) return launch_few<4>(o, out, st);
    return launch_few<8>(o, out, st);
  }
  const int sms = op_sms();
  if (sms < 2) return cudaErrorNoDevice;
  // columns a thread: the fewest that hold a's rows in one tile
  if (o.m <= 32) return launch_tiles<NarrowOp<16, T>>(o, out, false, 32, sms, st);
  if (o.m <= 64) return launch_tiles<NarrowOp<32, T>>(o, out, false, 64, sms, st);
  if (o.m <= 128) return launch_tiles<NarrowOp<64, T>>(o, out, false, 128, sms, st);
  return o.b_shift ? launch_tiles<WideOp<true, T>>(o, out, true, 256, sms, st)
                   : launch_tiles<WideOp<false, T>>(o, out, true, 256, sms, st);
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
  if (m * ((k + kBlock - 1) / kBlock) > 0x7fffffffull * 64)
    return report_error(OP_INVALID, "more than 2^37 blocks");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case ANNB200_F32:
      launch_quantize(static_cast<const float *>(x), stride, m, k, square != 0, codes, code_stride, scales, st);
      break;
    case ANNB200_F16:
      launch_quantize(static_cast<const __half *>(x), stride, m, k, square != 0, codes, code_stride, scales, st);
      break;
    default:
      launch_quantize(static_cast<const __nv_bfloat16 *>(x), stride, m, k, square != 0, codes, code_stride, scales, st);
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
  const Operands o = {a, b, a_stride, b_stride, a_scales, b_scales, a_square ? 7u : 0u, b_square ? 7u : 0u, m, n, k,
                      (k + kBlock - 1) / kBlock, out_stride};
  cudaError_t e;
  switch (out_dtype) {
    case ANNB200_F32: e = launch_matmul(o, static_cast<float *>(out), st); break;
    case ANNB200_F16: e = launch_matmul(o, static_cast<__half *>(out), st); break;
    default: e = launch_matmul(o, static_cast<__nv_bfloat16 *>(out), st);
  }
  if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "matmul blocks: %s", cudaGetErrorString(e));
  return op_launched("matmul blocks", 1);
}
