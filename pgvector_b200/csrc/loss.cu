// loss.cu - softmax loss of queries over all of a shard's rows, and its
// gradients (AnnB200SoftmaxLoss, AnnB200SoftmaxLossGrad).
//
// With l = scale * X W^T (X: nq x d queries, W: n x d rows):
//
//   forward   logits in 256 x 256 tiles on the tensor cores; a tile's epilogue
//             leaves, per query and half tile, the maximum and the sum of
//             exp2 of its 128 logits (in base 2). A reduction joins them.
//   gradient  in pieces of W: the piece's logits again, whose epilogue writes
//             G = grad (exp(l - lse) - onehot) in 16 bits; then dX += G W with
//             the piece's rows split over clusters (FP32 partial sums, each
//             written by one cluster: no atomics) and dW = G^T X. Both read G
//             and W or X as they lie, MN-major where K runs along rows.
//
// FP32 operands are two FP16 terms, x 2^e = high + low (22 bits), and three of
// the four products; e is such that the largest |x| is in [2^14, 2^15): for
// rows and, in the gradient, queries one e an array, since their sums run over
// rows and queries; in the forward call one a query.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "pair_gemm.cuh"

namespace annb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr uint64_t kPartBytes = 256ull << 20;   // the forward call's partial maxima and sums, at most about
constexpr uint64_t kPieceBytes = 512ull << 20;  // G of a piece, where a piece has 8,192 rows by then
constexpr uint32_t kPlanClusters = 74;          // clusters the plan splits for (148 SMs)

enum { MAX_ROWS = 0, MAX_QUERIES = 1, MAX_GRAD = 2 };   // the workspace's maxima (float bits)

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^-e of an array whose largest finite |x| has these bits (header comment).
__device__ __forceinline__ float undo_scale(uint32_t bits) {
  const int e = min(120, max(-120, 14 - ((int)(bits >> 23) - 127)));
  return __uint_as_float((uint32_t)(127 - e) << 23);
}
// The power of two that grad is divided by: at most its largest |value|.
__device__ __forceinline__ float grad_unit(uint32_t bits) {
  return __uint_as_float(max(bits & 0x7f800000u, 0x00800000u));
}
constexpr float kGradScale = 16384.0f;   // G is kept as grad / unit * 2^14 * (p - onehot): below 2^15

__device__ __forceinline__ bool has_target(int64_t t, uint64_t nrows) { return t >= 0 && t < (int64_t)nrows; }

// ---------------------------------------------------------------- laying operands out

// The largest finite |x| of an FP32 array (bits, by atomicMax: any order gives
// the same). Threads cover `tx` 4-value chunks of a row and 256 / tx rows.
__global__ void __launch_bounds__(256) array_max(const float *x, uint64_t stride, uint64_t rows, uint32_t dims,
                                                 uint32_t tx, const int64_t *targets, uint64_t nrows, uint32_t *out) {
  const uint32_t cx = threadIdx.x % tx, ry = threadIdx.x / tx, ty = 256 / tx;
  const bool vec = stride % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  uint32_t best = 0;
  auto take = [&](float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    if (b < 0x7f800000u) best = max(best, b);
  };
  for (uint64_t r = (uint64_t)blockIdx.x * ty + ry; r < rows; r += (uint64_t)gridDim.x * ty) {
    if (targets && !has_target(targets[r], nrows)) continue;
    const float *row = x + r * stride;
    for (uint32_t c = cx * 4; c < dims; c += tx * 4) {
      if (vec && c + 4 <= dims) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(row + c));
        take(v.x);
        take(v.y);
        take(v.z);
        take(v.w);
      } else {
        for (uint32_t j = c; j < min(dims, c + 4); j++) take(row[j]);
      }
    }
  }
  best = __reduce_max_sync(0xffffffffu, best);
  if (threadIdx.x % 32 == 0 && best) atomicMax(out, best);
}

// Per query 2^-e: of its own largest |x| (a warp a query), or the array's.
__global__ void __launch_bounds__(256) query_scales(const float *x, uint64_t stride, uint32_t nq, uint32_t dims,
                                                    const uint32_t *whole, float *scales) {
  const uint32_t q = (blockIdx.x * 256 + threadIdx.x) / 32, lane = threadIdx.x % 32;
  if (q >= nq) return;
  uint32_t best = whole ? *whole : 0;
  if (!whole)
    for (uint32_t c = lane; c < dims; c += 32) {
      const uint32_t b = __float_as_uint(x[q * stride + c]) & 0x7fffffffu;
      if (b < 0x7f800000u) best = max(best, b);
    }
  best = __reduce_max_sync(0xffffffffu, best);
  if (lane == 0) scales[q] = undo_scale(best);
}

__global__ void __launch_bounds__(256) grad_max(const float *grad, const int64_t *targets, uint32_t nq, uint64_t nrows,
                                                uint32_t *out) {
  const uint32_t q = blockIdx.x * 256 + threadIdx.x;
  uint32_t b = 0;
  if (q < nq && has_target(targets[q], nrows)) b = grad ? __float_as_uint(grad[q]) & 0x7fffffffu : 0x3f800000u;
  b = __reduce_max_sync(0xffffffffu, b < 0x7f800000u ? b : 0u);
  if (threadIdx.x % 32 == 0 && b) atomicMax(out, b);
}

// Rows of an operand in the layout TMA reads: `ld` values (a multiple of 8) a
// row, values past dims zero. FP32: two FP16 planes of x * 2^e; an infinity
// becomes NaN (its products with a low term of 0 would be). Queries without a
// target (targets given) become rows of zeros.
template <typename T, typename O, int PLANES>
__global__ void __launch_bounds__(256) pack_rows(const T *x, uint64_t stride, uint64_t rows, uint32_t dims, uint32_t ld,
                                                 uint32_t tx, const int64_t *targets, uint64_t nrows,
                                                 const float *row_scales, const uint32_t *whole, O *out,
                                                 uint64_t plane) {
  const uint32_t cx = threadIdx.x % tx, ry = threadIdx.x / tx, ty = 256 / tx;
  const bool vec = stride % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const float mul = PLANES == 2 && !row_scales ? 1.0f / undo_scale(*whole) : 1.0f;   // powers of two: exact
  for (uint64_t r = (uint64_t)blockIdx.x * ty + ry; r < rows; r += (uint64_t)gridDim.x * ty) {
    const bool zero = targets && !has_target(targets[r], nrows);
    const float s = PLANES == 2 && row_scales ? 1.0f / row_scales[r] : mul;
    const T *row = x + r * stride;
    for (uint32_t c = cx * 8; c < ld; c += tx * 8) {
      alignas(16) T v[8];
      if (!zero && vec && c + 8 <= dims) {
#pragma unroll
        for (int j = 0; j < (int)(8 * sizeof(T) / 16); j++)
          reinterpret_cast<uint4 *>(v)[j] = __ldg(reinterpret_cast<const uint4 *>(row + c) + j);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = !zero && c + j < dims ? row[c + j] : from_float<T>(0.0f);
      }
      alignas(16) O hi[8], lo[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (PLANES == 2) {
          float f = to_float(v[j]) * s;
          if (isinf(f)) f = NAN;
          hi[j] = from_float<O>(f);
          lo[j] = from_float<O>(isnan(f) ? 0.0f : f - to_float(hi[j]));
        } else {
          reinterpret_cast<uint16_t *>(hi)[j] = reinterpret_cast<const uint16_t *>(v)[j];
        }
      }
      *reinterpret_cast<uint4 *>(out + r * ld + c) = *reinterpret_cast<uint4 *>(hi);
      if (PLANES == 2) *reinterpret_cast<uint4 *>(out + plane + r * ld + c) = *reinterpret_cast<uint4 *>(lo);
    }
  }
}

// ---------------------------------------------------------------- logits

// Two values rounded to O, packed, and as FP32.
template <typename O> __device__ __forceinline__ uint32_t round2(f32x2 v, f32x2 &kept);
template <> __device__ __forceinline__ uint32_t round2<__nv_bfloat16>(f32x2 v, f32x2 &kept) {
  float a, b;
  unpack2(v, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const uint32_t u = *reinterpret_cast<const uint32_t *>(&h);
  kept = pack2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return u;
}
template <> __device__ __forceinline__ uint32_t round2<__half>(f32x2 v, f32x2 &kept) {
  float a, b;
  unpack2(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  kept = pack2(__low2float(h), __high2float(h));
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Tiles of 256 queries x 256 rows. GRAD: G of a piece; else the partial sums.
template <PairKind KIND_, int PLANES_, bool GRAD, typename O>
struct LogitsOp : PairNoHelpers {
  static constexpr PairKind KIND = KIND_;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr int PLANES = PLANES_, SCRATCH = GRAD ? kPairEpi * kBoxBytes : 0, MAX_STAGES = 8;
  static constexpr int CHUNK = PLANES == 2 ? 2 : 6;   // 24 steps of the tensor cores
  struct Args {
    CUtensorMap a[PLANES], b[PLANES];
    uint32_t bn;
    uint32_t mt, nt, kblocks;
    uint32_t nq, q0;         // queries; the first one of this launch
    uint64_t nrows, first;   // rows; the first one of this piece
    double scale2;           // scale * log2(e)
    const float *xscale;     // PLANES 2: per query
    const uint32_t *maxima;
    const int64_t *targets;
    float2 *part;            // forward: [query - q0][2 nt]
    float *tlogit;           // [query]
    const float *lse, *grad;
    CUtensorMap g[PLANES];   // gradient: G of the piece
    float *gsum;             // [query][2 nt]: the stored G summed over a half tile
  };
  static __device__ __forceinline__ uint32_t items(const Args &p) { return p.mt * p.nt; }
  static __device__ __forceinline__ PairItem item(const Args &p, uint32_t i) {
    const uint32_t n = i / p.mt, m = i % p.mt;   // a row tile against all queries before the next
    return {(int32_t)(p.q0 + m * 256), (int32_t)(p.first + (uint64_t)n * 256), 0, p.kblocks, n};
  }
  // What an item's epilogue reads of its query, loaded an item ahead.
  struct Row {
    int64_t target;
    float lse, grad, xscale;
  };
  static __device__ __forceinline__ uint32_t query_of(const PairItem &w, uint32_t rank) {
    return (uint32_t)w.a_row + rank * 128 + ((threadIdx.x >> 5) & 3) * 32 + (threadIdx.x & 31);
  }
  static __device__ __forceinline__ Row row_of(const Args &p, uint32_t i, uint32_t rank) {
    Row r = {-1, 0.0f, 0.0f, 1.0f};
    if (i >= items(p)) return r;
    const uint32_t q = query_of(item(p, i), rank);
    if (q >= p.nq) return r;
    r.target = p.targets[q];
    if (PLANES == 2) r.xscale = p.xscale[q];
    if (GRAD) {
      r.lse = p.lse[q];
      r.grad = p.grad ? p.grad[q] : 1.0f;
    }
    return r;
  }
  static __device__ __forceinline__ void epilogue(const Args &p, PairSums &sums, uint8_t *scratch, uint32_t rank,
                                                  uint32_t cluster, uint32_t clusters) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const double scale2 = PLANES == 2 ? p.scale2 * (double)undo_scale(p.maxima[MAX_ROWS]) : p.scale2;
    const float unit = GRAD ? grad_unit(p.maxima[MAX_GRAD]) : 1.0f;
    BoxStore box{scratch + warp * kBoxBytes};
    Row next = row_of(p, cluster, rank);
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      const PairItem w = item(p, i);
      const Row row = next;
      next = row_of(p, i + clusters, rank);
      const uint32_t q = query_of(w, rank);
      const bool valid = q < p.nq;
      const int64_t col0 = (int64_t)w.b_row + half * 128;   // this thread's first row of W
      f32x2 v[64];
      sums.template total<CHUNK, 4>(half * 128, w.kblocks, v);
      if (!__any_sync(0xffffffffu, valid)) continue;
      float k = PLANES == 2 ? (float)(scale2 * (double)row.xscale) : (float)scale2;
      if (k == 0.0f) k = FLT_MIN;   // (0 would make NaNs of the infinities that stand for no column)
      const int64_t left = (int64_t)p.nrows - col0;         // columns that are rows of W
      // the target's column, 128 where it is not here
      const int64_t rel = row.target - col0;
      const int at = valid && rel >= 0 && rel < 128 ? (int)rel : 128;
      const bool hit = __any_sync(0xffffffffu, at < 128);
      float s = 0.0f;                                       // of this thread's 128 columns
      if (!GRAD) {
        if (hit) {
          float t = 0.0f;
#pragma unroll
          for (int j = 0; j < 64; j++) {
            float a, b;
            unpack2(v[j], a, b);
            t = at == 2 * j ? a : (at == 2 * j + 1 ? b : t);
          }
          if (at < 128) p.tlogit[q] = t * k;
        }
        if (left < 128) {   // columns past the rows count for nothing
          const float none = k < 0.0f ? INFINITY : -INFINITY;
#pragma unroll
          for (int j = 0; j < 64; j++) {
            float a, b;
            unpack2(v[j], a, b);
            v[j] = pack2(2 * j < (int)left ? a : none, 2 * j + 1 < (int)left ? b : none);
          }
        }
        // the largest logit in base 2
        float top[4];
        const float start = k < 0.0f ? INFINITY : -INFINITY;
        top[0] = top[1] = top[2] = top[3] = start;
        if (k < 0.0f) {
#pragma unroll
          for (int j = 0; j < 64; j++) {
            float a, b;
            unpack2(v[j], a, b);
            top[j & 3] = min3(top[j & 3], a, b);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 64; j++) {
            float a, b;
            unpack2(v[j], a, b);
            top[j & 3] = max3(top[j & 3], a, b);
          }
        }
        const float most = k < 0.0f ? fminf(fminf(top[0], top[1]), fminf(top[2], top[3]))
                                    : fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const float m = left <= 0 ? -INFINITY : most * k;
        const float base = m == -INFINITY ? 0.0f : m;
        const f32x2 kk = pack2(k, k), bb = pack2(-base, -base);
        f32x2 e[4] = {};
#pragma unroll
        for (int j = 0; j < 64; j++) {
          float a, b;
          unpack2(fma2(v[j], kk, bb), a, b);
          e[j & 3] = add2(e[j & 3], pack2(exp2_approx(a), exp2_approx(b)));
        }
        float a, b;
        unpack2(add2(add2(e[0], e[1]), add2(e[2], e[3])), a, b);
        s = a + b;
        if (left <= 0) s = 0.0f;
        if (valid) p.part[(uint64_t)(q - p.q0) * (2 * p.nt) + 2 * w.index + half] = make_float2(m, s);
      } else {
        // G; columns past the rows go to the buffer's end, which is not read
        const bool kept = valid && has_target(row.target, p.nrows);
        const float lse2 = row.lse * kLog2e, g = kept ? row.grad / unit * kGradScale : 0.0f;
        const f32x2 kk = pack2(k, k), zz = pack2(-lse2, -lse2), gg = pack2(g, g);
#pragma unroll
        for (int j = 0; j < 64; j++) {
          float a, b;
          unpack2(fma2(v[j], kk, zz), a, b);
          v[j] = pack2(exp2_approx(a), exp2_approx(b));
        }
        if (hit) {
#pragma unroll
          for (int j = 0; j < 64; j++)
            v[j] = add2(v[j], pack2(at == 2 * j ? -1.0f : 0.0f, at == 2 * j + 1 ? -1.0f : 0.0f));
        }
#pragma unroll
        for (int j = 0; j < 64; j++) v[j] = mul2(v[j], gg);
        if (!kept) {        // (not 0 times what the query holds)
#pragma unroll
          for (int j = 0; j < 64; j++) v[j] = 0;
        }
        if (left < 128) {
#pragma unroll
          for (int j = 0; j < 64; j++) {
            float a, b;
            unpack2(v[j], a, b);
            v[j] = pack2(2 * j < (int)left ? a : 0.0f, 2 * j + 1 < (int)left ? b : 0.0f);
          }
        }
        const int32_t x = (int32_t)(col0 - (int64_t)p.first), y = (int32_t)(q - lane);
        f32x2 sum[2] = {};
        // of a plane: the values it keeps, taken off v, and their sum
#pragma unroll
        for (int plane = 0; plane < PLANES; plane++) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            box.reuse();
#pragma unroll
            for (int c = 0; c < 8; c++) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; j++) {
                f32x2 &f = v[32 * h + 4 * c + j];
                f32x2 kept_values;
                o[j] = round2<O>(f, kept_values);
                sum[j & 1] = add2(sum[j & 1], kept_values);
                if (plane + 1 < PLANES) f = fma2(kept_values, pack2(-1.0f, -1.0f), f);
              }
              box.put(c, make_uint4(o[0], o[1], o[2], o[3]));
            }
            box.store(&p.g[plane], x + h * 64, y);
          }
        }
        float a, b;
        unpack2(add2(sum[0], sum[1]), a, b);
        s = a + b;
        if (valid) p.gsum[(uint64_t)q * (2 * p.nt) + 2 * w.index + half] = s;
      }
    }
  }
};

// Join a query's partial sums: lse = (m + log2 s) ln 2, loss = lse - target logit.
__global__ void __launch_bounds__(128) join_parts(const float2 *part, uint32_t n, uint32_t q0, uint64_t nrows,
                                                  const int64_t *targets, const float *tlogit, float *loss, float *lse,
                                                  int32_t *status) {
  const uint32_t q = q0 + blockIdx.x;
  part += (uint64_t)blockIdx.x * n;
  __shared__ float top[4];
  __shared__ double sum[4];
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < n; i += 128) m = fmaxf(m, part[i].x);
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const float base = m == -INFINITY ? 0.0f : m;
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += 128) {
    const float2 v = part[i];
    s += v.y * exp2f(v.x - base);
  }
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (threadIdx.x % 32 == 0) sum[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    const double l = log2(s);
    const int64_t t = targets[q];
    const bool bad = t >= (int64_t)nrows;
    if (lse) lse[q] = (float)(((double)m + l) * kLn2);
    if (loss) loss[q] = t < 0 ? 0.0f : (bad ? NAN : (float)(((double)m - (double)tlogit[q] + l) * kLn2));
    if (status) status[q] = bad ? OP_INVALID : OP_OK;
  }
}

// ---------------------------------------------------------------- gradients

// dX partial sums: 256 queries x bn dimensions, K = a share of the piece's rows.
template <PairKind KIND_, int PLANES_>
struct QueriesOp : PairNoHelpers {
  static constexpr PairKind KIND = KIND_;
  static constexpr bool A_MN = false, B_MN = true;
  static constexpr int PLANES = PLANES_, SCRATCH = kPairEpi * kBoxBytes, MAX_STAGES = 8;
  static constexpr int CHUNK = PLANES == 2 ? 2 : 0;
  struct Args {
    CUtensorMap a[PLANES], b[PLANES];   // G (piece columns); W's rows from the piece's first on
    uint32_t bn;
    uint32_t mt, nt, splits;
    uint32_t kblocks;        // of the piece
    uint32_t nq, dims;
    int add;                 // to what earlier pieces left
    CUtensorMap part;        // [splits][nq][dims]
  };
  static __device__ __forceinline__ uint32_t items(const Args &p) { return p.mt * p.nt * p.splits; }
  static __device__ __forceinline__ PairItem item(const Args &p, uint32_t i) {
    const uint32_t tiles = p.mt * p.nt, s = i / tiles, t = i % tiles;
    const uint32_t k0 = (uint32_t)((uint64_t)p.kblocks * s / p.splits);
    const uint32_t k1 = (uint32_t)((uint64_t)p.kblocks * (s + 1) / p.splits);
    return {(int32_t)((t / p.nt) * 256), (int32_t)((t % p.nt) * p.bn), (int32_t)(k0 * 64), k1 - k0, s};
  }
  static __device__ __forceinline__ void epilogue(const Args &p, PairSums &sums, uint8_t *scratch, uint32_t rank,
                                                  uint32_t cluster, uint32_t clusters) {
    for (uint32_t i = cluster; i < items(p); i += clusters) tile(p, item(p, i), sums, scratch, rank);
  }
  static __device__ __forceinline__ void tile(const Args &p, const PairItem &w, PairSums &sums, uint8_t *scratch,
                                              uint32_t rank) {
    if (w.kblocks == 0) return;   // (a short last piece; its partial stays)
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const uint32_t q = (uint32_t)w.a_row + rank * 128 + (warp & 3) * 32 + lane;
    const uint32_t cols = p.bn / 2;
    f32x2 v[64];
    uint32_t tmem = 0;
    if (CHUNK) sums.template total<CHUNK + !CHUNK, 4>(half * cols, w.kblocks, v);
    else tmem = sums.acquire() + half * cols;
    BoxStore box{scratch + warp * kBoxBytes};
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
      const uint32_t d0 = (uint32_t)w.b_row + half * cols + c * 32;
      if (c * 32 >= cols || d0 >= p.dims || q - lane >= p.nq) break;
      uint32_t r[32];
      if (CHUNK) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          float a, b;
          unpack2(v[16 * c + j], a, b);
          r[2 * j] = __float_as_uint(a);
          r[2 * j + 1] = __float_as_uint(b);
        }
      } else {
        sums.load(tmem + c * 32, r);
      }
      box.reuse();
#pragma unroll
      for (int j = 0; j < 8; j++) box.put(j, make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]));
      box.store_sums(&p.part, (int32_t)d0, (int32_t)(q - lane), (int32_t)w.index, p.add != 0);
    }
    if (!CHUNK) sums.release();
  }
};

// dW: 256 of the piece's rows x bn dimensions, K = the queries.
template <PairKind KIND_, int PLANES_, typename T>
struct RowsOp : PairNoHelpers {
  static constexpr PairKind KIND = KIND_;
  static constexpr bool A_MN = true, B_MN = true;
  static constexpr int PLANES = PLANES_, SCRATCH = kPairEpi * kBoxBytes, MAX_STAGES = 8;
  static constexpr int CHUNK = PLANES == 2 ? 2 : 0;
  struct Args {
    CUtensorMap a[PLANES], b[PLANES];   // G (piece columns); X
    uint32_t bn;
    uint32_t mt, nt, kblocks;
    uint32_t rows, dims;     // rows of the piece
    double scale;
    const uint32_t *maxima;
    T *out;                  // the piece's first row
    int boxes;               // out's rows are 16-byte aligned: `map` stores them
    CUtensorMap map;
  };
  static __device__ __forceinline__ uint32_t items(const Args &p) { return p.mt * p.nt; }
  static __device__ __forceinline__ PairItem item(const Args &p, uint32_t i) {
    return {(int32_t)((i / p.nt) * 256), (int32_t)((i % p.nt) * p.bn), 0, p.kblocks, 0};
  }
  static __device__ __forceinline__ void epilogue(const Args &p, PairSums &sums, uint8_t *scratch, uint32_t rank,
                                                  uint32_t cluster, uint32_t clusters) {
    for (uint32_t i = cluster; i < items(p); i += clusters) tile(p, item(p, i), sums, scratch, rank);
  }
  static __device__ __forceinline__ void tile(const Args &p, const PairItem &w, PairSums &sums, uint8_t *scratch,
                                              uint32_t rank) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const uint32_t i = (uint32_t)w.a_row + rank * 128 + (warp & 3) * 32 + lane;
    double f = p.scale * (double)grad_unit(p.maxima[MAX_GRAD]) / kGradScale;
    if (PLANES == 2) f *= (double)undo_scale(p.maxima[MAX_QUERIES]);
    const float factor = (float)f;
    const uint32_t cols = p.bn / 2;
    f32x2 v[64];
    uint32_t tmem = 0;
    if (CHUNK) sums.template total<CHUNK + !CHUNK, 4>(half * cols, w.kblocks, v);
    else tmem = sums.acquire() + half * cols;
    T *row = p.out + (uint64_t)i * p.dims;
    BoxStore box{scratch + warp * kBoxBytes};
    constexpr uint32_t BOX = 128 / sizeof(T), V = 16 / sizeof(T);   // values of a box row, of a chunk
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
      const uint32_t d0 = (uint32_t)w.b_row + half * cols + c * 32;
      if (c * 32 >= cols || d0 >= p.dims || i - lane >= p.rows) break;
      uint32_t r[32];
      if (CHUNK) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          float a, b;
          unpack2(v[16 * c + j], a, b);
          r[2 * j] = __float_as_uint(a);
          r[2 * j + 1] = __float_as_uint(b);
        }
      } else {
        sums.load(tmem + c * 32, r);
      }
      const uint32_t at = c * 32 % BOX;     // of the box's values
      if (p.boxes && at == 0) box.reuse();
#pragma unroll
      for (uint32_t j = 0; j < 32; j += V) {
        alignas(16) T o[V];
#pragma unroll
        for (uint32_t u = 0; u < V; u++) o[u] = from_float<T>(__uint_as_float(r[j + u]) * factor);
        if (p.boxes) {
          box.put((at + j) / V, *reinterpret_cast<uint4 *>(o));
        } else if (i < p.rows) {
#pragma unroll
          for (uint32_t u = 0; u < V; u++)
            if (d0 + j + u < p.dims) row[d0 + j + u] = o[u];
        }
      }
      // the last 32 values of a box, or of the row
      if (p.boxes && (at + 32 == BOX || d0 + 32 >= p.dims))
        box.store(&p.map, (int32_t)((d0 - at) * (sizeof(T) / 2)), (int32_t)(i - lane));   // (in 16-bit values)
    }
    if (!CHUNK) sums.release();
  }
};

// A piece's sums of G into each query's (a warp a query).
__global__ void __launch_bounds__(256) fold_sums(const float *gsum, uint32_t n, uint32_t nq, int add, double *total) {
  const uint32_t q = (blockIdx.x * 256 + threadIdx.x) / 32, lane = threadIdx.x % 32;
  if (q >= nq) return;
  double s = 0.0;
  for (uint32_t i = lane; i < n; i += 32) s += gsum[(uint64_t)q * n + i];
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (lane == 0) total[q] = s + (add ? total[q] : 0.0);
}

// dX_i = scale * (the partial sums, in order, - (sum_j G_ij) w_target); zero for
// a query without a target. G's exact rows sum to 0, the rounded ones do not,
// and rows near each other (a cluster's) make sum_j G_ij w_j the small
// difference of large terms: what is left of the sum would weigh in with a
// whole row (10 times G's rounding where a cluster's rows differ by a tenth of
// their length). With it taken off at the target, the sum is over
// G_ij (w_j - w_target), and errors are relative to the differences.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) join_queries(const float *part, uint32_t splits, uint32_t nq, uint32_t dims,
                                                    double scale, const uint32_t *maxima, const double *total,
                                                    const T *rows, uint64_t stride, const int64_t *targets,
                                                    uint64_t nrows, T *out) {
  const uint32_t q = blockIdx.x, ld = (dims + 3) / 4 * 4;
  const uint64_t plane = (uint64_t)nq * ld;
  const double f = scale * (double)grad_unit(maxima[MAX_GRAD]) / kGradScale;
  const float factor = (float)f;
  const float undo = PLANES == 2 ? undo_scale(maxima[MAX_ROWS]) : 1.0f;
  const int64_t t = targets[q];
  const bool kept = has_target(t, nrows);
  const float left = kept ? -(float)total[q] : 0.0f;
  const T *row = rows + (kept ? (uint64_t)t * stride : 0);
  for (uint32_t d = threadIdx.x; d < dims; d += blockDim.x) {
    float v = 0.0f;
    if (kept) {
      const float *at = part + (uint64_t)q * ld + d;
      for (uint32_t k = 0; k < splits; k++) v += at[k * plane];
      v = fmaf(left, to_float(row[d]), v * undo) * factor;
    }
    out[(uint64_t)q * dims + d] = from_float<T>(v);
  }
}

// ---------------------------------------------------------------- the calls

uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

struct Carve {
  uint64_t off = 0;
  uint64_t take(uint64_t bytes) {
    const uint64_t o = off;
    off += up(bytes, 256);
    return o;
  }
};

// Whether TMA can read the rows where they are.
bool in_place(const void *p, uint64_t stride, uint32_t dtype) {
  return dtype != ANNB200_F32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0;
}

struct Plan {
  int planes;
  uint32_t ld;             // values a packed row
  bool pack_x, pack_w;
  uint64_t x, w, xscale, maxima, part, tlogit, g, gsum, gtotal, dq, total;
  uint32_t nt, chunk;      // forward: row tiles; queries a launch
  uint64_t piece;          // gradient: rows a piece
  uint32_t bn, dt, splits; // dimensions a tile, tiles, shares of a piece in dX
};

Plan plan_of(const AnnB200LossJob &j, bool grad) {
  Plan p = {};
  Carve c;
  const uint64_t nq = std::max(1u, j.nq);
  p.planes = j.dtype == ANNB200_F32 ? 2 : 1;
  p.ld = (uint32_t)up(j.dims, 8);
  p.pack_x = grad || !in_place(j.queries, j.query_stride, j.dtype);
  p.pack_w = !in_place(j.rows, j.row_stride, j.dtype);
  p.maxima = c.take(16);
  p.xscale = c.take(nq * 4);
  if (p.pack_x) p.x = c.take(nq * p.ld * 2 * p.planes);
  if (p.pack_w) p.w = c.take(j.nrows * p.ld * 2 * p.planes);
  p.nt = (uint32_t)((j.nrows + 255) / 256);
  if (!grad) {
    p.chunk = (uint32_t)std::min<uint64_t>(up(nq, 256), std::max<uint64_t>(256, kPartBytes / (16ull * p.nt) / 256 * 256));
    p.part = c.take(std::min<uint64_t>(nq, p.chunk) * p.nt * 16);
    p.tlogit = c.take(nq * 4);
  } else {
    // a piece: G of kPieceBytes (it stays in L2 for the products that read
    // it), but 8,192 rows at least, since each piece reads and writes dX's sums
    p.piece = std::max<uint64_t>(8192, kPieceBytes / (2 * p.planes * nq) / 256 * 256);
    p.piece = std::min<uint64_t>({p.piece, up(j.nrows, 256), 1u << 20});
    p.g = c.take(nq * p.piece * 2 * p.planes);
    p.gsum = c.take(nq * (p.piece / 128) * 4);
    p.gtotal = c.take(nq * 8);
    // 128 dimensions a tile where 256 would leave over an eighth of them empty
    const uint64_t full = up(j.dims, 256), fine = up(j.dims, 128);
    p.bn = fine * 8 < full * 7 ? 128 : 256;
    p.dt = (uint32_t)((j.dims + p.bn - 1) / p.bn);
    // shares of a piece's rows in dX: the fewest that keep nine of ten clusters busy
    const uint64_t tiles = (nq + 255) / 256 * p.dt, blocks = (std::min(p.piece, j.nrows) + 63) / 64;
    double best = 0.0;
    p.splits = 1;
    for (uint32_t s = 1; s <= kPlanClusters && s <= blocks; s++) {
      const double use = (double)(tiles * s) / (double)up(tiles * s, kPlanClusters);
      if (use > best + 1e-9) {
        best = use;
        p.splits = s;
      }
      if (best >= 0.9) break;
    }
    p.dq = c.take((uint64_t)p.splits * nq * up(j.dims, 4) * 4);
  }
  p.total = c.off;
  return p;
}

template <typename T, typename O, int PLANES>
void pack(const T *x, uint64_t stride, uint64_t rows, uint32_t dims, uint32_t ld, const int64_t *targets,
          uint64_t nrows, const float *scales, const uint32_t *whole, O *out, cudaStream_t st) {
  uint32_t tx = 1;
  while (tx < 256 && tx * 8 < ld) tx *= 2;
  const uint64_t blocks = (rows + 256 / tx - 1) / (256 / tx);
  pack_rows<T, O, PLANES><<<(unsigned)std::min<uint64_t>(blocks, 1u << 16), 256, 0, st>>>(
      x, stride, rows, dims, ld, tx, targets, nrows, scales, whole, out, rows * ld);
}

void max_of(const float *x, uint64_t stride, uint64_t rows, uint32_t dims, const int64_t *targets, uint64_t nrows,
            uint32_t *out, cudaStream_t st) {
  uint32_t tx = 1;
  while (tx < 256 && tx * 4 < dims) tx *= 2;
  const uint64_t blocks = (rows + 256 / tx - 1) / (256 / tx);
  array_max<<<(unsigned)std::min<uint64_t>(blocks, 1184), 256, 0, st>>>(x, stride, rows, dims, tx, targets, nrows, out);
}

// T: the operands' type; O: the products'.
template <typename T, typename O, PairKind KIND, int PLANES>
int run_loss(const AnnB200LossJob &j, bool grad, cudaStream_t st) {
  const Plan p = plan_of(j, grad);
  const int sms = op_sms();
  if (sms < 2) return report_error(OP_BACKEND_ERROR, "no current CUDA device");
  uint8_t *ws = static_cast<uint8_t *>(j.workspace);
  uint32_t *maxima = reinterpret_cast<uint32_t *>(ws + p.maxima);
  float *xscale = reinterpret_cast<float *>(ws + p.xscale);
  const T *x = static_cast<const T *>(j.queries), *w = static_cast<const T *>(j.rows);
  const int64_t *kept = grad ? j.targets : nullptr;   // the gradient leaves out queries without a target
  unsigned long long launches = 0;
  cudaError_t e = cudaSuccess;

  // operands as the tensor maps read them
  if (PLANES == 2 || grad) {
    e = cudaMemsetAsync(maxima, 0, 16, st);
    if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss: %s", cudaGetErrorString(e));
  }
  if (grad) {
    grad_max<<<(j.nq + 255) / 256, 256, 0, st>>>(j.grad, j.targets, j.nq, j.nrows, maxima + MAX_GRAD);
    launches++;
  }
  if (PLANES == 2) {
    const float *xf = reinterpret_cast<const float *>(x);
    max_of(reinterpret_cast<const float *>(w), j.row_stride, j.nrows, j.dims, nullptr, 0, maxima + MAX_ROWS, st);
    if (grad) max_of(xf, j.query_stride, j.nq, j.dims, kept, j.nrows, maxima + MAX_QUERIES, st);
    query_scales<<<(j.nq + 7) / 8, 256, 0, st>>>(xf, j.query_stride, j.nq, j.dims, grad ? maxima + MAX_QUERIES : nullptr,
                                                 xscale);
    launches += grad ? 3 : 2;
  }
  const O *xo = reinterpret_cast<const O *>(x), *wo = reinterpret_cast<const O *>(w);
  uint64_t xld = j.query_stride, wld = j.row_stride;
  if (p.pack_x) {
    O *to = reinterpret_cast<O *>(ws + p.x);
    pack<T, O, PLANES>(x, j.query_stride, j.nq, j.dims, p.ld, kept, j.nrows, xscale, nullptr, to, st);
    xo = to;
    xld = p.ld;
    launches++;
  }
  if (p.pack_w) {
    O *to = reinterpret_cast<O *>(ws + p.w);
    pack<T, O, PLANES>(w, j.row_stride, j.nrows, j.dims, p.ld, nullptr, 0, nullptr, maxima + MAX_ROWS, to, st);
    wo = to;
    wld = p.ld;
    launches++;
  }
  bool maps = true;
  auto map = [&](CUtensorMap *m, const O *base, uint64_t inner, uint64_t outer, uint64_t ld, uint64_t plane,
                 uint32_t box) {
    for (int i = 0; i < PLANES; i++)
      maps = maps && encode_operand_map(m + i, 2, base + i * plane, inner, outer, ld * 2, box);
  };

  const uint32_t kblocks = (j.dims + 63) / 64;
  auto logits = [&](auto &l) {
    map(l.a, xo, j.dims, j.nq, xld, (uint64_t)j.nq * p.ld, 128);
    map(l.b, wo, j.dims, j.nrows, wld, j.nrows * p.ld, 128);
    l.bn = 256;
    l.kblocks = kblocks;
    l.nq = j.nq;
    l.nrows = j.nrows;
    l.scale2 = (double)j.scale * 1.4426950408889634;
    l.xscale = xscale;
    l.maxima = maxima;
    l.targets = j.targets;
  };
  if (!grad) {
    using Op = LogitsOp<KIND, PLANES, false, O>;
    typename Op::Args l = {};
    logits(l);
    l.nt = p.nt;
    l.part = reinterpret_cast<float2 *>(ws + p.part);
    l.tlogit = reinterpret_cast<float *>(ws + p.tlogit);
    if (!maps) return report_error(OP_BACKEND_ERROR, "softmax loss: tensor map");
    for (uint32_t q0 = 0; q0 < j.nq; q0 += p.chunk) {
      const uint32_t n = std::min(p.chunk, j.nq - q0);
      l.q0 = q0;
      l.mt = (n + 255) / 256;
      // (a launch covers whole tiles of queries, except at their end)
      e = launch_pair<Op>(l, l.mt * l.nt, sms, st);
      if (e != cudaSuccess) break;
      join_parts<<<n, 128, 0, st>>>(l.part, 2 * p.nt, q0, j.nrows, j.targets, l.tlogit, j.loss, j.lse, j.status);
      launches += 2;
    }
    if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss: %s", cudaGetErrorString(e));
    return op_launched("softmax loss", launches);
  }

  O *g = reinterpret_cast<O *>(ws + p.g);
  float *dq = reinterpret_cast<float *>(ws + p.dq);
  const uint64_t gplane = (uint64_t)j.nq * p.piece;
  using LOp = LogitsOp<KIND, PLANES, true, O>;
  using QOp = QueriesOp<KIND, PLANES>;
  using ROp = RowsOp<KIND, PLANES, T>;
  typename LOp::Args l = {};
  logits(l);
  l.mt = (j.nq + 255) / 256;
  l.lse = j.lse;
  l.grad = j.grad;
  map(l.g, g, p.piece, j.nq, p.piece, gplane, 32);
  l.gsum = reinterpret_cast<float *>(ws + p.gsum);
  double *gtotal = reinterpret_cast<double *>(ws + p.gtotal);
  for (uint64_t first = 0; first < j.nrows && e == cudaSuccess; first += p.piece) {
    const uint64_t n = std::min(p.piece, j.nrows - first);
    l.first = first;
    l.nt = (uint32_t)((n + 255) / 256);
    e = maps ? launch_pair<LOp>(l, l.mt * l.nt, sms, st) : cudaErrorInvalidValue;
    launches++;
    if (j.dqueries && e == cudaSuccess) {
      typename QOp::Args a = {};
      map(a.a, g, n, j.nq, p.piece, gplane, 128);
      map(a.b, wo + first * wld, j.dims, n, wld, j.nrows * p.ld, 64);
      a.bn = p.bn;
      a.mt = l.mt;
      a.nt = p.dt;
      a.splits = p.splits;
      a.kblocks = (uint32_t)((n + 63) / 64);
      a.nq = j.nq;
      a.dims = j.dims;
      a.add = first != 0;
      maps = maps && encode_sums_map(&a.part, dq, j.dims, j.nq, p.splits, up(j.dims, 4) * 4);
      fold_sums<<<(j.nq + 7) / 8, 256, 0, st>>>(l.gsum, 2 * l.nt, j.nq, a.add, gtotal);
      e = maps ? launch_pair<QOp>(a, a.mt * a.nt * a.splits, sms, st) : cudaErrorInvalidValue;
      launches += 2;
    }
    if (j.drows && e == cudaSuccess) {
      typename ROp::Args a = {};
      map(a.a, g, n, j.nq, p.piece, gplane, 64);
      map(a.b, xo, j.dims, j.nq, xld, (uint64_t)j.nq * p.ld, 64);
      a.bn = p.bn;
      a.mt = (uint32_t)((n + 255) / 256);
      a.nt = p.dt;
      a.kblocks = (j.nq + 63) / 64;
      a.rows = (uint32_t)n;
      a.dims = j.dims;
      a.scale = (double)j.scale;
      a.maxima = maxima;
      a.out = static_cast<T *>(j.drows) + first * j.dims;
      a.boxes = (uint64_t)j.dims * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
      // (as 16-bit values, whatever T: a box is 128 bytes wide)
      if (a.boxes)
        maps = maps && encode_operand_map(&a.map, 2, a.out, j.dims * sizeof(T) / 2, n, j.dims * sizeof(T), 32);
      e = maps ? launch_pair<ROp>(a, a.mt * a.nt, sms, st) : cudaErrorInvalidValue;
      launches++;
    }
  }
  if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss gradient: %s", cudaGetErrorString(e));
  if (j.dqueries) {
    join_queries<T, PLANES><<<j.nq, j.dims <= 128 ? 128 : 256, 0, st>>>(
        dq, p.splits, j.nq, j.dims, (double)j.scale, maxima, gtotal, w, j.row_stride, j.targets, j.nrows,
        static_cast<T *>(j.dqueries));
    launches++;
  }
  return op_launched("softmax loss gradient", launches);
}

int check_job(const AnnB200LossJob *j) {
  if (!j) return report_error(OP_INVALID, "NULL job");
  if (!op_dtype(j->dtype)) return report_error(OP_INVALID, "type %u", j->dtype);
  if (j->dims == 0 || j->dims > 65536) return report_error(OP_INVALID, "%u dimensions", j->dims);
  if (j->nq > (1u << 22)) return report_error(OP_INVALID, "more than 2^22 queries");
  if (j->nrows == 0 || j->nrows > 0x7fffffffull) return report_error(OP_INVALID, "no rows, or 2^31 and more");
  if (j->query_stride < j->dims || j->row_stride < j->dims) return report_error(OP_INVALID, "rows overlap");
  if (!std::isfinite(j->scale)) return report_error(OP_INVALID, "scale is not finite");
  return OP_OK;
}

int run_job(const AnnB200LossJob *j, bool grad, void *stream) {
  int r = check_job(j);
  if (r != OP_OK || j->nq == 0) return r;
  if (!j->queries || !j->rows || !j->targets) return report_error(OP_INVALID, "NULL pointer");
  if (grad && !j->lse) return report_error(OP_INVALID, "the gradient needs lse");
  if (grad && !j->dqueries && !j->drows) return OP_OK;
  if (!j->workspace || (reinterpret_cast<uintptr_t>(j->workspace) & 255) ||
      j->workspace_bytes < plan_of(*j, grad).total)
    return report_error(OP_INVALID, "workspace too small or not 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (j->dtype) {
    case ANNB200_F32: return run_loss<float, __half, PAIR_F16, 2>(*j, grad, st);
    case ANNB200_F16: return run_loss<__half, __half, PAIR_F16, 1>(*j, grad, st);
    default: return run_loss<__nv_bfloat16, __nv_bfloat16, PAIR_BF16, 1>(*j, grad, st);
  }
}

}  // namespace
}  // namespace annb200

using namespace annb200;

extern "C" int AnnB200SoftmaxLossWorkspace(const AnnB200LossJob *job, uint64_t *loss_bytes, uint64_t *grad_bytes) {
  int r = check_job(job);
  if (r != OP_OK) return r;
  if (loss_bytes) *loss_bytes = plan_of(*job, false).total;
  if (grad_bytes) *grad_bytes = plan_of(*job, true).total;
  return OP_OK;
}
extern "C" int AnnB200SoftmaxLoss(const AnnB200LossJob *job, void *stream) { return run_job(job, false, stream); }
extern "C" int AnnB200SoftmaxLossGrad(const AnnB200LossJob *job, void *stream) { return run_job(job, true, stream); }
