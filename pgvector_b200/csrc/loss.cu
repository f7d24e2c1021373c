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
//
// What bounds it: the four products, 8 nq n d operations with the logits' second
// time. 4,096 x 65,536 x 768 bf16, 412 GFLOP each: logits 312 us, G 378 us, dX
// 280 us, dW 292 us. dX and dW run near the product loop's rate. A tile of the
// logits takes 9,100 clocks and one of G 11,400, where its products and loads
// alone would take 8,300: the epilogue (128 exponentials a thread, for G 128
// roundings and 64 KB out too) does not run wholly under the next tile's
// products. Below about 256 dimensions it bounds the call.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "pair_gemm.cuh"

namespace annb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.925963033e-8f;   // log2(e), and what FP32 leaves of it
constexpr double kLn2 = 0.69314718055994530942;
constexpr uint64_t kPartBytes = 256ull << 20;   // the forward call's partial maxima and sums, or those of 256 queries
constexpr uint64_t kPieceBytes = 512ull << 20;  // G of a piece (128 MB: 4,096 x 65,536 x 768 took 1,538 us for 1,450)
constexpr uint64_t kMostPieceBytes = 4ull << 30;
constexpr uint32_t kPlanClusters = 74;          // clusters the plan splits for (148 SMs)

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
// G in FP16 terms: FP16 holds 2^-24 to 2^16, so a query's row of G is kept as
// grad / unit * 2^14 * (p - onehot), below 2^15, where unit is its own |grad|'s
// power of two: what p falls to is then held to within 2^-39 of 1 whatever the
// other queries' weights are (with one unit for all, a weight of 2e-7 of the
// largest lost most of dX over 100,003 rows). dX's factor is
// a query's, so it undoes the unit; dW sums over queries, and is made with rows
// x_i * unit_i / (the largest unit), laid out a second time, where 2^-39 of the
// largest weight's share is all that is lost. BF16 has FP32's range: no unit.
constexpr float kGradScale = 16384.0f;
template <typename O> constexpr bool kGradUnits = std::is_same<O, __half>::value;
__device__ __forceinline__ float grad_unit(uint32_t bits) {   // of |grad|'s bits
  return __uint_as_float(max(bits & 0x7f800000u, 0x00800000u));
}

__device__ __forceinline__ bool has_target(int64_t t, uint64_t nrows) { return t >= 0 && t < (int64_t)nrows; }

// ---------------------------------------------------------------- laying operands out

// Maxima are found in two steps without atomics or a cleared word: a grid leaves
// one a block, and whoever needs the whole array's joins them.
constexpr int kRowParts = 592, kQueryParts = 64, kGradParts = 32;
struct Maxima {
  uint32_t rows[kRowParts], queries[kQueryParts], grad[kGradParts];
  uint32_t all_rows, all_queries;   // joined by the layout kernel
};
// The largest of a 256-thread block's values, for each of its threads.
__device__ __forceinline__ uint32_t block_max(uint32_t best) {
  __shared__ uint32_t top[8];
  best = __reduce_max_sync(0xffffffffu, best);
  __syncthreads();
  if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = best;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) best = max(best, top[i]);
  return best;
}
// The largest of a grid's parts, for each thread of a 256-thread block.
__device__ __forceinline__ uint32_t join_parts(const uint32_t *parts, int n) {
  uint32_t best = 0;
  for (int i = threadIdx.x; i < n; i += 256) best = max(best, parts[i]);
  return block_max(best);
}
// The largest query's unit (a warp's lanes together).
__device__ __forceinline__ float grad_unit(const Maxima *m) {
  static_assert(kGradParts == 32, "a part a lane");
  return grad_unit(__reduce_max_sync(0xffffffffu, m->grad[threadIdx.x & 31]));
}
// A value's bits, 0 where it is not finite.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// The largest finite |x| of the rows (FP32), of the queries with a target, and
// of those queries' weights: kRowParts, kQueryParts and kGradParts blocks, where
// they are asked for. `tx` threads a row, 16 bytes each.
template <typename T> struct FindMaxima {
  const T *w, *x;
  uint64_t w_stride, x_stride, nrows;
  uint32_t nq, dims, tx;
  uint32_t row_blocks, query_blocks, grad_blocks;
  const int64_t *targets;
  const float *grad;
  Maxima *out;
};
template <typename T>
__global__ void __launch_bounds__(256) find_maxima(const FindMaxima<T> p) {
  constexpr uint32_t V = 16 / sizeof(T);
  chain_next();
  const bool queries = blockIdx.x >= p.row_blocks;
  const uint32_t block = queries ? blockIdx.x - p.row_blocks : blockIdx.x, grid = queries ? p.query_blocks : p.row_blocks;
  uint32_t best = 0;
  if (queries && block >= p.query_blocks) {
    for (uint32_t q = (block - p.query_blocks) * 256 + threadIdx.x; q < p.nq; q += p.grad_blocks * 256)
      if (has_target(p.targets[q], p.nrows)) best = max(best, finite_bits(p.grad[q]));
    best = block_max(best);
    if (threadIdx.x == 0) p.out->grad[block - p.query_blocks] = best;
    return;
  }
  const T *from = queries ? p.x : p.w;
  const uint64_t stride = queries ? p.x_stride : p.w_stride, rows = queries ? p.nq : p.nrows;
  const uint32_t cx = threadIdx.x % p.tx, ry = threadIdx.x / p.tx, ty = 256 / p.tx;
  const bool vec = stride % V == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0;
  for (uint64_t r = (uint64_t)block * ty + ry; r < rows; r += (uint64_t)grid * ty) {
    if (queries && !has_target(p.targets[r], p.nrows)) continue;
    const T *row = from + r * stride;
    for (uint32_t c = cx * V; c < p.dims; c += p.tx * V) {
      if (vec && c + V <= p.dims) {
        alignas(16) T v[V];
        *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(row + c));
#pragma unroll
        for (uint32_t j = 0; j < V; j++) best = max(best, finite_bits(to_float(v[j])));
      } else {
        for (uint32_t j = c; j < min(p.dims, c + V); j++) best = max(best, finite_bits(to_float(row[j])));
      }
    }
  }
  best = block_max(best);
  if (threadIdx.x == 0) (queries ? p.out->queries : p.out->rows)[block] = best;
}

// Operands in the layout TMA reads: `ld` values (a multiple of 8) a row, values
// past dims zero. FP32: two FP16 planes of x * 2^e; an infinity becomes NaN (its
// products with a low term of 0 would be). weighted: dW's queries, x * 2^e * unit /
// the largest unit (kGradScale); of FP16 operands too, with the e of all queries.
template <typename T, typename O, int PLANES> struct Layout {
  const T *x, *w;
  uint64_t x_stride, w_stride, nrows;
  uint32_t nq, dims, ld;
  uint32_t tx;                     // threads a row of w, 8 values each
  uint32_t query_blocks, row_blocks;
  const int64_t *targets;
  const float *grad;
  bool leave_out;                  // the gradient's: queries without a target become rows of zeros, one e for all
  O *xo, *wo, *weighted;
  float *xscale;                   // PLANES 2: 2^-e of each query
  Maxima *maxima;
};
template <typename T, typename O, int PLANES, bool MUL = PLANES == 2>
__device__ __forceinline__ void pack8(const T *row, uint32_t c, uint32_t dims, bool vec, bool zero, float mul, O *out,
                                      uint64_t plane) {
  alignas(16) T v[8];
  if (!zero && vec && c + 8 <= dims) {
#pragma unroll
    for (int j = 0; j < (int)(8 * sizeof(T) / 16); j++)
      reinterpret_cast<uint4 *>(v)[j] = __ldg(reinterpret_cast<const uint4 *>(row + c) + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = !zero && c + j < dims ? row[c + j] : from_float<T>(0.0f);
  }
  if constexpr (PLANES == 1) {
    if constexpr (MUL) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = from_float<T>(to_float(v[j]) * mul);
    }
    *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(v);
  } else {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float f[2], l[2];
      __half h[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        f[u] = to_float(v[2 * j + u]) * mul;
        if (isinf(f[u])) f[u] = NAN;
        h[u] = __float2half_rn(f[u]);
        l[u] = isnan(f[u]) ? 0.0f : f[u] - __half2float(h[u]);
      }
      hi[j] = pack16<__half>(f[0], f[1]);
      lo[j] = pack16<__half>(l[0], l[1]);
    }
    *reinterpret_cast<uint4 *>(out) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(out + plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}
template <typename T, typename O, int PLANES>
__global__ void __launch_bounds__(256) lay_out(const Layout<T, O, PLANES> p) {
  chain_wait();
  chain_next();
  uint32_t block = blockIdx.x;
  if (block < p.query_blocks) {   // a warp a query
    const uint32_t lane = threadIdx.x % 32;
    const bool vec = p.x_stride % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0;
    uint32_t all = 0;
    if ((PLANES == 2 && p.leave_out) || (kGradUnits<O> && p.weighted)) {
      all = join_parts(p.maxima->queries, kQueryParts);
      if (block == 0 && threadIdx.x == 0) p.maxima->all_queries = all;
    }
    float largest = 1.0f;
    if (kGradUnits<O> && p.weighted) largest = grad_unit(p.maxima);
    const uint32_t q = block * 8 + threadIdx.x / 32;
    if (q >= p.nq) return;
    const T *row = p.x + q * p.x_stride;
    if (PLANES == 2 && !p.leave_out) {
      for (uint32_t c = lane; c < p.dims; c += 32) all = max(all, finite_bits(to_float(row[c])));
      all = __reduce_max_sync(0xffffffffu, all);
    }
    const bool zero = p.leave_out && !has_target(p.targets[q], p.nrows);
    const float undo = undo_scale(all), mul = 1.0f / undo;   // powers of two: exact
    for (uint32_t c = lane * 8; c < p.ld; c += 256)
      pack8<T, O, PLANES>(row, c, p.dims, vec, zero, mul, p.xo + (uint64_t)q * p.ld + c, (uint64_t)p.nq * p.ld);
    if (PLANES == 2 && lane == 0) p.xscale[q] = undo;
    if constexpr (kGradUnits<O>) {
      if (p.weighted) {
        // 2^e unit / largest as an exponent, from -126 on (a weight that is not finite, or not a query's with a
        // target, is none of those that the largest is taken from)
        const uint32_t w = __float_as_uint(p.grad[q]) & 0x7fffffffu;
        const float unit = !zero && w < 0x7f800000u ? grad_unit(w) : largest;
        const int up = (int)(__float_as_uint(mul) >> 23) + (int)(__float_as_uint(unit) >> 23) -
                       (int)(__float_as_uint(largest) >> 23);
        const float m = __uint_as_float((uint32_t)max(up, 1) << 23);
        for (uint32_t c = lane * 8; c < p.ld; c += 256)
          pack8<T, O, PLANES, true>(row, c, p.dims, vec, zero, m, p.weighted + (uint64_t)q * p.ld + c,
                                    (uint64_t)p.nq * p.ld);
      }
    }
    return;
  }
  block -= p.query_blocks;
  if (block < p.row_blocks) {
    const uint32_t cx = threadIdx.x % p.tx, ry = threadIdx.x / p.tx, ty = 256 / p.tx;
    const bool vec = p.w_stride % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
    float mul = 1.0f;
    if (PLANES == 2) {
      const uint32_t all = join_parts(p.maxima->rows, kRowParts);
      mul = 1.0f / undo_scale(all);
      if (block == 0 && threadIdx.x == 0) p.maxima->all_rows = all;
    }
    for (uint64_t r = (uint64_t)block * ty + ry; r < p.nrows; r += (uint64_t)p.row_blocks * ty)
      for (uint32_t c = cx * 8; c < p.ld; c += p.tx * 8)
        pack8<T, O, PLANES>(p.w + r * p.w_stride, c, p.dims, vec, false, mul, p.wo + r * p.ld + c, p.nrows * p.ld);
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

// Tiles of 256 queries x 256 rows, 128 columns a thread. GRAD: G of a piece; else
// the partial sums. FEW: up to 128 queries, which both CTAs multiply with all 256
// rows; each takes the results of half of them, 64 columns a thread, where one
// would have had nothing to do.
template <PairKind KIND_, int PLANES_, bool GRAD, bool FEW, typename O>
struct LogitsOp : PairNoHelpers {
  static constexpr PairKind KIND = KIND_;
  static constexpr bool A_MN = false, B_MN = false, A_SAME = FEW;
  static constexpr int COLS = FEW ? 64 : 128, PARTS = 256 / COLS;   // columns a thread; partial sums a tile
  static constexpr int PLANES = PLANES_, SCRATCH = GRAD ? 2 * kPairEpi * kBoxBytes : 0, MAX_STAGES = 8;
  static constexpr int CHUNK = PLANES == 2 ? 2 : 6;   // 24 steps of the tensor cores
  struct Args {
    CUtensorMap a[PLANES], b[PLANES];
    uint32_t bn;
    uint32_t mt, nt, kblocks;
    uint32_t nq, q0;         // queries; the first one of this launch
    uint64_t nrows, first;   // rows; the first one of this piece
    double scale2;           // scale * log2(e)
    const float *xscale;     // PLANES 2: per query
    const Maxima *maxima;
    const int64_t *targets;
    float2 *part;            // forward: [query - q0][PARTS nt]
    float *tlogit;           // [query]
    const float *lse, *grad;
    CUtensorMap g[PLANES];   // gradient: G of the piece
    float *gsum;             // [query][gsums = PARTS x a piece's row tiles]: the stored G, summed over pieces
    uint32_t gsums;
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
    return (uint32_t)w.a_row + (FEW ? 0 : rank * 128) + ((threadIdx.x >> 5) & 3) * 32 + (threadIdx.x & 31);
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
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t share = (FEW ? 2 * rank : 0) + (warp >> 2);   // which columns of a tile
    const double scale2 = PLANES == 2 ? p.scale2 * (double)undo_scale(p.maxima->all_rows) : p.scale2;
    BoxStore box{scratch + 2 * warp * kBoxBytes};
    uint32_t turn = 0;
    Row next = row_of(p, cluster, rank);
    for (uint32_t i = cluster; i < items(p); i += clusters) {
      const PairItem w = item(p, i);
      const Row row = next;
      next = row_of(p, i + clusters, rank);
      const uint32_t q = query_of(w, rank);
      const bool valid = q < p.nq;
      const int64_t col0 = (int64_t)w.b_row + share * COLS;   // this thread's first row of W
      f32x2 v[COLS / 2];
      sums.template total<CHUNK, COLS / 32>(share * COLS, w.kblocks, v);
      if (!__any_sync(0xffffffffu, valid)) continue;
      float k = PLANES == 2 ? (float)(scale2 * (double)row.xscale) : (float)scale2;
      if (k == 0.0f) k = FLT_MIN;   // (0 would make NaNs of the infinities that stand for no column)
      const int64_t left = (int64_t)p.nrows - col0;         // columns that are rows of W
      // the target's column, COLS where it is not here
      const int64_t rel = row.target - col0;
      const int at = valid && rel >= 0 && rel < COLS ? (int)rel : COLS;
      const bool hit = __any_sync(0xffffffffu, at < COLS);
      float s = 0.0f;                                       // of this thread's columns
      if (!GRAD) {
        if (hit) {
          float t = 0.0f;
#pragma unroll
          for (int j = 0; j < COLS / 2; j++) {
            float a, b;
            unpack2(v[j], a, b);
            t = at == 2 * j ? a : (at == 2 * j + 1 ? b : t);
          }
          if (at < COLS) p.tlogit[q] = t * k;
        }
        if (left < COLS) {   // columns past the rows count for nothing
          const float none = k < 0.0f ? INFINITY : -INFINITY;
#pragma unroll
          for (int j = 0; j < COLS / 2; j++) {
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
          for (int j = 0; j < COLS / 2; j++) {
            float a, b;
            unpack2(v[j], a, b);
            top[j & 3] = min3(top[j & 3], a, b);
          }
        } else {
#pragma unroll
          for (int j = 0; j < COLS / 2; j++) {
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
        for (int j = 0; j < COLS / 2; j++) {
          float a, b;
          unpack2(fma2(v[j], kk, bb), a, b);
          e[j & 3] = add2(e[j & 3], pack2(exp2_approx(a), exp2_approx(b)));
        }
        float a, b;
        unpack2(add2(add2(e[0], e[1]), add2(e[2], e[3])), a, b);
        s = a + b;
        if (left <= 0) s = 0.0f;
        if (valid) p.part[(uint64_t)(q - p.q0) * (PARTS * p.nt) + PARTS * w.index + share] = make_float2(m, s);
      } else {
        // G; columns past the rows go to the buffer's end, which is not read
        const bool kept = valid && has_target(row.target, p.nrows);
        // p = exp2(l2 - lse2) c: c is what rounding lse2 (the lse in base 2) lost
        const float lse2 = row.lse * kLog2e;
        const float c = exp2f(-(fmaf(row.lse, kLog2e, -lse2) + row.lse * kLog2eLow));
        const float held = kGradUnits<O> ? row.grad / grad_unit(__float_as_uint(row.grad) & 0x7fffffffu) * kGradScale
                                         : row.grad;
        const float g = kept ? held * c : 0.0f, one = 1.0f / c;
        const f32x2 kk = pack2(k, k), zz = pack2(-lse2, -lse2), gg = pack2(g, g);
#pragma unroll
        for (int j = 0; j < COLS / 2; j++) {
          float a, b;
          unpack2(fma2(v[j], kk, zz), a, b);
          v[j] = pack2(exp2_approx(a), exp2_approx(b));
        }
        if (hit) {
#pragma unroll
          for (int j = 0; j < COLS / 2; j++)
            v[j] = add2(v[j], pack2(at == 2 * j ? -one : 0.0f, at == 2 * j + 1 ? -one : 0.0f));
        }
#pragma unroll
        for (int j = 0; j < COLS / 2; j++) v[j] = mul2(v[j], gg);
        if (!kept) {        // (not 0 times what the query holds)
#pragma unroll
          for (int j = 0; j < COLS / 2; j++) v[j] = 0;
        }
        if (left < COLS) {
#pragma unroll
          for (int j = 0; j < COLS / 2; j++) {
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
          for (int h = 0; h < COLS / 64; h++) {
            box.box = scratch + (2 * warp + (turn++ & 1)) * kBoxBytes;   // two boxes in turn
            box.reuse<1>();
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
        if (valid) {   // (the same thread of every piece's tile: added in order)
          float *sum_at = p.gsum + (uint64_t)q * p.gsums + PARTS * w.index + share;
          *sum_at = p.first ? *sum_at + s : s;
        }
      }
    }
  }
};

// Join a query's partial sums: lse = (m + log2 s) ln 2, loss = lse - target logit.
__global__ void __launch_bounds__(128) join_sums(const float2 *part, uint32_t n, uint32_t q0, uint64_t nrows,
                                                  const int64_t *targets, const float *tlogit, float *loss, float *lse,
                                                  int32_t *status) {
  chain_wait();
  chain_next();
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
  static constexpr int CHUNK = PLANES == 2 ? 2 : 64;   // 24 or 256 steps of the tensor cores
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
    sums.template total<CHUNK, 4>(half * cols, w.kblocks, v);
    BoxStore box{scratch + warp * kBoxBytes};
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
      const uint32_t d0 = (uint32_t)w.b_row + half * cols + c * 32;
      if (c * 32 >= cols || d0 >= p.dims || q - lane >= p.nq) break;
      uint32_t r[32];
#pragma unroll
      for (int j = 0; j < 16; j++) {
        float a, b;
        unpack2(v[16 * c + j], a, b);
        r[2 * j] = __float_as_uint(a);
        r[2 * j + 1] = __float_as_uint(b);
      }
      box.reuse();
#pragma unroll
      for (int j = 0; j < 8; j++) box.put(j, make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]));
      box.store_sums(&p.part, (int32_t)d0, (int32_t)(q - lane), (int32_t)w.index, p.add != 0);
    }
  }
};

// dW: 256 of the piece's rows x bn dimensions, K = the queries.
template <PairKind KIND_, int PLANES_, typename T, typename O>
struct RowsOp : PairNoHelpers {
  static constexpr PairKind KIND = KIND_;
  static constexpr bool A_MN = true, B_MN = true;
  static constexpr int PLANES = PLANES_, SCRATCH = kPairEpi * kBoxBytes, MAX_STAGES = 8;
  static constexpr int CHUNK = PLANES == 2 ? 2 : 64;   // 24 or 256 steps of the tensor cores
  struct Args {
    CUtensorMap a[PLANES], b[PLANES];   // G (piece columns); X, weighted where the queries have weights
    uint32_t bn;
    uint32_t mt, nt, kblocks;
    uint32_t rows, dims;     // rows of the piece
    double scale;
    bool weighted;
    const Maxima *maxima;
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
    double f = p.scale;
    if (kGradUnits<O>) {
      f /= kGradScale;
      if (p.weighted) f *= (double)grad_unit(p.maxima);
      if (PLANES == 2 || p.weighted) f *= (double)undo_scale(p.maxima->all_queries);
    }
    const float factor = (float)f;
    const uint32_t cols = p.bn / 2;
    f32x2 v[64];
    sums.template total<CHUNK, 4>(half * cols, w.kblocks, v);
    BoxStore box{scratch + warp * kBoxBytes};
    constexpr uint32_t BOX = 128 / sizeof(T), V = 16 / sizeof(T);   // values of a box row, of a chunk
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
      const uint32_t d0 = (uint32_t)w.b_row + half * cols + c * 32;
      if (c * 32 >= cols || d0 >= p.dims || i - lane >= p.rows) break;
      uint32_t r[32];
#pragma unroll
      for (int j = 0; j < 16; j++) {
        float a, b;
        unpack2(v[16 * c + j], a, b);
        r[2 * j] = __float_as_uint(a);
        r[2 * j + 1] = __float_as_uint(b);
      }
      const uint32_t at = c * 32 % BOX;     // of the box's values
      if (at == 0) box.reuse();
#pragma unroll
      for (uint32_t j = 0; j < 32; j += V) {
        alignas(16) T o[V];
#pragma unroll
        for (uint32_t u = 0; u < V; u++) o[u] = from_float<T>(__uint_as_float(r[j + u]) * factor);
        box.put((at + j) / V, *reinterpret_cast<uint4 *>(o));
      }
      // the last 32 values of a box, or of the row
      if (at + 32 == BOX || d0 + 32 >= p.dims) {
        const uint32_t x = d0 - at, y = i - lane;
        if (p.boxes) box.store(&p.map, (int32_t)(x * (sizeof(T) / 2)), (int32_t)y);   // (in 16-bit values)
        else box.copy(p.out + (uint64_t)y * p.dims + x, p.dims, min(32u, p.rows - y), min(BOX, p.dims - x));
      }
    }
  }
};

// dX_i = scale * (the partial sums, in order, - (sum_j G_ij) w_target); zero for
// a query without a target. G's exact rows sum to 0, the rounded ones do not,
// and rows near each other (a cluster's) make sum_j G_ij w_j the small
// difference of large terms: what is left of the sum would weigh in with a
// whole row (10 times G's rounding where a cluster's rows differ by a tenth of
// their length). With it taken off at the target, the sum is over
// G_ij (w_j - w_target), and errors are relative to the differences.
template <typename T, typename O, int PLANES>
__global__ void __launch_bounds__(256) join_queries(const float *part, uint32_t splits, uint32_t nq, uint32_t dims,
                                                    double scale, const float *grad, const Maxima *maxima, const float *gsum,
                                                    uint32_t gsums, const T *rows, uint64_t stride,
                                                    const int64_t *targets, uint64_t nrows, T *out) {
  chain_wait();
  const uint32_t q = blockIdx.x, ld = (dims + 3) / 4 * 4;
  const uint64_t plane = (uint64_t)nq * ld;
  const int64_t t = targets[q];
  T *to = out + (uint64_t)q * dims;
  if (!has_target(t, nrows)) {
    for (uint32_t d = threadIdx.x; d < dims; d += 256) to[d] = from_float<T>(0.0f);
    return;
  }
  double f = scale;
  if (kGradUnits<O>) f *= (double)(grad ? grad_unit(__float_as_uint(grad[q]) & 0x7fffffffu) : 1.0f) / kGradScale;
  // the partial sums are in units of the rows' undo: the target's row is brought there, powers of two
  const float undo = PLANES == 2 ? undo_scale(maxima->all_rows) : 1.0f, up = 1.0f / undo;
  const float factor = (float)(f * (double)undo);
  const T *row = rows + (uint64_t)t * stride;
  const float *at = part + (uint64_t)q * ld;
  constexpr uint32_t EACH = 4;     // dimensions a thread: loaded before the sum of G is waited for
  float v[EACH], r[EACH];
  auto load = [&](uint32_t d0) {
#pragma unroll
    for (uint32_t u = 0; u < EACH; u++) {
      const uint32_t d = d0 + threadIdx.x + 256 * u;
      v[u] = 0.0f;
      r[u] = 0.0f;
      if (d < dims) {
        r[u] = to_float(row[d]) * up;
        for (uint32_t k = 0; k < splits; k++) v[u] += at[k * plane + d];
      }
    }
  };
  load(0);
  __shared__ double sum[8];
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < gsums; i += 256) s += gsum[(uint64_t)q * gsums + i];
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (threadIdx.x % 32 == 0) sum[threadIdx.x / 32] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 8; i++) s += sum[i];
  const float left = -(float)s;
  for (uint32_t d0 = 0; d0 < dims; d0 += 256 * EACH) {
    if (d0) load(d0);
#pragma unroll
    for (uint32_t u = 0; u < EACH; u++) {
      const uint32_t d = d0 + threadIdx.x + 256 * u;
      if (d < dims) to[d] = from_float<T>(fmaf(left, r[u], v[u]) * factor);
    }
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
  bool weighted;           // dW's queries are laid out apart (kGradScale)
  uint64_t x, w, xw, xscale, maxima, part, tlogit, g, gsum, dq, total;
  bool few;                // up to 128 queries (LogitsOp)
  uint32_t parts;          // partial sums a tile
  uint32_t nt, chunk;      // row tiles; forward: queries a launch
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
  p.maxima = c.take(sizeof(Maxima));
  p.xscale = c.take(nq * 4);
  if (p.pack_x) p.x = c.take(nq * p.ld * 2 * p.planes);
  if (p.pack_w) p.w = c.take(j.nrows * p.ld * 2 * p.planes);
  p.weighted = grad && j.grad && j.dtype != ANNB200_BF16;
  if (grad && j.dtype != ANNB200_BF16) p.xw = c.take(nq * p.ld * 2 * p.planes);   // (whether or not grad is set yet)
  p.nt = (uint32_t)((j.nrows + 255) / 256);
  p.few = nq <= 128;
  p.parts = p.few ? 4 : 2;
  if (!grad) {
    p.chunk = (uint32_t)std::min<uint64_t>(up(nq, 256), std::max<uint64_t>(256, kPartBytes / (8ull * p.parts * p.nt) / 256 * 256));
    p.part = c.take(std::min<uint64_t>(nq, p.chunk) * p.nt * p.parts * 8);
    p.tlogit = c.take(nq * 4);
  } else {
    // a piece: G of kPieceBytes, but 8,192 rows at least, since each piece adds
    // to dX's sums, as long as G stays within kMostPieceBytes
    const uint64_t row_bytes = 2ull * p.planes * nq;
    p.piece = std::max<uint64_t>({256, std::min<uint64_t>(8192, kMostPieceBytes / row_bytes / 256 * 256),
                                  kPieceBytes / row_bytes / 256 * 256});
    p.piece = std::min<uint64_t>({p.piece, up(j.nrows, 256), 1u << 20});
    p.g = c.take(nq * p.piece * 2 * p.planes);
    p.gsum = c.take(nq * p.parts * (p.piece / 256) * 4);
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

// T: the operands' type; O: the products'.
template <typename T, typename O, PairKind KIND, int PLANES, bool FEW>
int run_loss(const AnnB200LossJob &j, bool grad, cudaStream_t st) {
  const Plan p = plan_of(j, grad);
  const int sms = op_sms();
  if (sms < 2) return report_error(OP_BACKEND_ERROR, "no current CUDA device");
  uint8_t *ws = static_cast<uint8_t *>(j.workspace);
  Maxima *maxima = reinterpret_cast<Maxima *>(ws + p.maxima);
  float *xscale = reinterpret_cast<float *>(ws + p.xscale);
  const T *x = static_cast<const T *>(j.queries), *w = static_cast<const T *>(j.rows);
  unsigned long long launches = 0;
  cudaError_t e = cudaSuccess;

  // operands as the tensor maps read them
  const O *xo = reinterpret_cast<const O *>(x), *wo = reinterpret_cast<const O *>(w);
  uint64_t xld = j.query_stride, wld = j.row_stride;
  Layout<T, O, PLANES> lay = {};
  lay.x = x;
  lay.w = w;
  lay.x_stride = j.query_stride;
  lay.w_stride = j.row_stride;
  lay.nrows = j.nrows;
  lay.nq = j.nq;
  lay.dims = j.dims;
  lay.ld = p.ld;
  lay.tx = 1;
  while (lay.tx < 256 && lay.tx * 8 < p.ld) lay.tx *= 2;
  lay.targets = j.targets;
  lay.grad = j.grad;
  lay.leave_out = grad;
  lay.xscale = xscale;
  lay.maxima = maxima;
  if (p.pack_x) {
    lay.query_blocks = (j.nq + 7) / 8;
    xo = lay.xo = reinterpret_cast<O *>(ws + p.x);
    xld = p.ld;
  }
  if (p.pack_w) {
    const uint64_t per = 256 / lay.tx;
    lay.row_blocks = (uint32_t)std::min<uint64_t>((j.nrows + per - 1) / per, PLANES == 2 ? 4736 : 1u << 16);
    wo = lay.wo = reinterpret_cast<O *>(ws + p.w);
    wld = p.ld;
  }
  const bool weighted = p.weighted && j.drows;
  if (weighted) lay.weighted = reinterpret_cast<O *>(ws + p.xw);
  if (PLANES == 2 || weighted) {
    FindMaxima<T> find = {};
    find.w = w;
    find.x = x;
    find.w_stride = j.row_stride;
    find.x_stride = j.query_stride;
    find.nrows = j.nrows;
    find.nq = j.nq;
    find.dims = j.dims;
    find.tx = 1;
    while (find.tx < 256 && find.tx * (16 / sizeof(T)) < j.dims) find.tx *= 2;
    find.row_blocks = PLANES == 2 ? kRowParts : 0;
    find.query_blocks = grad ? kQueryParts : 0;
    find.grad_blocks = weighted ? kGradParts : 0;
    find.targets = j.targets;
    find.grad = j.grad;
    find.out = maxima;
    find_maxima<<<find.row_blocks + find.query_blocks + find.grad_blocks, 256, 0, st>>>(find);
    launches++;
  }
  if (const uint32_t blocks = lay.query_blocks + lay.row_blocks) {
    e = launch_chained(launches > 0, lay_out<T, O, PLANES>, blocks, 256, 0, st, lay);
    launches++;
    if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss: %s", cudaGetErrorString(e));
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
    using Op = LogitsOp<KIND, PLANES, false, FEW, O>;
    typename Op::Args l = {};
    logits(l);
    l.nt = p.nt;
    l.part = reinterpret_cast<float2 *>(ws + p.part);
    l.tlogit = reinterpret_cast<float *>(ws + p.tlogit);
    if (!maps) return report_error(OP_BACKEND_ERROR, "softmax loss: tensor map");
    for (uint32_t q0 = 0; q0 < j.nq && e == cudaSuccess; q0 += p.chunk) {
      const uint32_t n = std::min(p.chunk, j.nq - q0);
      l.q0 = q0;
      l.mt = (n + 255) / 256;
      // (a launch covers whole tiles of queries, except at their end)
      e = launch_pair<Op>(l, l.mt * l.nt, sms, st, launches > 0);
      if (e != cudaSuccess) break;
      e = launch_chained(true, join_sums, n, 128, 0, st, l.part, p.parts * p.nt, q0, j.nrows, j.targets, l.tlogit,
                         j.loss, j.lse, j.status);
      launches += 2;
    }
    if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss: %s", cudaGetErrorString(e));
    return op_launched("softmax loss", launches);
  }

  O *g = reinterpret_cast<O *>(ws + p.g);
  float *dq = reinterpret_cast<float *>(ws + p.dq);
  const uint64_t gplane = (uint64_t)j.nq * p.piece;
  using LOp = LogitsOp<KIND, PLANES, true, FEW, O>;
  using QOp = QueriesOp<KIND, PLANES>;
  using ROp = RowsOp<KIND, PLANES, T, O>;
  typename LOp::Args l = {};
  logits(l);
  l.mt = (j.nq + 255) / 256;
  l.lse = j.lse;
  l.grad = j.grad;
  map(l.g, g, p.piece, j.nq, p.piece, gplane, 32);
  l.gsum = reinterpret_cast<float *>(ws + p.gsum);
  l.gsums = (uint32_t)(p.parts * (p.piece / 256));
  for (uint64_t first = 0; first < j.nrows && e == cudaSuccess; first += p.piece) {
    const uint64_t n = std::min(p.piece, j.nrows - first);
    l.first = first;
    l.nt = (uint32_t)((n + 255) / 256);
    e = maps ? launch_pair<LOp>(l, l.mt * l.nt, sms, st, true) : cudaErrorInvalidValue;
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
      e = maps ? launch_pair<QOp>(a, a.mt * a.nt * a.splits, sms, st, true) : cudaErrorInvalidValue;
      launches++;
    }
    if (j.drows && e == cudaSuccess) {
      typename ROp::Args a = {};
      map(a.a, g, n, j.nq, p.piece, gplane, 64);
      map(a.b, weighted ? lay.weighted : xo, j.dims, j.nq, xld, (uint64_t)j.nq * p.ld, 64);
      a.weighted = weighted;
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
      e = maps ? launch_pair<ROp>(a, a.mt * a.nt, sms, st, true) : cudaErrorInvalidValue;
      launches++;
    }
  }
  if (j.dqueries && e == cudaSuccess) {
    e = launch_chained(true, join_queries<T, O, PLANES>, j.nq, 256, 0, st, dq, p.splits, j.nq, j.dims, (double)j.scale,
                       j.grad, maxima, l.gsum, l.gsums, w, j.row_stride, j.targets, j.nrows, static_cast<T *>(j.dqueries));
    launches++;
  }
  if (e != cudaSuccess) return report_error(OP_BACKEND_ERROR, "softmax loss gradient: %s", cudaGetErrorString(e));
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
  const bool few = j->nq <= 128;
  switch (j->dtype) {
    case ANNB200_F32:
      return few ? run_loss<float, __half, PAIR_F16, 2, true>(*j, grad, st)
                 : run_loss<float, __half, PAIR_F16, 2, false>(*j, grad, st);
    case ANNB200_F16:
      return few ? run_loss<__half, __half, PAIR_F16, 1, true>(*j, grad, st)
                 : run_loss<__half, __half, PAIR_F16, 1, false>(*j, grad, st);
    default:
      return few ? run_loss<__nv_bfloat16, __nv_bfloat16, PAIR_BF16, 1, true>(*j, grad, st)
                 : run_loss<__nv_bfloat16, __nv_bfloat16, PAIR_BF16, 1, false>(*j, grad, st);
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
