// pair_gemm.cuh - the tensor-core product loop of the operators: C = A B^T in
// tiles of 256 rows by up to 256 columns, one tile at a time on a pair of SMs.
//
// A cluster of two CTAs works on one tile with tcgen05.mma.cta_group::2: each
// CTA keeps its 128 rows of A and its half of B's columns in shared memory and
// its 128 x N part of the FP32 sums in tensor memory. Against one CTA a tile
// that halves what is loaded of B for the same products. Clusters are
// persistent: cluster c takes items c, c + clusters, ... of the operator's
// list. Roles in each CTA:
//
//   warps 0-7  epilogue: warp w reads tensor memory lanes 32 (w % 4) .. + 31
//              and columns of the half w / 4, so a thread holds half a row.
//   warp 8     TMA producer: the CTA's own tiles of each 128-byte K block, all
//              completing on the leader CTA's barrier.
//   warp 9     MMA issuer (leader CTA); tcgen05.commit frees the stage and
//              publishes the sums in both CTAs.
//   10 and 11  an operator's helpers, if it has any.
//
// Two sums of 256 columns each (more, where a tile has fewer columns) let the
// epilogue of one run under the products of the next. The tensor cores cut off,
// and do not round, what falls below a sum's last bit: over 48 steps of 16 (768
// dimensions) that came to 1.4e-6 of the sum, all of one sign, against 3e-8 in
// FP32 arithmetic, and over 2^21 queries (dW) to 0.7 %. So a sum is taken over
// CHUNK K blocks and the chunks are added up in registers, rounded: 24 steps where
// a result keeps 24 bits, 256 (at most 2^-15 of the sum) where it keeps 11 or 8,
// which costs under 1 % (4,096 x 65,536 x 768 bf16: 1,521 -> 1,530 us).
//
// Operands are K-major (rows of K) or MN-major (K rows of M or N, the transposed
// operand read as it lies), both in 128-byte-swizzled tiles. With two planes an
// operand is the sum of two FP16 terms and a K step issues three products of the
// four.
//
// What bounds it: a 256 x 256 tile's K block of 128 bytes is 512 clocks of
// products; with little in the epilogue 660 to 690 were measured (412 GFLOP of
// bf16 in 270 us, 1,526 TFLOP/s; the measured cuBLAS burst is 1,642), during
// which each SM takes in 32 KB, 46 bytes a clock. Short sums add a tile's
// setup and, once, the kernel's (1.2 us before the first load).
//
// Every wait is bounded; one that runs out ends the CTA's roles, and its
// epilogue goes through its remaining items with NaN for their sums.
#pragma once

#include <atomic>

#include "ops.cuh"
#include "tc.cuh"

namespace annb200 {

constexpr int kPairEpi = 8;                          // epilogue warps
constexpr int kPairThreads = 32 * (kPairEpi + 4);    // whole warpgroups, for the register split
// Registers a thread: 384 threads start with 168 each. The epilogue's 256 go up
// to 224 and the other 128 down to 56, each side at the top of its own branch,
// which no other joins. Together they take no more than the block started with.
constexpr int kPairEpiRegs = 224, kPairOtherRegs = 56;
static_assert(256 * kPairEpiRegs + 128 * kPairOtherRegs <= 384 * 168, "more registers than the block starts with");
constexpr int kPairTileBytes = 128 * 128;     // 128 rows of 128 bytes (or 128 bytes wide, 128 K rows)
constexpr int kPairSmem = 227 * 1024;

struct PairItem {
  int32_t a_row, b_row;   // first row of the tile's A and B (rows of the product, whichever way they lie)
  int32_t k0;             // first K element
  uint32_t kblocks;
  uint32_t index;         // the operator's own
};

enum PairKind { PAIR_F16, PAIR_BF16, PAIR_E4M3 };

// Instruction descriptor of a 256 x n tile over two SMs, FP32 sums.
template <PairKind KIND, bool A_MN, bool B_MN>
__device__ __forceinline__ uint32_t pair_idesc(uint32_t n) {
  const uint32_t fmt = KIND == PAIR_BF16 ? 1u : 0u;   // F16 and E4M3 are both 0 in their kinds
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
         ((n >> 3) << 17) | ((256u >> 4) << 24);
}

// Descriptor of an MN-major operand in the 128-byte swizzle: 128-byte runs of
// M/N, a row of them per K element; 8 K rows (1,024 bytes) apart along K,
// `lead` bytes to the next 64 M/N elements.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <PairKind KIND>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (KIND == PAIR_E4M3)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrive on the barrier at this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void pair_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Relaxed: what it tells (tensor memory has been read, tcgen05.wait::ld) is in
// registers; a release would wait for the epilogue's stores to memory as well.
__device__ __forceinline__ void remote_arrive(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// A tile into this CTA's dst; completes on the leader's barrier (a cluster address).
__device__ __forceinline__ void pair_load(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// What bounds a CTA's waits: the flag that a role has given up, and the launch's
// limit (pipeline_wait_ns), read only after some tries.
constexpr uint32_t kTryNs = 100000;
struct PairBounds {
  uint32_t abort;
  uint32_t pad;
  uint64_t ns;
};
// Wait for a phase, at most the limit and until another role of the CTA has given
// up. Each try may sleep up to the hint (100 us) and wakes when the phase ends:
// warps that poll take issue slots and shared-memory accesses from the others.
// The result is the thread's own: a phase can end, or a role give up, between two
// lanes' tries. A warp that goes on together takes __all_sync of it.
__device__ __forceinline__ bool pair_try_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(kTryNs)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool pair_wait(uint64_t *bar, uint32_t parity, volatile PairBounds *bounds) {
  if (pair_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  for (;;) {
    for (int i = 0; i < 32; i++)
      if (pair_try_wait(bar, parity)) return true;
    if (bounds->abort) return false;
    if (globaltimer() - t0 > bounds->ns) {
      bounds->abort = 1;
      return false;
    }
  }
}

// A warp's way out to memory: 32 rows of 128 bytes, a row a lane, put into
// shared memory in the 128-byte swizzle (each 16-byte chunk once: no bank
// conflicts) and stored as one box by the TMA, whole lines at a time. Rows past
// the tensor's end are left out by the TMA, columns 16 bytes at a time: a row whose
// end is not on a 16-byte boundary needs room up to it, or `copy` for its last box.
constexpr int kBoxBytes = 32 * 128;
struct BoxStore {
  uint8_t *box;
  // A row's 16-byte chunk.
  __device__ __forceinline__ uint8_t *at(uint32_t row, uint32_t chunk) const {
    return box + row * 128 + ((chunk ^ (row & 7)) << 4);
  }
  // Before the box is filled again: what was stored from it has been read (all
  // but the warp's last LATER stores have).
  template <int LATER = 0>
  __device__ __forceinline__ void reuse() {
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LATER) : "memory");
    __syncwarp();
  }
  __device__ __forceinline__ void put(uint32_t chunk, uint4 v) {
    *reinterpret_cast<uint4 *>(at(threadIdx.x & 31, chunk)) = v;
  }
  __device__ __forceinline__ void store(const CUtensorMap *map, int32_t x, int32_t y) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                       reinterpret_cast<uint64_t>(map)),
                   "r"(x), "r"(y), "r"(smem_u32(box))
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  // The box's first `rows` rows and `cols` values into rows the TMA cannot store
  // to (not on 16-byte boundaries), 32 values of a row at a time.
  template <typename T>
  __device__ __forceinline__ void copy(T *out, uint64_t stride, uint32_t rows, uint32_t cols) {
    const uint32_t lane = threadIdx.x & 31;
    constexpr uint32_t EACH = 4 / sizeof(T);   // values a lane, 32 apart
    __syncwarp();
#pragma unroll 4
    for (uint32_t r = 0; r < rows; r++)
#pragma unroll
      for (uint32_t u = 0; u < EACH; u++) {
        const uint32_t e = lane + 32 * u, byte = e * sizeof(T);
        if (e < cols) out[r * stride + e] = *reinterpret_cast<const T *>(at(r, byte >> 4) + (byte & 15));
      }
    __syncwarp();
  }
  // FP32 into a plane, stored or added.
  __device__ __forceinline__ void store_sums(const CUtensorMap *map, int32_t x, int32_t y, int32_t z, bool add) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      if (add)
        asm volatile(
            "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                reinterpret_cast<uint64_t>(map)),
            "r"(x), "r"(y), "r"(z), "r"(smem_u32(box))
            : "memory");
      else
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                         reinterpret_cast<uint64_t>(map)),
                     "r"(x), "r"(y), "r"(z), "r"(smem_u32(box))
                     : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  static __device__ __forceinline__ void finish() {
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
};

// What an epilogue warp needs of the loop: the sums of one accumulator after
// another. `ok` stays false once a wait has run out.
template <int ACCS>
struct PairSumsOf {
  static constexpr uint32_t WIDTH = 512 / ACCS;   // columns of an accumulator
  uint64_t *full;
  uint32_t empty_leader;     // cluster address of the leader's empty[0]
  volatile PairBounds *bounds;
  uint32_t tmem;
  uint32_t n;
  bool ok;
  // Tensor memory address of the next accumulator's columns for this warp's lanes.
  __device__ __forceinline__ uint32_t acquire() {
    if (ok) ok = __all_sync(0xffffffffu, pair_wait(full + n % ACCS, (n / ACCS) & 1, bounds));
    tc_fence_after();
    return tmem + (n % ACCS) * WIDTH;
  }
  __device__ __forceinline__ void release() {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0 && ok) remote_arrive(empty_leader + (n % ACCS) * 8);
    n++;
  }
  // N x 32 columns from `at` on, of the item's whole K: its chunks, added up.
  template <int CHUNK, int N>
  __device__ __forceinline__ void total(uint32_t at, uint32_t kblocks, f32x2 (&v)[16 * N]) {
#pragma unroll
    for (int j = 0; j < 16 * N; j++) v[j] = 0;
#pragma unroll 1
    for (uint32_t kb = 0; kb < kblocks; kb += CHUNK) {
      const uint32_t addr = acquire() + at;
      if (ok) {
        // one read ahead of the additions
        uint32_t r[2][32];
        TMEM_LD32(addr, r[0]);
        tmem_ld_wait();
        TMEM_KEEP32(r[0]);
#pragma unroll
        for (int c = 0; c < N; c++) {
          if (c + 1 < N) TMEM_LD32(addr + (c + 1) * 32, r[(c + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 16; j++)
            v[16 * c + j] = add2(v[16 * c + j],
                                 pack2(__uint_as_float(r[c & 1][2 * j]), __uint_as_float(r[c & 1][2 * j + 1])));
          if (c + 1 < N) {
            tmem_ld_wait();
            TMEM_KEEP32(r[(c + 1) & 1]);
          }
        }
      }
      release();
    }
    if (!ok) {
#pragma unroll
      for (int j = 0; j < 16 * N; j++) v[j] = pack2(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u));
    }
  }
};

using PairSums = PairSumsOf<2>;

// The shared memory of an operator's loop: stages of (A planes, B planes), the
// epilogue's scratch, barriers.
template <class Op>
struct PairShape {
  static constexpr int A_BYTES = Op::PLANES * kPairTileBytes;
  static constexpr int BAR_BYTES = 384;
  // b_bytes: one plane's B tile of this CTA
  static __host__ __device__ constexpr int stage(int b_bytes) { return A_BYTES + Op::PLANES * b_bytes; }
  static __host__ __device__ constexpr int stages(int b_bytes) {
    const int s = (kPairSmem - 1024 - BAR_BYTES - Op::SCRATCH) / stage(b_bytes);
    return s < Op::MAX_STAGES ? s : Op::MAX_STAGES;
  }
  static constexpr int smem(int b_bytes) { return 1024 + stages(b_bytes) * stage(b_bytes) + BAR_BYTES + Op::SCRATCH; }
};

// Op: KIND, A_MN, B_MN, PLANES, SCRATCH (bytes), MAX_STAGES (<= 12), CHUNK (K blocks a
// sum), ACCS (sums in tensor memory at a time: 512 / ACCS >= bn),
// A_SAME (both CTAs take the same 128 rows of A), HELPERS (0 or 2 warps), Args with maps a[PLANES],
// b[PLANES] and bn (columns of a tile), items(args), item(args, i),
// epilogue(args, sums, scratch, rank, cluster, clusters): all of the cluster's
// items; init and help where there are helpers.
struct PairNoHelpers {
  static constexpr int HELPERS = 0, ACCS = 2;
  static constexpr bool A_SAME = false;
  static __device__ __forceinline__ void init(uint8_t *) {}
  template <class Args>
  static __device__ __forceinline__ void help(const Args &, uint8_t *, uint32_t, uint32_t, uint32_t,
                                              volatile PairBounds *) {}
};

template <class Op>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_gemm(const __grid_constant__ typename Op::Args args, const uint64_t wait_ns) {
  using Shape = PairShape<Op>;
  constexpr int PLANES = Op::PLANES;
  constexpr int KE = Op::KIND == PAIR_E4M3 ? 128 : 64;   // K elements of a block
  constexpr int MAXS = Op::MAX_STAGES, ACCS = Op::ACCS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t b_bytes = args.bn * 64;                 // bn / 2 rows (or columns) of 128 bytes each K block
  const uint32_t stage_bytes = Shape::stage(b_bytes);
  const uint32_t stages = Shape::stages(b_bytes);
  uint8_t *scratch = smem + stages * stage_bytes;        // 1,024-byte aligned
  uint64_t *full = reinterpret_cast<uint64_t *>(scratch + Op::SCRATCH);
  uint64_t *empty = full + MAXS;
  uint64_t *tfull = empty + MAXS;
  uint64_t *tempty = tfull + ACCS;
  uint64_t *drain = tempty + ACCS;
  PairBounds *bounds = reinterpret_cast<PairBounds *>(drain + 1);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bounds + 1);
  static_assert((2 * MAXS + 2 * ACCS + 1) * 8 + sizeof(PairBounds) + 4 <= Shape::BAR_BYTES, "barriers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const uint32_t items = Op::items(args);

  if (threadIdx.x == 0) {
    Op::init(scratch);
    for (uint32_t s = 0; s < stages; s++) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < ACCS; b++) {
      mbar_init(tfull + b, 1);
      mbar_init(tempty + b, 2 * kPairEpi);
    }
    mbar_init(drain, 1);
    *bounds = {0u, 0u, wait_ns};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPairEpi + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_wait();
  chain_next();

  if (warp < kPairEpi) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairEpiRegs));
    PairSumsOf<ACCS> sums{tfull, map_to_leader(smem_u32(tempty)), bounds, tmem + (((uint32_t)warp & 3u) << 21), 0u, true};
    Op::epilogue(args, sums, scratch, rank, cluster, clusters);
    BoxStore::finish();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairOtherRegs));
    if (warp == kPairEpi) {
      if (lane == 0) {
        uint32_t s = 0, round = 0;
        // (a limit below one try's sleep could not run out while loads come in: it stands for loads that never do)
        bool ok = wait_ns >= kTryNs;
        for (uint32_t i = cluster; i < items && ok; i += clusters) {
          const PairItem w = Op::item(args, i);
          const int32_t ar = w.a_row + (Op::A_SAME ? 0 : (int32_t)rank * 128), br = w.b_row + (int32_t)(rank * (args.bn / 2));
          for (uint32_t kb = 0; kb < w.kblocks; kb++) {
            if (!pair_wait(empty + s, (round & 1) ^ 1, bounds)) {
              ok = false;
              break;
            }
            const uint32_t bar = map_to_leader(smem_u32(full + s));
            if (rank == 0) mbar_expect_tx(full + s, 2 * stage_bytes);
            const int32_t k = w.k0 + (int32_t)(kb * KE);
            const uint32_t a = smem_u32(smem + s * stage_bytes), b = a + Shape::A_BYTES;
#pragma unroll
            for (int p = 0; p < PLANES; p++) {
              if (Op::A_MN) {
                pair_load(a + p * kPairTileBytes, &args.a[p], ar, k, bar);
                pair_load(a + p * kPairTileBytes + 8192, &args.a[p], ar + 64, k, bar);
              } else {
                pair_load(a + p * kPairTileBytes, &args.a[p], k, ar, bar);
              }
              if (Op::B_MN) {
                for (uint32_t c = 0; c < args.bn / 2; c += 64)
                  pair_load(b + p * b_bytes + c * 128, &args.b[p], br + (int32_t)c, k, bar);
              } else {
                pair_load(b + p * b_bytes, &args.b[p], k, br, bar);
              }
            }
            if (++s == stages) {
              s = 0;
              round++;
            }
          }
        }
      }
      __syncwarp();
    } else if (warp == kPairEpi + 1) {
      if (lane == 0 && rank == 0) {
        const uint32_t idesc = pair_idesc<Op::KIND, Op::A_MN, Op::B_MN>(args.bn);
        constexpr uint32_t A_STEP = Op::A_MN ? 2048 : 32, B_STEP = Op::B_MN ? 2048 : 32;
        uint32_t s = 0, round = 0, acc = 0;
        bool ok = true;
        for (uint32_t i = cluster; i < items && ok; i += clusters) {
          const PairItem w = Op::item(args, i);
          for (uint32_t kb = 0; kb < w.kblocks; kb++) {
            const bool first = kb % Op::CHUNK == 0;
            const bool last = kb + 1 == w.kblocks || (kb + 1) % Op::CHUNK == 0;
            if (first && !pair_wait(tempty + acc % ACCS, ((acc / ACCS) & 1) ^ 1, bounds)) {
              ok = false;
              break;
            }
            if (!pair_wait(full + s, round & 1, bounds)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d = tmem + (acc % ACCS) * (512 / ACCS);
            const uint32_t a = smem_u32(smem + s * stage_bytes), b = a + Shape::A_BYTES;
            auto adesc = [&](uint32_t p, uint32_t kk) {
              const uint32_t at = a + p * kPairTileBytes + kk * A_STEP;
              return Op::A_MN ? sw128_mn_desc(at, 8192) : sw128_desc(at);
            };
            auto bdesc = [&](uint32_t p, uint32_t kk) {
              const uint32_t at = b + p * b_bytes + kk * B_STEP;
              return Op::B_MN ? sw128_mn_desc(at, 8192) : sw128_desc(at);
            };
#pragma unroll
            for (uint32_t kk = 0; kk < 4; kk++) {
              pair_mma<Op::KIND>(d, adesc(0, kk), bdesc(0, kk), idesc, !(first && kk == 0));
              if (PLANES == 2) {   // high by low and low by high terms; low by low is below FP32's half step
                pair_mma<Op::KIND>(d, adesc(0, kk), bdesc(1, kk), idesc, 1u);
                pair_mma<Op::KIND>(d, adesc(1, kk), bdesc(0, kk), idesc, 1u);
              }
            }
            pair_commit(empty + s);
            if (last) {
              pair_commit(tfull + acc % ACCS);
              acc++;
            }
            if (++s == stages) {
              s = 0;
              round++;
            }
          }
        }
        // the MMAs issued have ended, and the loads in flight have landed, before anything is freed
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drain))
                     : "memory");
        uint64_t t0 = globaltimer();
        while (!mbar_try_wait(drain, 0) && globaltimer() - t0 < kWaitNs) {
        }
        if (*static_cast<volatile uint32_t *>(&bounds->abort)) {
          t0 = globaltimer();
          for (uint32_t s = 0; s < stages; s++)
            for (uint32_t parity = 0; parity < 2; parity++)
              while (!mbar_try_wait(full + s, parity) && globaltimer() - t0 < kWaitNs) {
              }
        }
      }
      __syncwarp();
    } else if (Op::HELPERS) {
      Op::help(args, scratch, rank, cluster, clusters, bounds);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == kPairEpi + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// One cluster per pair of SMs, or per item where there are fewer. after: not its call's first kernel.
template <class Op>
cudaError_t launch_pair(const typename Op::Args &args, uint32_t items, int sms, cudaStream_t st, bool after) {
  const int b_bytes = (int)args.bn * 64;
  const int smem = PairShape<Op>::smem(b_bytes);
  // the attribute is a device's: set once on each
  static std::atomic<uint64_t> set{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(set.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(pair_gemm<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
    if (e != cudaSuccess) return e;
    set.fetch_or(bit, std::memory_order_relaxed);
  }
  const uint32_t clusters = items < (uint32_t)(sms / 2) ? items : (uint32_t)(sms / 2);
  return launch_chained(after, pair_gemm<Op>, 2 * clusters, kPairThreads, smem, st, args, pipeline_wait_ns());
}

}  // namespace annb200
