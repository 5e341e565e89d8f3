// Matrix products of 16-bit factors on the tensor cores, with the epilogue that
// the operator wants: the body shared by the feed-forward block and the LM head's
// loss.
//
//   C [M, N] = sum over the terms of A B^T,  A [M, k], B [N, k], fp32 sums
//
// Persistent CTAs (pairs of CTAs for tall problems) over tiles of 128 (256) rows by
// up to 256 columns.  Warp 0 feeds a ring of slices of k by TMA, one thread of warp 1
// issues `tcgen05.mma` into one of two TMEM accumulators, the other warps take the
// other through the epilogue meanwhile.
//
// What bounds it.  An SM's tensor core takes bn / 2 clocks for a 128 x bn x 16 step;
// filling and reading the step's operands takes (128 + bn) * 32 * 2 bytes through a
// port of 128 bytes a clock: 192 clocks for 128 at bn = 256.  With the rows of a
// pair (cta_group::2: 256 x 256, each CTA holding half of B) it is 128 for 128.
//
// Measured on a B200, 8,192 rows of 2,560 and 9,728 features, bf16, single launches:
// gated product 537 us (1,520 TFLOP/s), dx over k = 19,456 501 (1,630), both weights'
// gradients 528 (1,545); with the copies alone 454 and 502 us, with the MMAs alone 408
// (of 588 and 644 then).  Back to back the power limit takes a sixth off: the loss of
// 8,192 x 2,560 x 151,936 with gradients runs at 1,270 to 1,330 TFLOP/s.
//
// A factor's contiguous index may be k (128-byte rows of 64 k) or its own (64-wide
// blocks of rows of k); both come by TMA with the 128-byte swizzle, and what lies
// outside the factor is filled with zeros.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "tt_gemm.cuh"
#include "tt_sm100.cuh"
#include "tt_vec.cuh"

namespace tt {
namespace gemm {

using namespace sm100;

constexpr int kBK = 64;                    // k of a slice: 128 bytes
constexpr int kABytes = 128 * kBK * 2;     // of A in a slice
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 196608;         // of shared memory for the ring
constexpr int kEpiWarps = 8;               // two for each quarter of the lanes
constexpr int kSumWarps = 16;              // of epilogues that sum in chunks
constexpr int kChunk = 640;                // of k, a chunk

struct Problem {
  CUtensorMap a[2], b[2];
  int32_t steps[2];                        // slices of k of each term
  int32_t terms;
  int32_t M, N;
  int32_t bn;                              // columns of the accumulator
  int32_t tile_rows, tiles_m, tiles_n;
  int32_t group;                           // tiles of m that go through L2 together
  int32_t whole;                           // tiles whose sum over k is one CTA's; those
  int32_t parts, part_steps;               // behind them are summed in parts
  int32_t stages, stage_bytes;
  int32_t a_bytes;                         // of A that a CTA copies a slice
  int32_t a_blocks, b_blocks;              // whole blocks of 64: copied together
  int32_t dual;                            // B's halves are two factors: b[0] and b[1]
  int32_t* status;
};

// A slice is 64 of k wide, on pairs of CTAs 128: half the barriers, and fewer copies
// where blocks of 64 go together (8,192 x 2,560 over k = 19,456: 535 us, 509).
__host__ __device__ constexpr int blocks_of_k(int cg) { return cg; }

struct TileAt {
  int unit, begin, end, m, n;              // unit: of a sum in parts (else -1)
};

// Item i: a whole tile, or a part of one of the last ones.
__host__ __device__ __forceinline__ TileAt tile_at(const Problem& p, int i) {
  TileAt t;
  t.unit = i - p.whole;
  t.begin = 0;
  t.end = p.steps[0] + (p.terms > 1 ? p.steps[1] : 0);
  if (t.unit >= 0) {
    i = p.whole + t.unit / p.parts;
    t.begin = (t.unit % p.parts) * p.part_steps;
    t.end = t.end < t.begin + p.part_steps ? t.end : t.begin + p.part_steps;
  }
  // groups of `group` tiles of m, all n within a group, m fastest
  const int full = p.group * p.tiles_n;
  const int g = i / full, in = i - g * full;
  const int left = p.tiles_m - g * p.group, rows = left < p.group ? left : p.group;
  t.n = in / rows;
  t.m = g * p.group + in - t.n * rows;
  return t;
}

struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  int32_t abort;
};

constexpr int kStageRow = 33;              // floats of a row of a warp's 32 x 32 block
constexpr int kStageBytes = kEpiWarps * 32 * kStageRow * 4;
// barriers, ring, its alignment, the epilogue's blocks
constexpr int kGemmSmem = 1024 + kRingBytes + 1024 + kStageBytes;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// The address of CTA 0's copy of a shared-memory address of this CTA.
__device__ __forceinline__ uint32_t leader_addr(uint32_t a) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
  return r;
}

template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                       int c1) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
        "bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

// The blocks of 64 of a factor's own index that a slice has, in one copy
// (k contiguous: the slice's blocks of 64 k).
template <int CG>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c1,
                                       int c2) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
        "bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ uint64_t low_plus(uint64_t desc, uint32_t n) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"((uint32_t)desc + n), "r"((uint32_t)(desc >> 32)));
  return r;
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    mma_ss(d, a, b, idesc, accumulate);
}

// Arrives on `bar` of every CTA of the pair once the MMAs so far are done.
template <int CG>
__device__ __forceinline__ void commit_all(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc_commit(bar);
}

template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t* slot) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n\t"
                 "tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::"r"(smem_u32(slot))
                 : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n\t"
                 "tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::"r"(smem_u32(slot))
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_give(uint32_t taddr) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}

// Epi::tile(args, problem, tile, row, lane address, c0, block) takes one accumulator out
// of TMEM: a thread has one row of the tile (row: its index in C, possibly past M) and
// reads its columns c0 .. c0 + 31, c0 + 64 .. (c0: 0 or 32, another warp has the other
// half); all 32 lanes of a warp call it.  block: 32 x 33 floats of shared memory of the
// warp's own.
//
// An epilogue that sums in chunks (Epi::kChunks) adds up the accumulators of kChunk of k
// each in registers instead: the tensor cores cut off what falls below an accumulator's
// last bit at every 16 of k, always towards zero, and a logit over k = 2,560 comes out
// 5e-7 of itself too small (loss off by 1.4e-6 of itself, 3.5e-7 in chunks).  Sixteen
// warps have a row and 64 columns a thread: Epi::finish(args, problem, tile, row, c0,
// values).
template <typename Epi>
constexpr int warps_of() { return Epi::kChunks ? kSumWarps : kEpiWarps; }
template <typename Epi>
constexpr int threads_of() { return 64 + 32 * warps_of<Epi>(); }

template <int CG, bool kAMN, bool kBMN, typename Epi>
__global__ void __launch_bounds__(threads_of<Epi>(), 1)
    gemm_kernel(const __grid_constant__ Problem p, const __grid_constant__ typename Epi::Args ea) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  constexpr int kKb = blocks_of_k(CG);
  Barriers* sh = reinterpret_cast<Barriers*>(smem_raw);
  const uint32_t ring = (smem_u32(smem_raw) + 1024 + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const volatile int32_t* abort_flag = &sh->abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) mbar_init(&sh->full[s], 1), mbar_init(&sh->empty[s], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->acc_full[b], 1);
      mbar_init(&sh->acc_empty[b], warps_of<Epi>() * CG);
    }
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_take<CG>(&sh->tmem);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_barrier();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const int items = p.whole + (p.tiles_m * p.tiles_n - p.whole) * p.parts;
  const int first = blockIdx.x / CG, stride = gridDim.x / CG;
  auto fail = [&]() {
    sh->abort = 1;
    set_status(p.status, TT_ERR_DEVICE_TIMEOUT);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA
    if (lane == 0) {
      const int stages = p.stages;
      const uint32_t b_bytes = (uint32_t)(p.bn / CG) * 128;
      const uint32_t tx = (uint32_t)(p.a_bytes + b_bytes) * CG * kKb;
      const uint32_t full0 = smem_u32(&sh->full[0]);
      const uint32_t bar0 = CG == 2 ? leader_addr(full0) : full0;
      int s = 0;
      uint32_t phase = 0;                  // of the ring's current turn
      int64_t slot = 0;
      bool ok = true;
      for (int i = first; i < items && ok; i += stride) {
        const TileAt t = tile_at(p, i);
        const int m0 = t.m * 128 * CG + (int)rank * 128;
        for (int k = t.begin; k < t.end; ++k, ++slot) {
          if (slot >= stages && !mbar_wait(&sh->empty[s], phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const int term = k >= p.steps[0] && p.terms > 1;
          const int k0 = (k - (term ? p.steps[0] : 0)) * kBK * kKb;
          const uint32_t sa = ring + s * p.stage_bytes, sb = sa + kABytes * kKb;
          const uint32_t bar = bar0 + 8 * s;
          if (rank == 0) mbar_arrive_expect_tx(&sh->full[s], tx);
          // (blocks that cannot be copied together: one after another)
          if (p.a_blocks) {
            tma_3d<CG>(sa, &p.a[term], bar, kAMN ? k0 : m0, (kAMN ? m0 : k0) / 64);
          } else if constexpr (kAMN) {
            for (int c = 0; c < 2; ++c)
              tma_2d<CG>(sa + c * 8192 * kKb, &p.a[term], bar, m0 + 64 * c, k0);
          } else {
            for (int c = 0; c < kKb; ++c)
              tma_2d<CG>(sa + c * kABytes, &p.a[term], bar, k0 + 64 * c, m0);
          }
          const int n0 = p.dual ? t.n * (p.bn / 2) : t.n * p.bn + (int)rank * (p.bn / CG);
          const int b_rows = p.bn / CG;
          if (CG == 1 && p.dual) {
            tma_2d<CG>(sb, &p.b[0], bar, k0, n0);
            tma_2d<CG>(sb + b_rows / 2 * 128, &p.b[1], bar, k0, n0);
          } else {
            const CUtensorMap* map = &p.b[p.dual ? rank : term];
            if (p.b_blocks) {
              tma_3d<CG>(sb, map, bar, kBMN ? k0 : n0, (kBMN ? n0 : k0) / 64);
            } else if constexpr (kBMN) {
              for (int c = 0; c < b_rows; c += 64)
                tma_2d<CG>(sb + c * 128 * kKb, map, bar, n0 + c, k0);
            } else {
              for (int c = 0; c < kKb; ++c)
                tma_2d<CG>(sb + c * b_rows * 128, map, bar, k0 + 64 * c, n0);
            }
          }
          if (++s == stages) s = 0, phase ^= 1;
        }
      }
      if (ok) {
        // the last slices' releases have arrived before this CTA may end
        for (int64_t i = max((int64_t)0, slot - stages); i < slot && ok; ++i)
          ok = mbar_wait(&sh->empty[i % stages], (uint32_t)(i / stages) & 1, abort_flag);
      }
      if (!ok) {
        fail();
        // the copies under way land before the CTA ends (the pair's signal here)
        if (rank == 0)
          for (int64_t i = max((int64_t)0, slot - stages); i < slot; ++i)
            mbar_wait(&sh->full[i % stages], (uint32_t)(i / stages) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_f16_ab(Epi::kBf16, 128 * CG, p.bn, kAMN, kBMN);
      const int stages = p.stages;
      // 64-wide blocks of rows of k: 8 KB (kKb times) from block to block, 2 KB a step of
      // 16 k; rows of 64 k: 32 bytes a step, kKb times all rows
      const uint32_t rb = ring + kABytes * kKb;
      const uint64_t da0 = kAMN ? desc_sw128(ring, 8192 * kKb, 1024) : desc_sw128(ring, 16, 1024);
      const uint64_t db0 = kBMN ? desc_sw128(rb, 8192 * kKb, 1024) : desc_sw128(rb, 16, 1024);
      constexpr uint32_t kStepA = (kAMN ? 2048 : 32) >> 4, kStepB = (kBMN ? 2048 : 32) >> 4;
      constexpr uint32_t sub_a = (kAMN ? 8192 : kABytes) >> 4;
      const uint32_t sub_b = (uint32_t)(kBMN ? 8192 : p.bn / CG * 128) >> 4;
      int s = 0, acc = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int chunk = kChunk / (kBK * kKb);
      for (int i = first; i < items && ok; i += stride) {
        const TileAt t = tile_at(p, i);
        for (int from = t.begin, to; from < t.end && ok; from = to, ++acc) {
          to = Epi::kChunks ? min(t.end, from + chunk) : t.end;
          const int buf = acc & 1;
          if (acc >= 2 && !mbar_wait(&sh->acc_empty[buf], ((acc >> 1) - 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + buf * 256;
          for (int k = from; k < to; ++k) {
            if (!mbar_wait(&sh->full[s], phase, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            // (a descriptor's address is in its low word)
            const uint32_t off = (uint32_t)(s * p.stage_bytes) >> 4;
#pragma unroll
            for (int sub = 0; sub < kKb; ++sub)
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk)
                mma_f16<CG>(d, low_plus(da0, off + sub * sub_a + kk * kStepA),
                            low_plus(db0, off + sub * sub_b + kk * kStepB), idesc,
                            sub > 0 || kk > 0 ? 1u : (uint32_t)(k > from));
            commit_all<CG>(&sh->empty[s]);
            if (++s == stages) s = 0, phase ^= 1;
          }
          if (ok) commit_all<CG>(&sh->acc_full[buf]);
        }
      }
      if (!ok) fail();
      // every MMA issued is done before the accumulators are given back
      if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                smem_u32(&sh->drain))
            : "memory");
      else
        tc_commit(&sh->drain);
      mbar_wait(&sh->drain, 0, nullptr);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
    int acc = 0;
    // the accumulator's turn: true once it is there, and back to the MMAs
    auto take = [&]() {
      const bool ok = mbar_wait(&sh->acc_full[acc & 1], (acc >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        fail();
        return false;
      }
      tc_fence_after();
      return true;
    };
    auto give = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                           leader_addr(smem_u32(&sh->acc_empty[acc & 1])))
                       : "memory");
        else
          mbar_arrive(&sh->acc_empty[acc & 1]);
      }
      ++acc;
    };
    bool ok = true;
    for (int i = first; i < items && ok; i += stride) {
      const TileAt t = tile_at(p, i);
      const int row = t.m * 128 * CG + (int)rank * 128 + quad * 32 + lane;
      if constexpr (Epi::kChunks) {
        const int c0 = (warp - 2) / 4 * 64, chunk = kChunk / (kBK * kKb);
        float v[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] = 0.f;
#pragma unroll 1
        for (int k = t.begin; k < t.end; k += chunk) {
          if (!(ok = take())) break;
#pragma unroll
          for (int h = 0; h < 64; h += 16) {       // (as many as registers are left for)
            float x[16];
            tmem_ld16(lane_addr + (acc & 1) * 256 + c0 + h, x);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h + j] += x[j];
          }
          give();
        }
        if (ok) Epi::finish(ea, p, t, row, c0, v);
      } else {
        float* block =
            reinterpret_cast<float*>(smem_raw + 2048 + kRingBytes) + (warp - 2) * 32 * kStageRow;
        if (!(ok = take())) break;
        Epi::tile(ea, p, t, row, lane_addr + (acc & 1) * 256, warp < 6 ? 0 : 32, block);
        give();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_barrier();
  tc_fence_after();
  if (warp == 1) tmem_give<CG>(tmem);
}

// ---- host -----------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encoder() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// What TMA asks of a factor.
inline bool copyable(const Factor& f) {
  return (reinterpret_cast<uintptr_t>(f.p) & 15) == 0 && f.ld % 8 == 0;
}

// The map of a factor of `n` rows and k columns: boxes of 64 k by `rows`, or (blocks) kb
// of these in one box; where the rows are contiguous, of 64 rows by kb * 64 k, or
// (blocks) `rows` / 64 of these.  Only whole blocks can be copied together: what
// lies outside is told by the first index otherwise.
inline bool encode(CUtensorMap* m, bool bf16, const Factor& f, int64_t n, int64_t k, int rows,
                   bool blocks, int kb) {
  const EncodeTiledFn fn = encoder();
  if (!fn || !copyable(f)) return false;
  if (blocks) {
    const cuuint64_t dims[3] = {64u, (cuuint64_t)(f.mn ? k : n), (cuuint64_t)((f.mn ? n : k) / 64)};
    const cuuint64_t strides[2] = {(cuuint64_t)f.ld * 2, 128u};
    const cuuint32_t box[3] = {64u, (cuuint32_t)(f.mn ? 64 * kb : rows),
                               (cuuint32_t)(f.mn ? rows / 64 : kb)};
    const cuuint32_t estr[3] = {1u, 1u, 1u};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(f.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)(f.mn ? n : k), (cuuint64_t)(f.mn ? k : n)};
  const cuuint64_t strides[1] = {(cuuint64_t)f.ld * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)(f.mn ? 64 * kb : rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
            const_cast<void*>(f.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product is cut up: columns of the accumulator, tiles that are summed whole,
// and the parts of the sums of the others.
struct Plan {
  int cg, bn;
  int64_t whole;
  int parts;
  int64_t work;                            // bytes of the parts
};

// Clocks of a slice of 64 k in a tile: the tensor core's, or the shared-memory
// port's where that is more (see the top).
inline int64_t slice_clocks(int cg, int bn) {
  return cg == 1 ? 256 + 2 * bn : std::max(256 + bn, 2 * bn);
}

// Clocks of a tile's epilogue, which sums shorter than it cannot hide: a pair's has as
// many rows a CTA, and waits for the other CTA (both weights' gradients of 2,560 x 9,728
// over 64 tokens: 39 us by pairs, 29 by single CTAs; over 512: 52 and 48).  The gated
// product's is longer than that wait (8,192 x 256 x 1,024: 31 us by pairs, 39).
inline int64_t epilogue_clocks(int cg, int bn, bool dual) {
  // (a warp has 32 columns of every 64: a few of 64 take as long as all)
  const int blocks = ((dual ? bn / 2 : bn) + 63) / 64;
  return dual ? 4000 * blocks : (cg == 1 ? 1250 : 2000) * blocks;
}

// The cheapest of the forms by the tiles' waves.  `n_step`: what widths of the
// accumulator are a multiple of; `dual`: its halves stand for one column of C each.
// With `split` the tiles of the last wave, where they leave half of the SMs idle, are
// summed in parts (8,192 x 2,560 over k = 19,456: 320 tiles on 74 pairs of SMs, 5 waves
// or 4 and a third).
inline Plan plan_product(int64_t M, int64_t N, int64_t steps, int n_step, bool dual, bool split) {
  Plan best{};
  double least = 1e300;
  for (int cg = 1; cg <= 2; ++cg) {
    const int step = std::max(n_step, 16) * cg;
    const int64_t slots = vec::kSMs / cg;
    for (int bn = 256; bn >= step; bn -= step) {
      const int64_t cols = dual ? bn / 2 : bn;
      const int64_t tiles = ((M + 128 * cg - 1) / (128 * cg)) * ((N + cols - 1) / cols);
      const int64_t rest = tiles % slots;
      const int64_t most = rest && split ? std::min(slots / rest, steps / 8) : 1;
      const double clocks = (double)slice_clocks(cg, bn);
      const double end = (double)epilogue_clocks(cg, bn, dual);
      auto tile = [&](int64_t n) { return std::max((double)n * clocks, end) + 600; };
      for (int64_t parts = 1; parts <= std::max<int64_t>(1, most);
           parts = next_parts(parts, most)) {
        // (a tile's start and end, which nothing hides: 600 clocks; the parts' way
        // through L2 and the launch that adds them up)
        const int64_t whole = parts > 1 ? tiles - rest : tiles;
        double t = (double)((whole + slots - 1) / slots) * tile(steps) + 1500;
        const int64_t unit = (int64_t)128 * cg * bn * 4;
        if (parts > 1)
          t += tile((steps + parts - 1) / parts) + 5000 +
               (double)(rest * (parts + 1) * unit) / 3000;
        if (t < least * 0.999 || (parts == 1 && cg > best.cg && t <= least))
          least = t, best = Plan{cg, bn, whole, (int)parts, parts > 1 ? rest * parts * unit : 0};
      }
    }
  }
  return best;
}

// Fills the problem (maps, tiles, ring) for up to two terms; false where a factor
// cannot be copied by TMA.
inline bool set_up(Problem* q, const Plan& plan, bool bf16, int64_t M, int64_t N, const Term* terms,
                   int n_terms, bool dual, int32_t* status) {
  const int cg = plan.cg, bn = plan.bn;
  const int a_rows =
      cg == 1 && !terms[0].a.mn ? (int)std::min<int64_t>(128, (M + 7) / 8 * 8) : 128;
  const int b_rows = dual ? bn / 2 : bn / cg;
  q->terms = dual ? 1 : n_terms;
  int64_t steps = 0;
  const bool amn = terms[0].a.mn, bmn = terms[0].b.mn;
  bool k64 = true;                          // whole blocks of 64 k
  for (int i = 0; i < n_terms; ++i) k64 &= terms[i].k % 64 == 0;
  q->a_blocks = amn ? M % 64 == 0 : k64 && cg == 2;
  q->b_blocks = bmn ? N % 64 == 0 : k64 && cg == 2;
  const int kb = blocks_of_k(cg);
  for (int i = 0; i < 2; ++i) {
    const Term& t = terms[i < n_terms ? i : 0];
    if (!encode(&q->a[i], bf16, t.a, M, t.k, a_rows, q->a_blocks, kb) ||
        !encode(&q->b[i], bf16, t.b, N, t.k, b_rows, q->b_blocks, kb))
      return false;
    q->steps[i] = (int32_t)((t.k + kBK * kb - 1) / (kBK * kb));
    if (i < q->terms) steps += q->steps[i];
  }
  q->M = (int32_t)M, q->N = (int32_t)N, q->bn = bn, q->dual = dual;
  const int64_t cols = dual ? bn / 2 : bn;
  q->tile_rows = 128 * cg;
  q->tiles_m = (int32_t)((M + 128 * cg - 1) / (128 * cg));
  q->tiles_n = (int32_t)((N + cols - 1) / cols);
  // (a wave's tiles about as many of m as of n)
  q->group = std::min(q->tiles_m, cg == 2 ? 8 : 12);
  q->whole = (int32_t)plan.whole;
  q->part_steps = (int32_t)((steps + plan.parts - 1) / plan.parts);
  q->parts = (int32_t)((steps + q->part_steps - 1) / q->part_steps);
  q->stage_bytes = (kABytes + bn / cg * 128) * kb;
  q->stages = std::min(kMaxStages, kRingBytes / q->stage_bytes);
  q->a_bytes = terms[0].a.mn ? kABytes : a_rows * 128;
  q->status = status;
  return (int64_t)q->tiles_m * q->tiles_n < ((int64_t)1 << 30);
}

template <int CG, bool kAMN, bool kBMN, typename Epi>
int launch(const Problem& q, const typename Epi::Args& ea, cudaStream_t st) {
  auto* kernel = gemm_kernel<CG, kAMN, kBMN, Epi>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem) !=
      cudaSuccess)
    return TT_ERR_CUDA;
  const int64_t items = q.whole + ((int64_t)q.tiles_m * q.tiles_n - q.whole) * q.parts;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)(std::min<int64_t>(items, vec::kSMs / CG) * CG));
  c.blockDim = dim3(threads_of<Epi>());
  c.dynamicSmemBytes = kGemmSmem;
  c.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {CG, 1, 1};
  c.attrs = attr;
  c.numAttrs = CG == 2 ? 1 : 0;
  if (cudaLaunchKernelEx(&c, kernel, q, ea) != cudaSuccess) return TT_ERR_CUDA;
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

template <bool kAMN, bool kBMN, typename Epi>
int launch(const Plan& plan, const Problem& q, const typename Epi::Args& ea, cudaStream_t st) {
  return plan.cg == 2 ? launch<2, kAMN, kBMN, Epi>(q, ea, st)
                      : launch<1, kAMN, kBMN, Epi>(q, ea, st);
}

// 32 bytes, on their boundary.
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x),
               "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// A 32 x 32 block of C: each lane 32 values of a row of its own at `p` (null: none), of
// which `left` are in C.  Where rows are on 16-byte boundaries (wide) a lane stores its
// own, of a narrower block as many packs as are whole; else the warp stores row after row
// out of shared memory, 32 elements next to one another (elements of 32 rows at a time
// cost an odd width three times the rest).
template <typename T>
__device__ __forceinline__ void store_block(T* p, const float (&v)[32], int left, bool wide,
                                            float* block) {
  constexpr int V = 16 / (int)sizeof(T);
  if (wide && left >= 32) {
    if (!p) return;
    // (whole sectors of 32 bytes where rows allow: two stores of 16 would each go to L2)
    const bool sectors = (reinterpret_cast<uintptr_t>(p) & 31) == 0;
#pragma unroll
    for (int i = 0; i < 32; i += 2 * V) {
      float w[2][V];
#pragma unroll
      for (int j = 0; j < V; ++j) w[0][j] = v[i + j], w[1][j] = v[i + V + j];
      const uint4 a = vec::pack<T, V>(w[0]), b = vec::pack<T, V>(w[1]);
      if (sectors) {
        store32(p + i, a, b);
      } else {
        *reinterpret_cast<uint4*>(p + i) = a;
        *reinterpret_cast<uint4*>(p + i + V) = b;
      }
    }
    return;
  }
  if (wide) {
    if (!p) return;
#pragma unroll
    for (int i = 0; i < 32; i += V) {
      if (i + V <= left) {
        float w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = v[i + j];
        vec::store<T, V>(p + i, w);
      } else if (i < left) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (i + j < left) p[i + j] = from_f32<T>(v[i + j]);
      }
    }
    return;
  }
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 32; ++i) block[lane * kStageRow + i] = v[i];
  __syncwarp();
#pragma unroll 4
  for (int r = 0; r < 32; ++r) {
    T* row = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(p), r));
    if (row && lane < left) row[lane] = from_f32<T>(block[r * kStageRow + lane]);
  }
  __syncwarp();
}

// A product of 16-bit factors into C (tensor cores).  `work` as in fp32_product;
// steps: slices of 64 of k, of all terms.
int tc_product(bool bf16, int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r,
               void* work, int64_t work_bytes, int32_t* status, cudaStream_t st);
int64_t tc_work(int64_t M, int64_t N, int64_t steps, bool b_mn);

}  // namespace gemm
}  // namespace tt
