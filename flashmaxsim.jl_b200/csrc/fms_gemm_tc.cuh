// fms_gemm_tc.cuh -- the tcgen05 matrix-product engine of the token-encoder
// operators: C tiles of 128 rows per CTA, operands streamed by TMA through a ring
// of shared-memory stages, accumulators in TMEM (two, so that the epilogue of one
// tile runs under the products of the next), persistent CTAs.
//
// CG = 2 pairs two CTAs of a cluster on one 256 x BN tile (cta_group::2): each
// loads its own 128 rows of A and half of B's rows, so a tile step of 64 columns
// moves 64 KB for 8.4 MFLOP, 128 flop per byte read from L2 against 85 for one
// CTA's 128 x 256 tile.  CG = 1 serves problems with too few tiles for pairs.
//
// An operand is K-major (rows of 128 bytes along the sum, 128-byte swizzle) or
// MN-major (its rows run along the sum: 64-element column chunks of 64 sum rows,
// the chunks 8 KB apart), so no operand is ever transposed in memory.
//
// Warp 0 loads (one lane), warp 1 issues the MMAs (one lane of the leader CTA),
// warps 2-9 drain accumulators: the subpartition a warp may read is its id mod 4,
// so each subpartition has two warps, one for each half of the columns.  Every
// wait is bounded: it gives up after two seconds, raises the health flag and lets
// all roles leave, once the copies and products in flight have ended (bounded as well).
#pragma once
#include <cuda.h>

#include "fms_common.cuh"
#include "fms_internal.h"
#include "fms_launch.cuh"
#include "fms_tc_ptx.cuh"

namespace fms {
namespace gemm {

constexpr int MT = 128;         // accumulator rows of a CTA
constexpr int NEPI = 8;         // epilogue warps
constexpr int NTHREADS = (2 + NEPI) * 32;
constexpr int ROWB = 128;       // bytes of a stage row (one swizzle atom wide)
constexpr int SMEM_BYTES = 192 * 1024;  // ring stages
constexpr int OUT_BYTES = 4096;         // per epilogue warp: 32 rows x 64 16-bit columns on their way out

template <int BN, int CG>
struct Ring {
  static constexpr int A_BYTES = MT * ROWB;
  static constexpr int B_BYTES = BN / CG * ROWB;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = SMEM_BYTES / STAGE > 8 ? 8 : SMEM_BYTES / STAGE;
};

// ------------------------------------------------------------------ PTX of CTA pairs

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of CTA `rank`'s copy of a shared-memory variable.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(p)), "r"(rank));
  return a;
}
// Arrive on a barrier of the cluster.  Ordered after the warp's TMEM reads by the fence
// before it; release at cluster scope would wait for the epilogue's stores as well.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ptx::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait (cluster scope); false when it gave up or another role did.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    if (try_wait_cluster(bar, parity)) return true;
    if ((it & 255u) == 255u) {
      if (*abort) return false;
      const uint64_t now = ptx::globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > 2000000000ull) {
        *abort = 1;
        return false;
      }
    }
  }
}

// After a wait gave up: until the phase completes, the abort flag notwithstanding, or 10 ms.
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = ptx::globaltimer_ns();
  while (!try_wait_cluster(bar, parity) && ptx::globaltimer_ns() - t0 < 10000000ull) {
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

template <int CG, bool I8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define FMS_MMA(G, K)                                                               \
  asm volatile(                                                                     \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                             \
      "tcgen05.mma.cta_group::" G ".kind::" K " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                   \
      : "memory")
  if (CG == 2) {
    if (I8) FMS_MMA("2", "i8");
    else FMS_MMA("2", "f16");
  } else {
    if (I8) FMS_MMA("1", "i8");
    else FMS_MMA("1", "f16");
  }
#undef FMS_MMA
}

// Arrive on `bar` (in every CTA of the tile) when all MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            ptx::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    ptx::mma_commit(bar);
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(dst)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    ptx::tmem_alloc(dst, cols);
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  if (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    ptx::tmem_dealloc(addr, cols);
}

// Shared-memory descriptor of an operand tile.  K-major: 8-row atoms 1024 bytes
// apart.  MN-major: 8-sum-row atoms 1024 bytes apart, 64-element chunks 8192.
template <bool MN>
__device__ __forceinline__ uint64_t desc(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(MN ? 8192 >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version of sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

// Health flag of this file's kernels: a wait gave up.  The flag and its reader are each
// translation unit's own.
static __device__ int g_error = 0;

static inline int read_error(int reset) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_error, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int z = 0;
    e = cudaMemcpyToSymbol(g_error, &z, sizeof(int));
  }
  return e == cudaSuccess ? v : (int)e;
}

// ------------------------------------------------------------------ the work of a launch

// Which products a launch computes.
enum Op : int {
  OP_PAIR_B,    // C = A [B0 | B1]^T: one A, the halves of the tile's columns from two B
  OP_SUM,       // C = A0 B0 + A1 B1 (the sum runs over both pairs)
  OP_STACK_A,   // C = [A0 ; A1] B0: the row tiles of two A one after the other
  OP_ONE,       // C = A0 B0
};

struct Work {
  int mt, nt, splits;   // tiles along rows (pairs of CTAs count once) and columns, parts of the sum
  int mt0;              // OP_STACK_A: row tiles of A0
  int kb;               // blocks of the sum (64 16-bit or 128 8-bit elements)
  int kb0;              // OP_SUM: blocks of the first pair
  uint32_t idesc;
};

struct Tile {
  int m, n, split, k0, k1;
};

__device__ __forceinline__ Tile tile_at(const Work& w, int64_t t) {
  Tile r;
  r.n = (int)(t % w.nt);
  t /= w.nt;
  r.m = (int)(t % w.mt);
  r.split = (int)(t / w.mt);
  r.k0 = (int)((int64_t)w.kb * r.split / w.splits);
  r.k1 = (int)((int64_t)w.kb * (r.split + 1) / w.splits);
  return r;
}

// ------------------------------------------------------------------ kernel

// Epi::run(params, tile, this lane's row of the product, half, TMEM address, ahead, out,
// release) handles 32 lanes x half of the columns of an accumulator (of either half of it for
// OP_PAIR_B); Epi::fetch may load what it needs for that into `ahead` while the products
// still run; `out` is the warp's OUT_BYTES of shared memory; it calls `release` once, when
// it has read the accumulator.
template <int OP, int CG, int BN, bool A_MN, bool B_MN, bool I8, class Epi>
__global__ void __launch_bounds__(NTHREADS, 1)
kernel(const __grid_constant__ CUtensorMap tA0, const __grid_constant__ CUtensorMap tA1,
       const __grid_constant__ CUtensorMap tB0, const __grid_constant__ CUtensorMap tB1, const Work W,
       const __grid_constant__ typename Epi::Params E) {
  using R = Ring<BN, CG>;
  constexpr int KEL = I8 ? 128 : 64;                // sum elements of a stage
  constexpr int KSTEP = A_MN ? 2048 : 32;           // descriptor bytes of one MMA's sum (16 or 32 elements)
  constexpr int KSTEP_B = B_MN ? 2048 : 32;
  constexpr int ACC = BN <= 32 ? 32 : BN <= 64 ? 64 : BN <= 128 ? 128 : 256;  // TMEM columns of an accumulator
  constexpr int COLS = 2 * ACC;
  extern __shared__ __align__(1024) unsigned char dsm[];
  __shared__ __align__(8) uint64_t full[R::STAGES], empty[R::STAGES], accf[2], acce[2];
  __shared__ uint32_t tmem_s;
  __shared__ volatile int abort_s;
  unsigned char* ring =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < R::STAGES; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&accf[i], 1);
      ptx::mbar_init(&acce[i], NEPI * CG);
    }
    abort_s = 0;
    ptx::fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<CG>(&tmem_s, COLS);
  ptx::tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  ptx::tc_fence_after();
  dependency_wait();
  const uint32_t tmem = tmem_s;
  const int64_t tiles = (int64_t)W.mt * W.nt * W.splits;
  const int64_t first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    // Like the MMA warp: all lanes run the loop, an elected one issues.
    const uint32_t ring_s = __shfl_sync(0xffffffffu, ptx::smem_u32(ring), 0);
    const uint32_t full_s = __shfl_sync(0xffffffffu, CG == 2 ? cluster_addr(full, 0) : ptx::smem_u32(full), 0);
    const int rk = __shfl_sync(0xffffffffu, (int)rank, 0);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int64_t t = first; ok && t < tiles; t += stride) {
      const Tile T = tile_at(W, t);
      const bool second = OP == OP_STACK_A && T.m >= W.mt0;
      const int m0 = (((second ? T.m - W.mt0 : T.m)) * CG + rk) * MT;
      const int n0 = OP == OP_PAIR_B ? T.n * (BN / 2) : T.n * BN + rk * (BN / CG);
      for (int kb = T.k0; kb < T.k1; ++kb) {
        if (!__all_sync(0xffffffffu, wait(&empty[s], ph ^ 1, &abort_s))) {
          ok = false;
          break;
        }
        const uint32_t a = ring_s + s * R::STAGE, b = a + R::A_BYTES, bar = full_s + s * 8;
        const bool next = OP == OP_SUM && kb >= W.kb0;
        const int k = next ? kb - W.kb0 : kb;
        if (elect_one()) {
          if (rk == 0) ptx::mbar_expect_tx(&full[s], CG * R::STAGE);
          const CUtensorMap* mA = second || next ? &tA1 : &tA0;
          const CUtensorMap* mB = next || (OP == OP_PAIR_B && CG == 2 && rk == 1) ? &tB1 : &tB0;
          if (A_MN) {
#pragma unroll
            for (int c = 0; c < MT / 64; ++c) tma_load<CG>(a + c * 8192, mA, m0 + c * 64, k * 64, bar);
          } else {
            tma_load<CG>(a, mA, k * KEL, m0, bar);
          }
          if (B_MN) {
#pragma unroll
            for (int c = 0; c < BN / CG / 64; ++c) tma_load<CG>(b + c * 8192, mB, n0 + c * 64, k * 64, bar);
          } else {
            tma_load<CG>(b, mB, k * KEL, n0, bar);
            if (OP == OP_PAIR_B && CG == 1) tma_load<CG>(b + R::B_BYTES / 2, &tB1, k * KEL, n0, bar);
          }
        }
        __syncwarp();
        if (++s == R::STAGES) s = 0, ph ^= 1;
      }
    }
    // The ring is left to nobody's writes: wait (bounded) for the copies in flight.
    // In the leader every stage's barrier completes when both CTAs' copies have landed;
    // the other CTA's stages are released by the leader's commits.
    const int next = s;
    const uint32_t lap = ph;
    for (int i = 0; ok && i < R::STAGES; ++i) {
      ok = __all_sync(0xffffffffu, wait(&empty[s], ph ^ 1, &abort_s));
      if (++s == R::STAGES) s = 0, ph ^= 1;
    }
    // Where a wait gave up there may be no more commits: the leader waits for each stage's
    // last copies.  The other CTA, which cannot ask for them, stays until the leader is at
    // the cluster's last barrier.
    if (!ok && rk == 0)
      for (int i = 0; i < R::STAGES; ++i) settle(&full[i], i < next ? lap : lap ^ 1);
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA
    // The whole warp runs the loop, so that descriptors stay in uniform registers; one
    // elected lane issues.
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t ring_s = __shfl_sync(0xffffffffu, ptx::smem_u32(ring), 0);
    int s = 0, buf = 0;
    uint32_t ph = 0, bph = 0;
    bool ok = true;
    for (int64_t t = first; ok && t < tiles; t += stride) {
      const Tile T = tile_at(W, t);
      if (!__all_sync(0xffffffffu, wait(&acce[buf], bph ^ 1, &abort_s))) break;
      ptx::tc_fence_after();
      const uint32_t d = base + buf * ACC;
      for (int kb = T.k0; kb < T.k1; ++kb) {
        if (!__all_sync(0xffffffffu, wait(&full[s], ph, &abort_s))) {
          ok = false;
          break;
        }
        const uint32_t a = ring_s + s * R::STAGE, b = a + R::A_BYTES;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma<CG, I8>(d, desc<A_MN>(a + j * KSTEP), desc<B_MN>(b + j * KSTEP_B), W.idesc, kb > T.k0 || j > 0);
          commit<CG>(&empty[s]);
        }
        __syncwarp();
        if (++s == R::STAGES) s = 0, ph ^= 1;
      }
      if (elect_one()) commit<CG>(&accf[buf]);
      __syncwarp();
      if (++buf == 2) buf = 0, bph ^= 1;
    }
    // A wait gave up: the products in flight still read shared memory and write TMEM.
    if (__any_sync(0xffffffffu, abort_s != 0)) {
      if (elect_one()) commit<CG>(&accf[buf]);
      __syncwarp();
      settle(&accf[buf], bph);
    }
  } else if (warp >= 2) {
    // ------------------------------------------------------------ epilogue
    const int sub = warp & 3, half = (warp - 2) >> 2;
    unsigned char* const out = ring + R::STAGES * R::STAGE + (warp - 2) * OUT_BYTES;
    int buf = 0;
    uint32_t bph = 0;
    for (int64_t t = first; t < tiles; t += stride) {
      const Tile T = tile_at(W, t);
      const int64_t row = (int64_t)(T.m * CG + (int)rank) * MT + sub * 32 + lane;
      typename Epi::template Ahead<BN> ahead;
      Epi::template fetch<BN>(E, T, row, half, ahead);
      const bool ok = wait(&accf[buf], bph, &abort_s);
      if (!__all_sync(0xffffffffu, ok)) break;
      ptx::tc_fence_after();
      const uint32_t addr = tmem + buf * ACC + ((uint32_t)(sub * 32) << 16);
      Epi::template run<BN>(E, T, row, half, addr, ahead, out, [&]() {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) arrive_cluster(cluster_addr(&acce[buf], 0));
          else ptx::mbar_arrive(&acce[buf]);
        }
      });
      if (++buf == 2) buf = 0, bph ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // stores out of `out`
  }
  __syncwarp();
  __syncthreads();
  if (threadIdx.x == 0 && abort_s) g_error = 1;
  if (CG == 2) cluster_sync_all();
  if (warp == 1) tmem_dealloc<CG>(tmem, COLS);
}

// ------------------------------------------------------------------ epilogue pieces

// The loads so far are complete: ties the registers to the wait, so that no use of them
// is scheduled before it.
__device__ __forceinline__ void landed(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
        "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
        "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
        "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
// tcgen05.ld of 32 columns of this warp's lanes, complete on return.
__device__ __forceinline__ void load32(uint32_t addr, uint32_t (&r)[32]) {
  ptx::tmem_ld32(addr, r);
  landed(r);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// 32 consecutive 16-bit values of one row (two per register); `n` of them exist, rows
// start on 32 bytes.
template <typename T>
__device__ __forceinline__ void load_row32(const T* p, uint32_t (&v)[16], int n) {
  if (n >= 32) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(v[8 * q]), "=r"(v[8 * q + 1]), "=r"(v[8 * q + 2]), "=r"(v[8 * q + 3]), "=r"(v[8 * q + 4]),
                     "=r"(v[8 * q + 5]), "=r"(v[8 * q + 6]), "=r"(v[8 * q + 7])
                   : "l"(p + 16 * q));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
      const uint32_t lo = 2 * i < n ? h[2 * i] : 0u, hi = 2 * i + 1 < n ? h[2 * i + 1] : 0u;
      v[i] = lo | hi << 16;
    }
  }
}

// ------------------------------------------------------------------ the way out
//
// A warp's 32 rows x 128 bytes go through its `out` and leave by whole rows: by the copy
// engine where the matrix's rows start on 16 bytes, by coalesced stores elsewhere.
// (Stores by lane, each to a row of its own, held up the epilogue.)

// Values of this lane's row into `out`: 16-byte piece q of the row at q ^ (row mod 8), the
// 128-byte swizzle that the store's map names.
template <int N>
__device__ __forceinline__ void put(unsigned char* out, int lane, int first, const uint32_t (&v)[N]) {
#pragma unroll
  for (int q = 0; q < N / 4; ++q)
    *reinterpret_cast<uint4*>(out + lane * 128 + (((first + q) ^ (lane & 7)) << 4)) =
        make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// `out` is free again: its last store has been read out of it (all lanes).
__device__ __forceinline__ void out_free(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
// `out` to (col, row) of a map (all lanes; rows and columns past its end are left out).
__device__ __forceinline__ void out_store(const unsigned char* out, const CUtensorMap* map, int col, int row, int lane) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(col), "r"(row), "r"(ptx::smem_u32(out))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// `out` to the matrix at p, `ld` elements of SIZE bytes between its rows; `rows` rows and
// `cols` columns exist.
template <int SIZE>
__device__ __forceinline__ void out_rows(const unsigned char* out, void* p, int64_t ld, int rows, int cols, int lane) {
  __syncwarp();
  const bool words = SIZE == 4 || (ld % 2 == 0 && (reinterpret_cast<uintptr_t>(p) & 3) == 0);
  const int c = SIZE == 4 ? lane : 2 * lane;  // of the lane's word
  char* at = static_cast<char*>(p) + (int64_t)c * SIZE;
  const int64_t step = ld * SIZE;
  const unsigned char* mine = out + (lane & 3) * 4;
  rows = min(rows, 32);
  if (SIZE == 4 || words) {
    if (c + (SIZE == 4 ? 0 : 1) < cols) {  // a word a row
#pragma unroll 8
      for (int r = 0; r < rows; ++r, at += step)
        *reinterpret_cast<uint32_t*>(at) =
            *reinterpret_cast<const uint32_t*>(mine + r * 128 + (((lane >> 2) ^ (r & 7)) << 4));
    } else if (c < cols) {  // the last column, alone
      for (int r = 0; r < rows; ++r, at += step)
        *reinterpret_cast<uint16_t*>(at) =
            *reinterpret_cast<const uint16_t*>(mine + r * 128 + (((lane >> 2) ^ (r & 7)) << 4));
    }
  } else {
#pragma unroll 4  // (words put together from two lanes for odd rows were slower: 93 us against 73)
    for (int r = 0; r < rows; ++r, at += step) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(mine + r * 128 + (((lane >> 2) ^ (r & 7)) << 4));
      if (c < cols) *reinterpret_cast<uint16_t*>(at) = (uint16_t)w;
      if (c + 1 < cols) *reinterpret_cast<uint16_t*>(at + 2) = (uint16_t)(w >> 16);
    }
  }
  __syncwarp();
}

// ------------------------------------------------------------------ host side

inline uint32_t idesc_f16(int dtype, int M, int N, bool a_mn, bool b_mn) {
  const uint32_t f = dtype == FMS_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Which tile a product takes.  Measured per block of the sum: the 256 x 256 tile of a CTA
// pair takes the MMAs' 512 cycles, narrower tiles what their loads take at about 60
// bytes per cycle and SM; a launch adds about 2500 cycles for its first loads and last
// epilogue.  Pairs of 256 columns win where there are tiles for all SMs; few rows or
// columns take narrower tiles that use more SMs.
struct Shape {
  int cg, bn;
  double step;
};
constexpr Shape SHAPES[] = {{2, 256, 546.0}, {2, 128, 410.0}, {1, 64, 400.0}};
inline int pick_shape(int64_t rows, int64_t cols, int kb, int sms) {
  int best = 0;
  double cost = 1e300;
  for (int i = 0; i < 3; ++i) {
    const Shape& h = SHAPES[i];
    const int64_t t = ((rows + 128 * h.cg - 1) / (128 * h.cg)) * ((cols + h.bn - 1) / h.bn);
    const int64_t slots = sms / h.cg;
    const double c = (double)((t + slots - 1) / slots) * (kb * h.step + 600.0) + 2500.0;
    if (c < cost) cost = c, best = i;
  }
  return best;
}

template <int OP, int CG, int BN, bool A_MN, bool B_MN, bool I8, class Epi>
cudaError_t launch(const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0, const CUtensorMap& b1,
                   const Work& w, const typename Epi::Params& e, int sms, cudaStream_t s) {
  auto k = kernel<OP, CG, BN, A_MN, B_MN, I8, Epi>;
  constexpr int smem = Ring<BN, CG>::STAGES * Ring<BN, CG>::STAGE + NEPI * OUT_BYTES + 1024;
  cudaError_t err = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (err != cudaSuccess) return err;
  const int64_t tiles = (int64_t)w.mt * w.nt * w.splits;
  int64_t grid = sms / CG;
  if (grid > tiles) grid = tiles;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)(grid * CG));
  c.blockDim = dim3(NTHREADS);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)CG, 1, 1};
  c.attrs = at;
  c.numAttrs = CG == 2 ? 2 : 1;
  return cudaLaunchKernelEx(&c, k, a0, a1, b0, b1, w, e);
}

}  // namespace gemm
}  // namespace fms
