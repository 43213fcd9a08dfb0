// The product of two matrices in 8 bits (q8.h) on the 5th-generation tensor
// cores,
//
//   C[m, n] = act(xs[m] ws[n] sum_k X[m, k] W[n, k] + bias[n]) + residual[m, n],
//
// with X and W in e4m3 and the sum in fp32 in tensor memory.  A scale belongs to
// a whole row, so it leaves the sum and is one product per output: the weight's
// first, which is the one of moderate size (a row of x may hold numbers up to bf16's
// largest, and its scale times a sum may pass fp32's range where the result does
// not; for weights from 1e-29 to 1e29 the sum times their scale does not).  A 128-byte
// swizzled row of an operand tile holds 128 values, and one tcgen05.mma of
// kind::f8f6f4 takes 32 of them: the same bytes per instruction as in bf16, twice
// the products.
//
// * q8_split_kernel -- few rows.  The weight tile is the M = 128 side, the rows
//   (up to 128) are the N side, and K is split over the CTAs of a cluster, whose
//   fp32 partials meet in distributed shared memory.  Bound by reading W: 16 rows,
//   3584 -> 37888 with SwiGLU, 22.4 us in a graph, 6.1 TB/s of its 137 MB.
// * q8_pair_kernel -- many rows.  Pairs of CTAs (cta_group::2) on tiles of 256 rows
//   x 64, 128 or 256 features, persistent, two accumulators in tensor memory, so
//   that the epilogue of a tile runs beside the main loop of the next.  Bound by the
//   tensor pipe and the power cap: 2048 rows, 3584 -> 37888 with SwiGLU, 176 us
//   alone (3.1 PFLOP/s, tensor pipe 89 % active at 1.49 GHz), 222 back to back.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"
#include "q8.h"

namespace ll {
namespace q8 {

constexpr int BK = 128;  // values (bytes) of a k-block: one swizzled row

__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// A store of 16 bytes that the barrier `bar`, of the same CTA as `addr`, counts as they arrive.
__device__ __forceinline__ void st_async(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)),
               "r"(__float_as_uint(v.w)), "r"(bar)
               : "memory");
}
// Says that this CTA's stores are issued; orders nothing.
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_barrier_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// For lanes that may have parted: behind loads that some of them skip, a
// __syncwarp() for the wait above costs 61 rows, 8192 -> 5120 11.63 us for 11.50.
__device__ __forceinline__ void cluster_lanes_barrier_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_barrier_wait();
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One thread of a converged warp.  The main loops are one thread's, and what counts
// beside a k-block's products (512 cycles for 256 x 256) are that thread's own
// instructions.  The copies and MMAs take their operands from uniform registers:
// behind `elect.sync`, in a warp whose number and accumulator address come from a
// shuffle, the compiler keeps them there; behind `lane == 0` it moved each operand
// over for every instruction, 80 cycles an MMA at least (39 now) and 510 to 545
// cycles a k-block of any size.  For the same reason the loops are unrolled over
// the stages, with shared addresses known up to a constant, and a wait's slow path
// is out of line.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(p));
  return p != 0;
}
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int* err, int code) {
  return mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity, err, code);
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int* err, int code) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0 || wait_long(bar, parity, err, code);
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load(uint32_t dst, const void* tmap, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator, both operands e4m3
// (format 0) and K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Arrives on the barrier at this offset in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          bar),
      "h"((uint16_t)0x3)
      : "memory");
}
__device__ __forceinline__ void commit_pair_local(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void load_pair(uint32_t dst, const void* tmap, uint32_t leader_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(leader_bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void store_box(const void* tmap, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// Brings a box into L2.  Unlike a load into shared memory it may run ahead of the
// wait for the kernels before: L2 is where their writes are seen, so a box that
// one of them still writes is not held stale.
__device__ __forceinline__ void prefetch_box(const void* tmap, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tmap), "r"(x), "r"(y)
               : "memory");
}

// The approximate quotient is off by 2 ulp, and 0 for a divisor past 2^126, where x
// is below -87 and silu(x) below 1e-36.
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }
// Lets what is in flight land (copies, products, other CTAs' stores) before a CTA of
// which a wait ran out exits.  Such a CTA stores no result that is not whole: what it
// would have written stays as it was, and the error word says so.
__device__ __forceinline__ void linger() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 2000000ull) {
  }
}

struct alignas(64) Maps {
  CUtensorMap w, x, c, r;
};

// ---------------------------------------------------------------------------
// Few rows: D[128 features, BNX rows] = W_tile . X_tile^T over a CTA's share of
// the k-blocks.  Bound by reading W: every CTA's first ring of weights is on its
// way to L2 before the wait for the kernel ahead.  grid (cluster, feature tiles, row tiles).
//
// Each CTA of a cluster sums and stores a share of the groups of four rows.  The others
// send it their partials of them as they read them from tensor memory, 16 bytes (four
// rows of a feature) a thread, by stores that its barrier counts: no barrier of the
// cluster is waited for until everything is stored.  (Four bytes a store and one
// cluster barrier behind them, us: 1 row, 3584 -> 3584, 4.4 for 4.0; 32 rows 5.6 for 4.6; 61
// rows, 8192 -> 5120, 11.8 for 11.0; counted stores of four bytes 3.9, 5.5 and 13.0.
// Before that, partials that stay where they are, read behind one barrier: 16 rows, 18944 ->
// 3584, 14.2 for 13.6; bulk copies between shared memories 13.9.)  They have memory of
// their own beside the ring, since the others may be done first; a lone CTA's take the ring.
//
// The epilogue's code is met cold by every CTA, so its loop is not unrolled (twice: 61 rows,
// 8192 -> 5120, 11.2 us for 11.0); the warps that wait for the product fetch scales and bias,
// and the two that feed it, which come late, do nothing before the sums (1 row, 512 ->
// 1024, 2.3 us for 2.9).  It costs a lone CTA of many rows up to 4 % more than one
// row a thread did (61 rows, 3584 -> 37888, 25.9 for 25.2) and is up to a fifth faster in
// clusters.
//
// DEEP: one CTA a SM with a ring of 220 KB for two with 108 KB each.  Half as many
// CTAs hold as many bytes on their way and read X half as often, and that is a third
// of the reads of 64 rows.  61 rows, 18944 -> 3584: 15.4 us for 16.5 with two a SM;
// 3584 -> 3584: 6.4 for 7.6 (now 14.4 and 5.2).  128 rows: 18944 -> 3584 in clusters of
// four 19.8 us, for 28.1 in pairs of CTAs on tiles of 64 features.
constexpr int SPLIT_MAX_CLUSTER = 8;
constexpr int SPLIT_DEEP = 10;  // added to a cluster's size: the deep ring
template <int BNX, bool DEEP>
struct SplitCfg {
  static constexpr int W_BYTES = 128 * BK;
  static constexpr int X_BYTES = BNX * BK;
  static constexpr int MAX_CLUSTER = DEEP || BNX < 64 ? SPLIT_MAX_CLUSTER : (BNX == 64 ? 3 : 1);
  // partials: for each CTA of the cluster its share of the groups of four rows, 128 features each
  static constexpr int recv_groups() {
    int most = 0;
    for (int cs = 2; cs <= MAX_CLUSTER; ++cs) {
      const int n = cs * ((BNX + 4 * cs - 1) / (4 * cs));
      most = n > most ? n : most;
    }
    return most;
  }
  static constexpr int GROUP_BYTES = 4 * 128 * 4;
  static constexpr int RECV_BYTES = recv_groups() * GROUP_BYTES;
  static constexpr int STAGES = ((DEEP ? 220 : 108) * 1024 - RECV_BYTES) / (W_BYTES + X_BYTES);
  static constexpr int TMEM_COLS = BNX < 32 ? 32 : BNX;
  static constexpr int SMEM = STAGES * (W_BYTES + X_BYTES) + RECV_BYTES + 1024;
  static_assert(BNX / 4 * GROUP_BYTES <= STAGES * (W_BYTES + X_BYTES), "a lone CTA's sums overlay the ring");
};

template <int BNX, bool SWIGLU, bool DEEP>
__global__ void __launch_bounds__(192, DEEP ? 1 : 2)
    q8_split_kernel(const __grid_constant__ Maps tm, const __grid_constant__ LLQ8Gemm p, int* err) {
  using Cfg = SplitCfg<BNX, DEEP>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + STAGES * Cfg::W_BYTES;
  __shared__ uint64_t full[STAGES], empty[STAGES], tfull, rfull;  // rfull: the other CTAs' partials
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float sxs[BNX];
  __shared__ float2 scol[128];  // scale and bias of a feature

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int cs = gridDim.x, crank = blockIdx.x, nb = blockIdx.y;
  const int num_kb = (p.K + BK - 1) / BK, per = (num_kb + cs - 1) / cs;
  const int kb0 = min(num_kb, crank * per), kb1 = min(num_kb, kb0 + per);
  const int m0 = blockIdx.z * BNX, rows = min(BNX, p.M - m0);
  // groups of four rows: all of them, a CTA's share, this CTA's first one and number
  const int groups = (rows + 3) / 4, share = (groups + cs - 1) / cs;
  const int first = min(groups, crank * share), mine = min(groups - first, share);
  // partials [cs][share][128 features][4 rows]; a lone CTA's lie over the ring, once the product is done
  float4* part = reinterpret_cast<float4*>(cs > 1 ? smem + STAGES * (Cfg::W_BYTES + Cfg::X_BYTES) : smem);
  pdl_trigger();

  if (tid <= 2 * STAGES) {
    mbar_init(tid == 2 * STAGES ? &tfull : (tid < STAGES ? &full[tid] : &empty[tid - STAGES]), 1);
    fence_mbar_init();
  } else if (tid == 2 * STAGES + 1) {
    mbar_init(&rfull, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&rfull, Cfg::GROUP_BYTES * mine * (cs - 1));
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(&tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  if (cs > 1) cluster_arrive();  // this CTA runs: the others may write into its shared memory

  const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), w0 = smem_u32(sW), x0 = smem_u32(sX);
  bool done = true;  // no wait of this thread ran out
  if (warp == 0) {
    if (elect_one()) {
      // every input may be an output of the kernel ahead
      for (int kb = kb0; kb < min(kb1, kb0 + STAGES); ++kb) prefetch_box(&tm.w, kb * BK, nb * 128);
      pdl_wait();
      bool ok = true;
      uint32_t phase = 1;
      for (int kb = kb0; kb < kb1 && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
          if (kb >= kb1) break;
          if (!wait(empty0 + 8 * s, phase, err, kErrSmemEmptyTimeout)) {
            ok = false;
            break;
          }
          expect(full0 + 8 * s, Cfg::W_BYTES + Cfg::X_BYTES);
          load(w0 + s * Cfg::W_BYTES, &tm.w, full0 + 8 * s, kb * BK, nb * 128);
          load(x0 + s * Cfg::X_BYTES, &tm.x, full0 + 8 * s, kb * BK, m0);
          ++kb;
        }
      }
      done = ok;
    }
  } else if (warp == 1) {
    if (elect_one()) {
      pdl_wait();  // a wait's limit is for the copies, not for the kernel ahead
      constexpr uint32_t idesc = idesc_e4m3(128, BNX);
      const uint64_t wd = umma_desc_sw128_kmajor(w0), xd = umma_desc_sw128_kmajor(x0);
      bool ok = true;
      uint32_t phase = 0, accumulate = 0;
      for (int kb = kb0; kb < kb1 && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
          if (kb >= kb1) break;
          if (!wait(full0 + 8 * s, phase, err, kErrTmaFullTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma(tmem, wd + (s * Cfg::W_BYTES >> 4) + 2 * k, xd + (s * Cfg::X_BYTES >> 4) + 2 * k, idesc,
                k == 0 ? accumulate : 1u);
          commit(empty0 + 8 * s);
          accumulate = 1;
          ++kb;
        }
      }
      if (ok) umma_commit(&tfull);  // else the sums are not whole: those who wait for them give up too
      done = ok;
    }
  }
  __syncwarp();
  pdl_wait();  // the scales and the residual are the previous kernel's; C may still be read by it
  // A warp's turn is four rows of 32 features, a feature a lane; two lanes then trade,
  // so that each has two rows of two features (with SwiGLU of a gate and its up, 16 further
  // on).  What the epilogue reads is fetched while the product runs, by the warps that
  // have nothing else to do, which also have the first turns.
  const int turns = mine * 4, turn0 = (warp + 4) % 6;  // of the CTA; this warp's first one
  const bool high = SWIGLU ? lane >= 16 : lane & 1;     // has the last two rows
  // of a turn: this lane's first row and column of C
  auto row_of = [&](int turn) { return (first + (turn >> 2)) * 4 + (high ? 2 : 0); };
  auto col_of = [&](int turn) {
    return SWIGLU ? nb * 64 + (turn & 3) * 16 + (lane & 15) : nb * 128 + (turn & 3) * 32 + (lane & ~1);
  };
  const int cols = SWIGLU ? p.N / 2 : p.N;
  auto residual_at = [&](int turn, int i) -> uint32_t {
    const int row = row_of(turn) + i, col = col_of(turn);
    if (turn >= turns || row >= rows || col >= cols) return 0;
    const __nv_bfloat16* at = p.residual + (m0 + row) * p.ldr + col;
    return SWIGLU ? *reinterpret_cast<const uint16_t*>(at) : *reinterpret_cast<const uint32_t*>(at);
  };
  constexpr int AHEAD = BNX / 16;  // turns (one for 61 rows, 8192 -> 5120: 13.6 us; four 12.4)
  uint32_t next[AHEAD][2] = {};
  if (p.residual != nullptr) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      next[i][0] = residual_at(turn0 + 6 * i, 0);
      next[i][1] = residual_at(turn0 + 6 * i, 1);
    }
  }
  if (warp >= 2) {
    const int i = tid - 64, n = nb * 128 + i;
    if (i < BNX) sxs[i] = i < rows ? p.xs[m0 + i] : 0.f;
    const float bias = p.bias != nullptr && n < p.N ? __bfloat162float(p.bias[n]) : 0.f;
    scol[i] = make_float2(n < p.N ? p.ws[n] : 0.f, bias);
    // lanes leave a wait one by one; the loads below take a whole warp
    done = __all_sync(0xffffffffu, mbar_wait(&tfull, 0, err, kErrTmemFullTimeout));
    tc_fence_after();
  }
  if (cs > 1) cluster_lanes_barrier_wait();
  if (warp >= 2 && done) {  // TMEM lane quarter of this warp: features; columns: rows
    const int feat = (warp & 3) * 32 + lane;
    const bool none = kb1 <= kb0;
    float4* slot = part + crank * share * 128 + feat;  // of this CTA, in every CTA
    const uint32_t slot_addr = smem_u32(slot), bar_addr = smem_u32(&rfull);
    int owner = 0, left = share;  // groups that are still the owner's
    uint32_t to = mapa(slot_addr, 0), bar = mapa(bar_addr, 0);
#pragma unroll 1
    for (int c = 0; c < BNX && c < rows; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tmem + (uint32_t((warp & 3) * 32) << 16) + c, r);  // BNX 16: columns 16.. unused
      tmem_ld_wait();
      constexpr int COLS = BNX < 32 ? BNX : 32;
#pragma unroll
      for (int i = 0; i < COLS; i += 4) {
        if (c + i >= rows) break;
        float4 v = make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]),
                               __uint_as_float(r[i + 3]));
        if (none) v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (owner == crank) slot[(share - left) * 128] = v;
        else st_async(to + (share - left) * Cfg::GROUP_BYTES, v, bar);
        if (--left == 0) {
          ++owner;
          left = share;
          to = mapa(slot_addr, min(owner, cs - 1));
          bar = mapa(bar_addr, min(owner, cs - 1));
        }
      }
    }
  }
  __syncwarp();
  if (cs > 1) cluster_arrive_relaxed();
  const bool received = cs == 1 || mbar_wait(&rfull, 0, err, kErrSmemEmptyTimeout);
  tc_fence_before();
  const bool ok = __syncthreads_and(done && received);
  tc_fence_after();
  if (ok) {
#pragma unroll 1
    for (int turn = turn0; turn < turns; turn += 6) {
      const uint32_t r0 = next[0][0], r1 = next[0][1];
      if (p.residual != nullptr) {
#pragma unroll
        for (int i = 0; i + 1 < AHEAD; ++i) {
          next[i][0] = next[i + 1][0];
          next[i][1] = next[i + 1][1];
        }
        next[AHEAD - 1][0] = residual_at(turn + 6 * AHEAD, 0);
        next[AHEAD - 1][1] = residual_at(turn + 6 * AHEAD, 1);
      }
      // the partials in split order, the scales (the weight's first), bias
      const float4* at = part + turn * 32 + lane;
      float4 v = *at;
      if (cs > 1) {
        float4 t[Cfg::MAX_CLUSTER];
#pragma unroll
        for (int r = 1; r < Cfg::MAX_CLUSTER; ++r)
          t[r] = r < cs ? at[r * share * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 1; r < Cfg::MAX_CLUSTER; ++r)
          v = make_float4(v.x + t[r].x, v.y + t[r].y, v.z + t[r].z, v.w + t[r].w);
      }
      const float2 s = scol[(turn & 3) * 32 + lane];
      const float4 xs = *reinterpret_cast<const float4*>(sxs + (first + (turn >> 2)) * 4);
      v = make_float4(fmaf(v.x * s.x, xs.x, s.y), fmaf(v.y * s.x, xs.y, s.y), fmaf(v.z * s.x, xs.z, s.y),
                      fmaf(v.w * s.x, xs.w, s.y));
      const float a0 = __shfl_xor_sync(0xffffffffu, high ? v.x : v.z, SWIGLU ? 16 : 1);
      const float a1 = __shfl_xor_sync(0xffffffffu, high ? v.y : v.w, SWIGLU ? 16 : 1);
      const int row = row_of(turn), col = col_of(turn);
      const bool one = col < cols && row < rows, two = col < cols && row + 1 < rows;
      __nv_bfloat16* c = p.C + (m0 + row) * p.ldc + col;
      if constexpr (SWIGLU) {
        const float y0 = high ? silu(a0) * v.z : silu(v.x) * a0, y1 = high ? silu(a1) * v.w : silu(v.y) * a1;
        if (one) c[0] = __float2bfloat16_rn(y0 + __uint_as_float(r0 << 16));
        if (two) c[p.ldc] = __float2bfloat16_rn(y1 + __uint_as_float(r1 << 16));
      } else {
        const float2 f0 = unpack_bf16x2(r0), f1 = unpack_bf16x2(r1);
        const float2 y0 = high ? make_float2(a0, v.z) : make_float2(v.x, a0);
        const float2 y1 = high ? make_float2(a1, v.w) : make_float2(v.y, a1);
        if (one) *reinterpret_cast<uint32_t*>(c) = pack_bf16x2(y0.x + f0.x, y0.y + f0.y);
        if (two) *reinterpret_cast<uint32_t*>(c + p.ldc) = pack_bf16x2(y1.x + f1.x, y1.y + f1.y);
      }
    }
  }
  if (!ok) linger();  // products and copies in flight
  __syncwarp();
  if (warp == 1) tmem_dealloc(tmem, Cfg::TMEM_COLS);  // every read of it is behind the barrier
  if (cs > 1) {
    cluster_barrier_wait();  // no CTA leaves before the others' stores to it are issued
    if (!ok) linger();       // nor, where it did not count them, before they land
  }
}

// ---------------------------------------------------------------------------
// Many rows: CTA r of a pair loads rows [128 r, +128) of the tile's 256 rows of X
// and its half of the tile's BN rows of W; the leader issues the MMAs (M = 256, N =
// BN, K = 32), which accumulate rows [128 r, +128) in CTA r's tensor memory.  Loads
// of both complete on the leader's `full` barrier, commits arrive in both CTAs.
//
// The epilogue hides behind the next tile's k-blocks only if it is the shorter: four
// warps that read scales and bias from global memory took 449 us for 2048 x 3584 ->
// 37888 with SwiGLU, eight with both in shared memory and the approximate quotient
// 203.  Results and residual go through boxes of 32 x 32 in shared memory, by bulk
// tensor copies; residual loads by the threads cost 5087 x 3584 -> 3584 11 us, these 1.
constexpr int PAIR_BOX = 32 * 64;    // epilogue staging: 32 rows x 32 bf16 columns
constexpr int PAIR_BOXES = 3;        // of a warp: one is stored, one worked on, one being filled with residual
template <int BN>
struct PairCfg {
  static constexpr int STAGES = BN == 256 ? 5 : (BN == 128 ? 7 : 8);
  // eight: two to a quarter of TMEM's lanes, each with half of the tile's columns
  static constexpr int EPI_WARPS = BN == 64 ? 4 : 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int X_BYTES = 128 * BK;      // a CTA's half of X's k-block
  static constexpr int W_BYTES = BN / 2 * BK;   // and of W's
  static constexpr int COLS = BN / (EPI_WARPS / 4);  // accumulator columns of an epilogue warp
  static constexpr int EPI_BYTES = EPI_WARPS * (PAIR_BOXES * PAIR_BOX + 2 * COLS * 4);  // boxes; scales and bias
  static constexpr int SMEM = STAGES * (X_BYTES + W_BYTES) + EPI_BYTES + 1024 + 512;
  static constexpr int TMEM_COLS = 2 * BN;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Groups of `group_m` row tiles, rows fastest inside a group: the tiles in flight
// share few rows of X and of W, both from L2.
__device__ __forceinline__ void pair_tile(int t, int num_m, int num_n, int group_m, int& mb, int& nb) {
  const int per_group = group_m * num_n;
  const int first_m = (t / per_group) * group_m;
  const int gm = min(num_m - first_m, group_m);
  const int r = t % per_group;
  mb = first_m + r % gm;
  nb = r / gm;
}

template <int BN, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg<BN>::THREADS, 1)
    q8_pair_kernel(const __grid_constant__ Maps tm, const __grid_constant__ LLQ8Gemm p, int group_m, int* err) {
  using Cfg = PairCfg<BN>;
  constexpr int PAIR_STAGES = Cfg::STAGES, PAIR_COLS = Cfg::COLS, PAIR_EPI_WARPS = Cfg::EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sW = smem + PAIR_STAGES * Cfg::X_BYTES;
  uint8_t* sBox = sW + PAIR_STAGES * Cfg::W_BYTES;                                              // [warps][boxes]
  float* sCol = reinterpret_cast<float*>(sBox + PAIR_EPI_WARPS * PAIR_BOXES * PAIR_BOX);  // [warps][scales, bias]
  uint64_t* full = reinterpret_cast<uint64_t*>(sCol + PAIR_EPI_WARPS * 2 * PAIR_COLS);
  uint64_t* empty = full + PAIR_STAGES;
  uint64_t* tfull = empty + PAIR_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint64_t* rfull = drain + 1;  // [warps][boxes]: residual has landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + PAIR_EPI_WARPS * PAIR_BOXES);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t crank = cluster_rank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int num_m = (p.M + 255) / 256, num_n = (p.N + BN - 1) / BN;
  const int ntiles = num_m * num_n, num_kb = (p.K + BK - 1) / BK;
  pdl_trigger();

  // full, empty, tfull, tempty, drain and rfull lie in a row: a barrier a thread
  static_assert(2 * PAIR_STAGES + 5 + PAIR_EPI_WARPS * PAIR_BOXES <= 64, "two warps initialise the barriers");
  if (threadIdx.x < 2 * PAIR_STAGES + 5 + PAIR_EPI_WARPS * PAIR_BOXES) {
    uint64_t* bar = full + threadIdx.x;
    // tempty: the epilogue warps of both CTAs, on the leader
    mbar_init(bar, bar == tempty || bar == tempty + 1 ? 2 * PAIR_EPI_WARPS : 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)Cfg::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (warp == 0 && elect_one() && pair < ntiles) {  // the first ring of weights on its way to L2
    int mb, nb;
    pair_tile(pair, num_m, num_n, group_m, mb, nb);
    for (int k = 0; k < min(p.K, PAIR_STAGES * BK); k += BK) prefetch_box(&tm.w, k, nb * BN + (int)crank * (BN / 2));
  }
  __syncwarp();
  pdl_wait();

  const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), w0 = smem_u32(sW), x0 = smem_u32(sX);
  bool done = true;  // no wait of this thread ran out
  if (warp == 0) {
    if (elect_one()) {
      prefetch_tmap(&tm.x);
      prefetch_tmap(&tm.w);
      const uint32_t leader_full0 = mapa(full0, 0);
      int t = pair, k = 0, mb = 0, nb = 0;
      pair_tile(t, num_m, num_n, group_m, mb, nb);
      int xrow = mb * 256 + (int)crank * 128, wrow = nb * BN + (int)crank * (BN / 2);
      bool ok = true;
      for (uint32_t phase = 1; t < ntiles && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < PAIR_STAGES; ++s) {
          if (t >= ntiles) break;
          if (!wait(empty0 + 8 * s, phase, err, kErrSmemEmptyTimeout)) {
            ok = false;
            break;
          }
          if (crank == 0) expect(full0 + 8 * s, 2 * (Cfg::X_BYTES + Cfg::W_BYTES));
          load_pair(x0 + s * Cfg::X_BYTES, &tm.x, leader_full0 + 8 * s, k, xrow);
          load_pair(w0 + s * Cfg::W_BYTES, &tm.w, leader_full0 + 8 * s, k, wrow);
          k += BK;
          if (k >= p.K) {
            k = 0;
            t += npairs;
            if (t < ntiles) {
              pair_tile(t, num_m, num_n, group_m, mb, nb);
              xrow = mb * 256 + (int)crank * 128;
              wrow = nb * BN + (int)crank * (BN / 2);
            }
          }
        }
      }
      done = ok;
    }
  } else if (warp == 1) {
    if (crank == 0 && elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3(256, BN);
      const uint64_t xd = umma_desc_sw128_kmajor(x0), wd = umma_desc_sw128_kmajor(w0);
      int t = pair, kb = 0, acc = 0;
      uint32_t aphase = 1;
      bool ok = true;
      for (uint32_t phase = 0; t < ntiles && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < PAIR_STAGES; ++s) {
          if (t >= ntiles) break;
          if (kb == 0) {
            if (!wait(smem_u32(&tempty[acc]), aphase, err, kErrTmemEmptyTimeout)) {
              ok = false;
              break;
            }
          }
          if (!wait(full0 + 8 * s, phase, err, kErrTmaFullTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * BN;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_pair(d_tmem, xd + (s * Cfg::X_BYTES >> 4) + 2 * k, wd + (s * Cfg::W_BYTES >> 4) + 2 * k, idesc,
                     k == 0 ? (uint32_t)kb : 1u);
          commit_pair(empty0 + 8 * s);
          if (++kb == num_kb) {
            commit_pair(smem_u32(&tfull[acc]));
            kb = 0;
            t += npairs;
            if (++acc == 2) {
              acc = 0;
              aphase ^= 1;
            }
          }
        }
      }
      // every MMA issued is done before its accumulator is given back
      commit_pair_local(drain);
      mbar_wait(drain, 0, nullptr, 0);
      done = ok;
    }
    __syncwarp();
  } else {
    // warp w reads TMEM lanes [32 (w % 4), +32) (lane = row) of the tile's columns [COLS half, +COLS)
    const int q = warp & 3, e = warp - 2, half = e >> 2;
    const uint32_t leader_tempty0 = mapa(smem_u32(&tempty[0]), 0), leader_tempty1 = mapa(smem_u32(&tempty[1]), 0);
    uint8_t* boxes = sBox + e * PAIR_BOXES * PAIR_BOX;
    uint64_t* rbar = rfull + e * PAIR_BOXES;
    float* scol = sCol + e * 2 * PAIR_COLS;
    float* sbias = scol + PAIR_COLS;
    constexpr int STEP = SWIGLU ? 64 : 32;  // accumulator columns of a box of 32 output columns
    int acc = 0, b = 0;  // the box that is next
    uint32_t aphase = 0, bphase = 0;
    for (int t = pair; t < ntiles; t += npairs) {
      int mb, nb;
      pair_tile(t, num_m, num_n, group_m, mb, nb);
      const int row0 = mb * 256 + (int)crank * 128 + q * 32, row = row0 + lane;
      const int colw = nb * BN + half * PAIR_COLS;  // this warp's first accumulator column
      // what does not depend on the product, while it runs
      const float xs = row < p.M ? p.xs[row] : 1.f;
      // four columns a lane, of the first COLS / 4 lanes; N % 8 == 0: all four are there or none is
      const int cl = colw + 4 * lane;
      const bool mine = 4 * lane < PAIR_COLS;
      const float4 ws4 = mine && cl < p.N ? *reinterpret_cast<const float4*>(p.ws + cl) : make_float4(0, 0, 0, 0);
      const uint2 bias4 = p.bias != nullptr && mine && cl < p.N ? *reinterpret_cast<const uint2*>(p.bias + cl)
                                                                 : make_uint2(0, 0);
      // fills box `at` with the residual of accumulator columns [c, c + STEP),
      // once the store that last read the box is done with it
      auto fetch_residual = [&](int at, int c) {
        if (p.residual == nullptr || lane != 0 || c >= PAIR_COLS || colw + c >= p.N || row0 >= p.M) return;
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        mbar_arrive_expect_tx(&rbar[at], PAIR_BOX);
        tma_load_2d(boxes + at * PAIR_BOX, &tm.r, &rbar[at], SWIGLU ? (colw + c) / 2 : colw + c, row0);
      };
      fetch_residual(b, 0);
      __syncwarp();  // the tile before is read
      if (mine) {
        const float2 b0 = unpack_bf16x2(bias4.x), b1 = unpack_bf16x2(bias4.y);
        *reinterpret_cast<float4*>(scol + 4 * lane) = ws4;
        *reinterpret_cast<float4*>(sbias + 4 * lane) = make_float4(b0.x, b0.y, b1.x, b1.y);
      }
      __syncwarp();
      // lanes leave a wait one by one; the loads below take a whole warp
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], aphase, err, kErrTmemFullTimeout))) {
        done = false;
        break;
      }
      tc_fence_after();
      const uint32_t tbase = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * BN + half * PAIR_COLS);
      // (r[i] ws) xs + bias of columns [c, c + 32); every lane reads the same of them
      auto scaled = [&](const uint32_t (&r)[32], int c, int i) {
        const float4 s = *reinterpret_cast<const float4*>(scol + c + i);
        const float4 t = *reinterpret_cast<const float4*>(sbias + c + i);
        return make_float4(fmaf(__uint_as_float(r[i]) * s.x, xs, t.x), fmaf(__uint_as_float(r[i + 1]) * s.y, xs, t.y),
                           fmaf(__uint_as_float(r[i + 2]) * s.z, xs, t.z),
                           fmaf(__uint_as_float(r[i + 3]) * s.w, xs, t.w));
      };
#pragma unroll 1
      for (int c = 0; c < PAIR_COLS && done; c += 64) {
        if (colw + c >= p.N || row0 >= p.M) break;  // outside C
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(tbase + c, r[0]);
        tmem_ld_32x32b_x32(tbase + c + 32, r[1]);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 64 / STEP; ++h) {
          const int cb = c + h * STEP;  // of this box
          if (colw + cb >= p.N) break;
          const int out0 = SWIGLU ? (colw + cb) / 2 : colw + cb;
          float v[32];
          if constexpr (SWIGLU) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 g = scaled(r[j], c + 32 * j, i), u = scaled(r[j], c + 32 * j, i + 16);
                v[16 * j + i] = silu(g.x) * u.x;
                v[16 * j + i + 1] = silu(g.y) * u.y;
                v[16 * j + i + 2] = silu(g.z) * u.z;
                v[16 * j + i + 3] = silu(g.w) * u.w;
              }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 y = scaled(r[h], cb, i);
              v[i] = y.x;
              v[i + 1] = y.y;
              v[i + 2] = y.z;
              v[i + 3] = y.w;
            }
          }
          // 16-byte chunk k of row r is chunk k ^ ((r >> 1) & 3) of a box, the 64-byte
          // swizzle of the maps; rows past M and columns past N are clipped there
          uint4* d = reinterpret_cast<uint4*>(boxes + b * PAIR_BOX + lane * 64);
          const int swz = (lane >> 1) & 3;
          if (p.residual != nullptr) {
            fetch_residual(b == PAIR_BOXES - 1 ? 0 : b + 1, cb + STEP);
            if (!__all_sync(0xffffffffu, mbar_wait(&rbar[b], bphase, err, kErrTmaFullTimeout))) {
              done = false;
              break;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 rv = d[k ^ swz];
              const uint32_t ru[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = unpack_bf16x2(ru[j]);
                v[8 * k + 2 * j] += f.x;
                v[8 * k + 2 * j + 1] += f.y;
              }
            }
          } else {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PAIR_BOXES - 1) : "memory");
            __syncwarp();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            d[k ^ swz] = make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                                    pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            store_box(&tm.c, boxes + b * PAIR_BOX, out0, row0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          __syncwarp();
          if (++b == PAIR_BOXES) {
            b = 0;
            bphase ^= 1;
          }
        }
      }
      if (!done) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(acc == 0 ? leader_tempty0 : leader_tempty1);
      if (++acc == 2) {
        acc = 0;
        aphase ^= 1;
      }
    }
    // the boxes are read; the grid's end completes the writes
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }

  if (!done) linger();  // neither CTA leaves before
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"((uint32_t)Cfg::TMEM_COLS)
                 : "memory");
  }
}

// ---------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeFn>(f)
               : nullptr;
  }();
  return fn;
}

// Row-major [rows, K] of e4m3: boxes of 128 values x box_rows, 128-byte swizzle, zeros out of bounds.
static bool operand_map(CUtensorMap* tm, const void* ptr, int rows, int K, int64_t ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const EncodeFn enc = encode_fn();
  return enc != nullptr && enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// C, or the residual: boxes of 32 columns (64 bytes) x 32 rows, 64-byte swizzle.
static bool output_map(CUtensorMap* tm, const void* ptr, int rows, int cols, int64_t ld) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {32, 32}, estr[2] = {1, 1};
  const EncodeFn enc = encode_fn();
  return enc != nullptr && enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Kern>
static int launch(Kern kern, dim3 grid, int smem, int cluster, cudaStream_t stream, unsigned long long& done,
                  const Maps& tm, const LLQ8Gemm& p, int* err) {
  if (!smem_on_device(kern, smem, done)) return -7;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, tm, p, err) == cudaSuccess ? 0 : -5;
}

// CTAs that share a feature tile's K, two a SM: as many as have places (larger clusters
// than pairs do not fill the SMs to the last place), also where K is shorter than
// that, since they share the epilogue too; two for more tiles than places, whose last
// round would be a long one.  Over 1133 random sizes (1 to 32 rows, behind their
// quantisation) 1.0 % slower than the best of 1 to 8 CTAs in the geometric mean.
constexpr int SPLIT_PLACES = 248, SPLIT_ROUND = 296;
static int split_rule(int tiles, int num_kb) {
  int cs = SPLIT_PLACES / tiles;
  if ((tiles > SPLIT_PLACES / 2 && tiles <= SPLIT_ROUND / 2) || (tiles > SPLIT_ROUND && num_kb >= 64)) cs = 2;
  return cs < 1 ? 1 : (cs > SPLIT_MAX_CLUSTER ? SPLIT_MAX_CLUSTER : cs);
}

// The same with one CTA a SM: the largest cluster with which all tiles run at once, 0
// for more tiles than SMs.  The places are what the occupancy calculator gives clusters
// of each size: they lie within a GPC, whose SMs clusters of seven and eight do not fill.
static int deep_rule(int64_t tiles) {
  constexpr int places[SPLIT_MAX_CLUSTER + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};
  for (int cs = SPLIT_MAX_CLUSTER; cs >= 1; --cs)
    if (tiles * cs <= places[cs]) return cs;
  return 0;
}

// The kernel for 33 to 64 rows: up to 74 feature tiles, half the SMs, the deep ring (with
// more it loses as often as it wins).  Over 716 random sizes 0.4 % slower than the best of
// all.
static int middle_rule(int N, int K) {
  const int tiles = (N + 127) / 128, num_kb = (K + BK - 1) / BK;
  return tiles > 74 ? split_rule(tiles, num_kb) : SPLIT_DEEP + deep_rule(tiles);
}

// The kernel for more than 64 rows: the one with the least modelled time, a start
// and then, for each round of tiles, the k-blocks and the part of the epilogue that
// the next tile does not hide; for the deep split kernel a CTA's k-blocks and an
// epilogue by rows.  The figures (us) are fitted to 2033 random sizes (65 to 5000 rows)
// timed with every kernel but that one, 0.3 % slower than the best in the geometric mean
// (tiles of 64, 128 or 256 features alone 32, 12 and 23 %), and to 656 sizes (65 to 160
// rows) with it; over 616 others 0.7 % slower than the best.
static int kernel_rule(int M, int N, int K, int sms) {
  struct Cost {
    int kernel, tile_rows, tile_features, places;
    double start, block, tile;
  };
  const Cost costs[] = {{64, 256, 64, sms / 2, 3.6, 0.085, 0.9},
                        {128, 256, 128, sms / 2, 3.3, 0.14, 1.15},
                        {256, 256, 256, sms / 2, 3.85, 0.225, 1.15},
                        {1, 128, 128, 2 * sms, 4.45, 0.34, 1.55}};
  const int num_kb = (K + BK - 1) / BK;
  int best = 0;
  double least = 0;
  for (const Cost& c : costs) {
    // more row tiles than a grid has places along z: short rows, few features
    if (c.kernel <= SPLIT_MAX_CLUSTER && M > 128 * 65535) continue;
    const int64_t tiles =
        (int64_t)((M + c.tile_rows - 1) / c.tile_rows) * ((N + c.tile_features - 1) / c.tile_features);
    const double t = c.start + (double)((tiles + c.places - 1) / c.places) * (num_kb * c.block + c.tile);
    if (best == 0 || t < least) {
      best = c.kernel;
      least = t;
    }
  }
  const int cs = deep_rule((int64_t)((M + 127) / 128) * ((N + 127) / 128));
  if (cs > 0) {
    const double t = 4.0 + (num_kb + cs - 1) / cs * 0.23 + 1.7 * (M < 128 ? M : 128) / 128;
    if (t < least) best = SPLIT_DEEP + cs;
  }
  return best;
}

template <int BNX, bool SWIGLU, bool DEEP = false>
static int split_run(const LLQ8Gemm& p, int cs, int* err, cudaStream_t stream) {
  Maps tm;
  if (!operand_map(&tm.w, p.w, p.N, p.K, p.ldw, 128) || !operand_map(&tm.x, p.x, p.M, p.K, p.ldx, BNX)) return -2;
  tm.c = tm.r = tm.x;  // not read
  const dim3 grid(cs, (p.N + 127) / 128, (p.M + BNX - 1) / BNX);
  if (grid.y > 65535 || grid.z > 65535) return -3;
  static unsigned long long done = 0;
  return launch(q8_split_kernel<BNX, SWIGLU, DEEP>, grid, SplitCfg<BNX, DEEP>::SMEM, cs, stream, done, tm, p, err);
}
template <bool SWIGLU>
static int split_launch(const LLQ8Gemm& p, int kernel, int* err, cudaStream_t stream) {
  const int tiles = (p.N + 127) / 128, num_kb = (p.K + BK - 1) / BK;
  const bool deep = kernel > SPLIT_DEEP;
  int cs = deep ? kernel - SPLIT_DEEP : (kernel > 0 ? kernel : split_rule(tiles, num_kb));
  if (!deep && p.M > 32) {
    const int most = p.M > 64 ? SplitCfg<128, false>::MAX_CLUSTER : SplitCfg<64, false>::MAX_CLUSTER;
    cs = cs < most ? cs : most;
  }
  if (deep && p.M > 64) return split_run<128, SWIGLU, true>(p, cs, err, stream);
  if (deep) return split_run<64, SWIGLU, true>(p, cs, err, stream);
  if (p.M > 64) return split_run<128, SWIGLU>(p, cs, err, stream);
  if (p.M <= 16) return split_run<16, SWIGLU>(p, cs, err, stream);
  if (p.M <= 32) return split_run<32, SWIGLU>(p, cs, err, stream);
  return split_run<64, SWIGLU>(p, cs, err, stream);
}

template <int BN, bool SWIGLU>
static int pair_launch(const LLQ8Gemm& p, int sms, int* err, cudaStream_t stream) {
  using Cfg = PairCfg<BN>;
  Maps tm;
  if (!operand_map(&tm.x, p.x, p.M, p.K, p.ldx, 128) || !operand_map(&tm.w, p.w, p.N, p.K, p.ldw, BN / 2) ||
      !output_map(&tm.c, p.C, p.M, SWIGLU ? p.N / 2 : p.N, p.ldc))
    return -2;
  tm.r = tm.c;  // read with a residual only
  if (p.residual != nullptr && !output_map(&tm.r, p.residual, p.M, SWIGLU ? p.N / 2 : p.N, p.ldr)) return -2;
  const int num_m = (p.M + 255) / 256;
  const int64_t tiles = (int64_t)num_m * ((p.N + BN - 1) / BN);
  if (tiles > (1ll << 30)) return -3;
  const int pairs = tiles < sms / 2 ? (int)tiles : sms / 2;
  // as many row tiles a group as keep their rows of X within 40 MB of L2
  int64_t group = (40ll << 20) / ((int64_t)256 * p.K);
  group = group < 8 ? 8 : group;
  group = group > num_m ? num_m : group;
  static unsigned long long done = 0;
  auto kern = q8_pair_kernel<BN, SWIGLU>;
  if (!smem_on_device(kern, Cfg::SMEM, done)) return -7;
  const cudaError_t e =
      launch_pdl(kern, dim3(2 * pairs), dim3(Cfg::THREADS), Cfg::SMEM, stream, tm, p, (int)group, err);
  return e == cudaSuccess ? 0 : -5;
}

}  // namespace q8
}  // namespace ll

// `kernel`: 0 by the rule below; 1 to 8 the split kernel with that many CTAs to a
// feature tile (at most three for more than 32 rows, one for more than 64), 11 to 18
// the same with the deep ring and 1 to 8; 64, 128 or 256 the pair kernel with tiles of so
// many features.
extern "C" int ll_q8_gemm(const LLQ8Gemm* p, int swiglu, int kernel, int* err, cudaStream_t stream) {
  using namespace ll::q8;
  if (p->M <= 0) return 0;
  if (p->N <= 0 || p->K <= 0 || (p->K % 16) || (p->N % 8) || (swiglu && (p->N % 32))) return -3;
  if ((p->ldx % 16) || (p->ldw % 16) || (p->ldc % 8) || (p->ldr % 8)) return -3;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return -5;
  if (kernel == 0 && p->M > 64) kernel = kernel_rule(p->M, p->N, p->K, sms);
  else if (kernel == 0 && p->M > 32) kernel = middle_rule(p->N, p->K);
  if (kernel <= SPLIT_MAX_CLUSTER && p->N > 128 * 65535) kernel = 256;  // more feature tiles than a grid has places
  const auto run = [&](auto gated) {
    constexpr bool G = decltype(gated)::value;
    if ((kernel >= 0 && kernel <= SPLIT_MAX_CLUSTER) ||
        (kernel > SPLIT_DEEP && kernel <= SPLIT_DEEP + SPLIT_MAX_CLUSTER))
      return split_launch<G>(*p, kernel, err, stream);
    if (kernel == 64) return pair_launch<64, G>(*p, sms, err, stream);
    if (kernel == 128) return pair_launch<128, G>(*p, sms, err, stream);
    if (kernel == 256) return pair_launch<256, G>(*p, sms, err, stream);
    return -3;
  };
  return swiglu ? run(std::true_type{}) : run(std::false_type{});
}
