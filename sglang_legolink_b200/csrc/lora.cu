// The low-rank half of the adapter projection (lora.h): low = scale x A^T.
//
// Per plane (a row tile's adapter) and 128-row half of the tile: a 128 x rank
// product over K on tcgen05, x rows on the M side and the adapter's ranks on
// the N side, K split over the CTAs of a cluster.  It is bound by reading x
// (K / rank is large: 36 MB of x against 0.3 MB of A at 5087 rows x 3584,
// rank 48), so what counts is bytes in flight: the cluster split puts up to
// two CTAs with a ~96 KB ring on every SM whatever the number of row tiles.
// The CTAs' fp32 partials meet in distributed shared memory and are summed in
// CTA order, so a row's bits do not depend on timing.  That case takes 18 us
// with cold caches; warm about 14: 4 until the last cluster has started, 1.3 to
// read the plan and set up, 5 for the loads (8 TB/s, from L2 where two planes
// share rows), 4 for the partials.
//
// low is kept as two bf16 planes, hi = bf16(v) and lo = bf16(v - hi): the
// product that reads them takes bf16 operands, and one bf16 would put 2^-9 of
// every low-rank value into the result, as much again as rounding the result
// itself; hi + lo holds 16 bits and costs one more k-block per 64 ranks of a
// plane (none up to rank 32, lora.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "lora.h"

namespace ll {

constexpr int LOW_BM = 128;
constexpr int LOW_BK = 64;
constexpr int LOW_MAX_CLUSTER = 8;
constexpr int LOW_RING = 96 * 1024;

struct LowShape {
  int npad;      // ranks rounded up to the MMA's multiple of 16
  int x_rows;    // rows of the x box
  int stages;
  int tmem_cols;
  int part_ld;   // floats per row of the partials
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t low_mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void low_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// grid: (cluster, halves of a row tile, planes); cluster dims (cs, 1, 1)
__global__ void __launch_bounds__(128, 2)
    lora_low_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, int M, int K,
                    const __grid_constant__ LLLora lo, const __grid_constant__ LowShape shp, int* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int a_bytes = shp.npad * LOW_BK * 2, x_bytes = shp.x_rows * LOW_BK * 2;
  uint8_t* sX = smem;
  uint8_t* sA = smem + shp.stages * LOW_BM * LOW_BK * 2;
  float* part = reinterpret_cast<float*>(smem);  // over the ring, once the product is done
  __shared__ uint64_t full[8], empty[8], tfull;
  __shared__ uint32_t tmem_slot;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = gridDim.x, crank = blockIdx.x;
  const int plane = blockIdx.z;

  // which rows and which adapter: the same for every CTA of the cluster
  const int planes = lo.tile_ptr[lo.tiles];
  if (plane >= planes) {
    pdl_wait();  // with no plane at all, this grid's end must still mean the previous one's
    return;
  }
  const int t = lo.plane_tile[plane], adapter = lo.plane_adapter[plane];
  const int m0 = t * lo.tile_rows + blockIdx.y * LOW_BM;
  if (planes > lo.max_planes || t < 0 || t >= lo.tiles || adapter < 0 || adapter >= lo.adapters) {
    if (tid == 0) record_error(err, kErrBadIndex);
    pdl_wait();
    return;
  }
  if (m0 >= M) {
    pdl_wait();
    return;
  }
  const int rows = min(LOW_BM, M - m0), slot = plane - lo.tile_ptr[t];
  const bool mine = tid < rows && lo.row_slot[m0 + tid] == slot;
  const int ld = lo.ld();
  bf16* low = lo.low + ((size_t)plane * lo.halves() * lo.tile_rows + blockIdx.y * LOW_BM) * ld;
  const size_t to_lo = lo.to_lo();
  const int groups = (lo.packed() ? 32 : lo.rank) / 4;  // 4 columns a thread
  if (!__syncthreads_or(mine)) {   // no row of this half uses the adapter
    pdl_wait();
    pdl_trigger();
    for (int i = crank * 128 + tid; i < rows * groups; i += cs * 128) {
      bf16* d = low + (size_t)(i / groups) * ld + 4 * (i % groups);
      *reinterpret_cast<uint2*>(d) = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(d + to_lo) = make_uint2(0, 0);
    }
    return;
  }

  if (tid == 0) {
    for (int s = 0; s < shp.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, shp.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int num_kb = (K + LOW_BK - 1) / LOW_BK;
  const int per = (num_kb + cs - 1) / cs;
  const int kb0 = min(num_kb, crank * per), kb1 = min(num_kb, kb0 + per);

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmA);
    // the adapter does not depend on the previous kernel: its first tiles
    // are on their way before the wait for x
    const int pre = min(kb1 - kb0, shp.stages);
    for (int i = 0; i < pre; ++i) {
      mbar_arrive_expect_tx(&full[i], a_bytes + x_bytes);
      tma_load_3d(sA + i * a_bytes, &tmA, &full[i], (kb0 + i) * LOW_BK, 0, adapter);
    }
    pdl_wait();
    // only now: every CTA that lets the product start has seen x complete, so
    // the product may read x at once (lora_gemv_kernel, `x_ready`)
    pdl_trigger();
    for (int i = 0; i < pre; ++i)
      tma_load_2d(sX + i * LOW_BM * LOW_BK * 2, &tmX, &full[i], (kb0 + i) * LOW_BK, m0);
    int stage = pre % shp.stages;
    uint32_t phase = pre == shp.stages ? 1 : 0;
    bool ok = true;
    for (int kb = kb0 + pre; kb < kb1; ++kb) {
      if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrSmemEmptyTimeout)) {
        ok = false;
        break;
      }
      mbar_arrive_expect_tx(&full[stage], a_bytes + x_bytes);
      tma_load_3d(sA + stage * a_bytes, &tmA, &full[stage], kb * LOW_BK, 0, adapter);
      tma_load_2d(sX + stage * LOW_BM * LOW_BK * 2, &tmX, &full[stage], kb * LOW_BK, m0);
      if (++stage == shp.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) {  // let the copies in flight land before the CTA exits
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t idesc = umma_idesc_bf16_f32(LOW_BM, shp.npad);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&full[stage], phase, err, kErrTmaFullTimeout)) break;
      tc_fence_after();
      const uint64_t xd = umma_desc_sw128_kmajor(smem_u32(sX + stage * LOW_BM * LOW_BK * 2));
      const uint64_t ad = umma_desc_sw128_kmajor(smem_u32(sA + stage * a_bytes));
#pragma unroll
      for (int k = 0; k < LOW_BK / 16; ++k)
        umma_bf16(tmem, xd + 2 * k, ad + 2 * k, idesc, (kb != kb0 || k != 0) ? 1u : 0u);
      umma_commit(&empty[stage]);
      if (++stage == shp.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    umma_commit(&tfull);
  }
  __syncwarp();
  pdl_wait();  // `low` may still be read by the previous product
  const bool ok = __syncthreads_and(mbar_wait(&tfull, 0, err, kErrTmemFullTimeout));
  tc_fence_after();
  // this thread's row of the partial product (TMEM lane = row)
  if (warp * 32 < rows) {
    for (int c = 0; c < lo.rank; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tmem + (uint32_t(warp * 32) << 16) + c, r);
      tmem_ld_wait();
      float* d = part + (size_t)tid * shp.part_ld + c;
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        if (c + i < lo.rank && tid < rows)  // the partials have `rows` rows, not the warp's 32
          *reinterpret_cast<float4*>(d + i) =
              kb1 > kb0 ? make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]),
                                      __uint_as_float(r[i + 3]))
                        : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  tc_fence_before();
  low_cluster_sync();
  tc_fence_after();
  if (ok) {
    const float scale = lo.scale[adapter];
    const uint32_t base = smem_u32(part);
    for (int i = crank * 128 + tid; i < rows * groups; i += cs * 128) {
      const int row = i / groups, g = i % groups;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (4 * g < lo.rank && lo.row_slot[m0 + row] == slot) {
        float4 p[LOW_MAX_CLUSTER];  // all of them in flight at once
        const uint32_t at = base + (uint32_t)(row * shp.part_ld + 4 * g) * 4;
#pragma unroll
        for (int r = 0; r < LOW_MAX_CLUSTER; ++r)
          p[r] = r < cs ? ld_cluster_f32x4(low_mapa(at, r)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < LOW_MAX_CLUSTER; ++r) {
          v.x += p[r].x;
          v.y += p[r].y;
          v.z += p[r].z;
          v.w += p[r].w;
        }
        v.x *= scale;
        v.y *= scale;
        v.z *= scale;
        v.w *= scale;
      }
      const uint32_t h0 = pack_bf16x2(v.x, v.y), h1 = pack_bf16x2(v.z, v.w);
      const float2 f0 = unpack_bf16x2(h0), f1 = unpack_bf16x2(h1);
      bf16* d = low + (size_t)row * ld + 4 * g;
      *reinterpret_cast<uint2*>(d) = make_uint2(h0, h1);
      // an infinite value has no remainder
      const float r0 = v.x - f0.x, r1 = v.y - f0.y, r2 = v.z - f1.x, r3 = v.w - f1.y;
      auto rest = [](float r) { return r == r && fabsf(r) < 3.0e38f ? r : 0.f; };
      *reinterpret_cast<uint2*>(d + to_lo) =
          make_uint2(pack_bf16x2(rest(r0), rest(r1)), pack_bf16x2(rest(r2), rest(r3)));
    }
  }
  low_cluster_sync();  // the partials live until every CTA has read them
  if (warp == 1) tmem_dealloc(tmem, shp.tmem_cols);
}

// ---------------------------------------------------------------------------
// The product for up to 128 rows (decode), and for more where 128 x 128 tiles
// leave SMs free: as the small-M GEMM, the weight tile is the M = 128 side of
// the MMA and the rows (128 a CTA at most) are the N side, and K is split so
// that every SM streams weights.  Here the splits of a feature tile are a
// cluster: their fp32 partials stay in shared memory and each CTA sums, in
// split order, and stores its share of the rows.  Nothing goes through global
// memory and no CTA waits for a last one to add up 128 features x M rows x all
// splits (at 61 rows x 5120 features, 7 splits, that fix-up alone was 40 of 62
// us).  Each split takes its share of the k-blocks of K, then its share of the
// adapters'.
//
// Behind the few-row kernel (2 to 5 us) the first ring of weights is on its way
// while that one waits for x and runs.  Behind the tensor-core kernel (10 us
// and more) this one starts when x is there (`x_ready`) and runs the k-blocks
// of K beside it; the wait comes before the adapters' k-blocks: 300 rows, 3584
// -> 4608, rank 48, 27.9 -> 22.2 us, 300 x 3584 x 18944 84.7 -> 66.8.  (The same
// behind the few-row kernel: 16 rows, 3584 -> 37888, 48.4 -> 50.0.)
//
// Bound by reading weights: 16 rows, 3584 -> 37888 with SwiGLU and 6 adapters of
// rank 32 (288 MB) in 48.7 us for both kernels in a graph, 5.9 TB/s.
constexpr int GEMV_RING = 108 * 1024;
// Clusters do not fill the SMs to the last place (two CTAs a SM, 296 places):
// 36 clusters of 8 and 40 of 7 ran a second round.  us a call with 2 / 4 / 6 /
// 8 (7) CTAs (hi and lo in blocks of their own): 1 row x 4608 features 12.9 /
// 10.1 / 8.6 / 14.3, 61 rows x 5120 43.2 / 31.1 / 27.9 / 38.7.
constexpr int GEMV_MAX_CLUSTER = 6;
constexpr int GEMV_PLACES = 248;
template <int BNX>
struct GemvCfg {
  static constexpr int W_BYTES = 128 * LOW_BK * 2;
  static constexpr int X_BYTES = BNX * LOW_BK * 2;
  static constexpr int STAGES = GEMV_RING / (W_BYTES + X_BYTES);
  static constexpr int TMEM_COLS = BNX < 32 ? 32 : BNX;
  static constexpr int LD = 132;  // floats per row of the partials
  static constexpr int SMEM = STAGES * (W_BYTES + X_BYTES) + 1024;
  static_assert(BNX * LD * 4 <= STAGES * (W_BYTES + X_BYTES), "the partials overlay the ring");
};

struct alignas(64) GemvMaps {
  CUtensorMap w, x, low, b;
};

__device__ __forceinline__ float gemv_silu(float x) { return x / (1.0f + __expf(-x)); }

template <int BNX, bool SWIGLU>
__global__ void __launch_bounds__(192, 2)
    lora_gemv_kernel(const __grid_constant__ GemvMaps tm, bf16* __restrict__ C, int64_t ldc,
                     const bf16* __restrict__ bias, int rows, int N, int K, const __grid_constant__ LLLora lo,
                     bool x_ready, int* err) {
  using Cfg = GemvCfg<BNX>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + STAGES * Cfg::W_BYTES;
  float* part = reinterpret_cast<float*>(smem);  // [M][LD], over the ring, once the product is done
  __shared__ uint64_t full[STAGES], empty[STAGES], tfull;
  __shared__ uint32_t tmem_slot;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = gridDim.x, crank = blockIdx.x, nb = blockIdx.y;
  const int num_kb = (K + LOW_BK - 1) / LOW_BK;
  const int per_plane = lo.steps();
  const int m0 = blockIdx.z * BNX, M = min(BNX, rows - m0);  // this CTA's rows
  const int t = m0 / lo.tile_rows, p0 = max(0, lo.tile_ptr[t]);
  const int num_extra = max(0, min(lo.tile_ptr[t + 1], lo.max_planes) - p0) * per_plane;
  C += m0 * ldc;
  const int per = (num_kb + cs - 1) / cs, eper = (num_extra + cs - 1) / cs;
  const int kb0 = min(num_kb, crank * per), kb1 = min(num_kb, kb0 + per);
  const int e0 = min(num_extra, crank * eper), e1 = min(num_extra, e0 + eper);
  const int steps = kb1 - kb0 + e1 - e0;
  pdl_trigger();

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int pre = min(kb1 - kb0, STAGES);
      for (int i = 0; i < pre; ++i) {
        mbar_arrive_expect_tx(&full[i], Cfg::W_BYTES + Cfg::X_BYTES);
        tma_load_2d(sW + i * Cfg::W_BYTES, &tm.w, &full[i], (kb0 + i) * LOW_BK, nb * 128);
      }
      bool waited = !x_ready;
      if (waited) pdl_wait();
      for (int i = 0; i < steps; ++i) {
        const int kb = kb0 + i;
        if (i >= pre) {
          if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrSmemEmptyTimeout)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], Cfg::W_BYTES + Cfg::X_BYTES);
        }
        if (kb < kb1) {
          if (i >= pre) tma_load_2d(sW + stage * Cfg::W_BYTES, &tm.w, &full[stage], kb * LOW_BK, nb * 128);
          tma_load_2d(sX + stage * Cfg::X_BYTES, &tm.x, &full[stage], kb * LOW_BK, m0);
        } else {
          if (!waited) pdl_wait();
          waited = true;
          const int e = e0 + kb - kb1;
          const int plane = p0 + e / per_plane, s = e % per_plane, rb = s >> 1;
          tma_load_3d(sW + stage * Cfg::W_BYTES, &tm.b, &full[stage], rb * LOW_BK, nb * 128,
                      lo.plane_adapter[plane]);
          tma_load_2d(sX + stage * Cfg::X_BYTES, &tm.low, &full[stage], rb * LOW_BK,
                      (plane * lo.halves() + (s & 1)) * lo.tile_rows + m0 % lo.tile_rows);
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) {  // let the copies in flight land before the CTA exits
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_bf16_f32(128, BNX);
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < steps; ++i) {
        if (!mbar_wait(&full[stage], phase, err, kErrTmaFullTimeout)) break;
        tc_fence_after();
        const uint64_t ad = umma_desc_sw128_kmajor(smem_u32(sW + stage * Cfg::W_BYTES));
        const uint64_t bd = umma_desc_sw128_kmajor(smem_u32(sX + stage * Cfg::X_BYTES));
        const uint64_t again = lo.packed() && i >= kb1 - kb0 ? 4 : 0;  // lo meets B's first columns again
#pragma unroll
        for (int k = 0; k < LOW_BK / 16; ++k)
          umma_bf16(tmem, ad + 2 * k - (k >= 2 ? again : 0), bd + 2 * k, idesc, (i | k) != 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      umma_commit(&tfull);
    }
  }
  __syncwarp();
  pdl_wait();  // the output may still be read by an earlier kernel's successor
  const bool ok = __syncthreads_and(mbar_wait(&tfull, 0, err, kErrTmemFullTimeout));
  tc_fence_after();
  if (warp >= 2) {  // TMEM lane quarter of this warp: features; columns: rows
    const int f = (warp & 3) * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < BNX && c < M; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tmem + (uint32_t((warp & 3) * 32) << 16) + c, r);  // BNX 16: columns 16.. unused
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c + i < M && c + i < BNX) part[(c + i) * Cfg::LD + f] = steps > 0 ? __uint_as_float(r[i]) : 0.f;
    }
  }
  tc_fence_before();
  low_cluster_sync();
  tc_fence_after();
  if (ok) {
    const uint32_t base = smem_u32(part);
    auto sum4 = [&](int row, int f) {
      float4 p[GEMV_MAX_CLUSTER];
      const uint32_t at = base + (uint32_t)(row * Cfg::LD + f) * 4;
#pragma unroll
      for (int r = 0; r < GEMV_MAX_CLUSTER; ++r) p[r] = r < cs ? ld_cluster_f32x4(low_mapa(at, r)) : make_float4(0, 0, 0, 0);
      float4 v = p[0];
#pragma unroll
      for (int r = 1; r < GEMV_MAX_CLUSTER; ++r) {
        v.x += p[r].x;
        v.y += p[r].y;
        v.z += p[r].z;
        v.w += p[r].w;
      }
      if (bias != nullptr) {
        const uint2 bv = *reinterpret_cast<const uint2*>(bias + nb * 128 + f);
        const float2 b0 = unpack_bf16x2(bv.x), b1 = unpack_bf16x2(bv.y);
        v.x += b0.x;
        v.y += b0.y;
        v.z += b1.x;
        v.w += b1.y;
      }
      return v;
    };
    constexpr int GROUPS = SWIGLU ? 16 : 32;  // 4-feature groups a row
    for (int i = crank * 192 + tid; i < M * GROUPS; i += cs * 192) {
      const int row = i / GROUPS, g = i % GROUPS;
      if constexpr (SWIGLU) {  // 16 gate features, then the matching 16 up features
        const int f = (g >> 2) * 32 + (g & 3) * 4;
        if (nb * 128 + f >= N) continue;
        const float4 a = sum4(row, f), u = sum4(row, f + 16);
        *reinterpret_cast<uint2*>(C + row * ldc + nb * 64 + 4 * g) =
            make_uint2(pack_bf16x2(gemv_silu(a.x) * u.x, gemv_silu(a.y) * u.y),
                       pack_bf16x2(gemv_silu(a.z) * u.z, gemv_silu(a.w) * u.w));
      } else {
        if (nb * 128 + 4 * g >= N) continue;
        const float4 v = sum4(row, 4 * g);
        *reinterpret_cast<uint2*>(C + row * ldc + nb * 128 + 4 * g) =
            make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      }
    }
  }
  low_cluster_sync();  // the partials live until every CTA has read them
  if (warp == 1) tmem_dealloc(tmem, Cfg::TMEM_COLS);
}

// A load that stays behind pdl_wait(): one through a __restrict__ pointer to
// const may be moved above it, since nothing in the kernel writes there.
__device__ __forceinline__ uint4 ld_after_wait(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Few rows (decode): dot products, `ks` warps of a CTA to each (row, rank),
// every warp with its share of the adapter's row in registers before the wait
// for x.  No shared tiles, and one of these CTAs a SM leaves registers for the
// product's two, which load weights meanwhile; what counts is the time from x
// to the stored value, 1.5 us less than the tensor-core kernel's chain (tiles,
// TMEM, partials, cluster).  A is read once per row here, from L2 where rows
// share it.  Fewer registers (4 vectors a lane, 62) and more CTAs a SM: 61 rows
// 25.6 to 27.7 us a call for 26.8, one row 9.7 to 10.6 for 9.6.
//
// Each (row, rank) is a CTA's share, two CTAs a SM: used up to one round of the
// 296 places, two (one and a half where K is short) where a tile has many
// planes, each of which costs the tensor-core kernel CTAs and loads.  us a call
// with this kernel / the tensor cores', 4608 features: 48 rows, K = 3584, rank
// 16 (192 CTAs) 11.4 / 12.7; 64, 1024, 32 (256) 10.3 / 11.0; 48, 3584, 32 (384)
// 13.6 / 12.8; 96, 3584, 16 (384) with 6 planes 16.0 / 14.8, with 57 24.8 /
// 27.2; 61, 8192, 16 (488) with 26 planes 26.0 / 27.7; 64, 3584, 48 (768) with 6
// planes 17.7 / 14.3.
constexpr int ROWS_PLACES = 296, ROWS_SHORT = 444, ROWS_LONG = 592, ROWS_PLANES = 8;
constexpr int ROWS_VEC = 8;  // 16-byte vectors a lane holds: 2048 elements of K a warp
__global__ void __launch_bounds__(256, 2) lora_low_rows_kernel(const bf16* x, int64_t ldx, int M, int K,
                                                               const __grid_constant__ LLLora lo, int ks, int* err) {
  __shared__ float parts[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = 8 / ks, share = warp % ks;
  const int m = blockIdx.x, r = blockIdx.y * per + warp / ks;
  pdl_trigger();
  const int t = m / lo.tile_rows;
  const int p0 = lo.tile_ptr[t], np = lo.tile_ptr[t + 1] - p0, slot = lo.row_slot[m];
  if (p0 < 0 || np < 0 || p0 + np > lo.max_planes || slot >= np) {
    if (threadIdx.x == 0) record_error(err, kErrBadIndex);
    pdl_wait();
    return;
  }
  int a = slot >= 0 ? lo.plane_adapter[p0 + slot] : -1;
  if (slot >= 0 && (a < 0 || a >= lo.adapters)) {
    if (threadIdx.x == 0) record_error(err, kErrBadIndex);
    a = -1;
  }
  float v = 0.f;
  if (a >= 0 && r < lo.rank) {
    const int nv = K / 8, chunk = (nv + ks - 1) / ks;
    const int v0 = share * chunk, v1 = min(nv, v0 + chunk);
    const uint4* xr = reinterpret_cast<const uint4*>(x + m * ldx);
    const uint4* ar = reinterpret_cast<const uint4*>(lo.a + ((size_t)a * lo.rank + r) * K);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    uint4 av[ROWS_VEC], xv[ROWS_VEC];
    for (int b = v0; b < v1; b += 32 * ROWS_VEC) {
#pragma unroll
      for (int i = 0; i < ROWS_VEC; ++i) {
        const int j = b + lane + 32 * i;
        av[i] = j < v1 ? ar[j] : make_uint4(0, 0, 0, 0);
      }
      if (b == v0) pdl_wait();
#pragma unroll
      for (int i = 0; i < ROWS_VEC; ++i) {
        const int j = b + lane + 32 * i;
        xv[i] = j < v1 ? ld_after_wait(xr + j) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < ROWS_VEC; ++i) {
        const uint32_t xu[4] = {xv[i].x, xv[i].y, xv[i].z, xv[i].w}, au[4] = {av[i].x, av[i].y, av[i].z, av[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = unpack_bf16x2(xu[j]), q = unpack_bf16x2(au[j]);
          s[j] = fmaf(p.x, q.x, s[j]);
          s[j] = fmaf(p.y, q.y, s[j]);
        }
      }
    }
    v = warp_sum((s[0] + s[1]) + (s[2] + s[3]));
  }
  pdl_wait();  // `low` may still be read by an earlier product
  if (ks > 1) {
    if (lane == 0) parts[warp] = v;
    __syncthreads();
    if (share != 0) return;
    v = parts[warp];
    for (int i = 1; i < ks; ++i) v += parts[warp + i];
  }
  if (r >= lo.rank) return;
  if (a >= 0) v *= lo.scale[a];
  const bf16 hi = __float2bfloat16(v);
  const float rest = v - __bfloat162float(hi);
  const bf16 rem = __float2bfloat16(rest == rest && fabsf(rest) < 3.0e38f ? rest : 0.f);  // none of an infinite value
  const bf16 zero = __float2bfloat16(0.f);
  const size_t to_lo = lo.to_lo();
  for (int j = lane; j < np; j += 32) {
    bf16* d = lo.low + ((size_t)(p0 + j) * lo.halves() * lo.tile_rows + m % lo.tile_rows) * lo.ld() + r;
    d[0] = j == slot ? hi : zero;
    d[to_lo] = j == slot ? rem : zero;
    if (lo.packed())
      for (int z = lo.rank; r + z < 32; z += lo.rank) d[z] = d[z + 32] = zero;
  }
}

typedef CUresult (*LowEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static LowEncodeFn low_encode_fn() {
  static const LowEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<LowEncodeFn>(p)
               : nullptr;
  }();
  return fn;
}

// bf16 tensor map of `rank` dimensions, 64 elements of the innermost in 128-byte swizzled rows
static bool low_tmap(CUtensorMap* tm, const void* ptr, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                     const cuuint32_t* box) {
  const cuuint32_t estr[3] = {1, 1, 1};
  const LowEncodeFn enc = low_encode_fn();
  return enc != nullptr &&
         enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace ll

using namespace ll;

// The few-row kernel's grid, and whether it is the one to take.
static dim3 rows_grid(int M, int K, int rank, int* ks) {
  *ks = 1;  // warps of a row and rank
  while (*ks < 8 && *ks * ROWS_VEC * 256 < K) *ks *= 2;
  return dim3(M, (rank + 8 / *ks - 1) / (8 / *ks));
}
static bool by_rows(int M, int K, const LLLora& lo) {
  int ks;
  const dim3 g = rows_grid(M, K, lo.rank, &ks);
  return (int64_t)g.x * g.y <= (lo.max_planes <= ROWS_PLANES ? ROWS_PLACES : (ks > 1 ? ROWS_LONG : ROWS_SHORT));
}

extern "C" int ll_lora_low(const bf16* x, int64_t ldx, int M, int K, const LLLora* lo, int* err, cudaStream_t stream) {
  if (M <= 0) return 0;
  if ((K % 8) || (ldx % 8) || lo->rank <= 0 || lo->rank > LL_LORA_MAX_RANK || (lo->rank % 8)) return -3;
  if (lo->max_planes < 1 || lo->max_planes > 65535) return -3;
  if (by_rows(M, K, *lo)) {
    int ks;
    const dim3 grid = rows_grid(M, K, lo->rank, &ks);
    const cudaError_t e =
        launch_pdl(lora_low_rows_kernel, grid, dim3(256), 0, stream, x, ldx, M, K, *lo, ks, err);
    return e == cudaSuccess ? 0 : -5;
  }
  LowShape shp;
  shp.npad = (lo->rank + 15) / 16 * 16;
  shp.x_rows = M < LOW_BM ? (M + 7) / 8 * 8 : LOW_BM;
  const int stage_bytes = (LOW_BM + shp.npad) * LOW_BK * 2;
  shp.stages = LOW_RING / stage_bytes < 8 ? LOW_RING / stage_bytes : 8;
  shp.tmem_cols = 32;
  while (shp.tmem_cols < shp.npad) shp.tmem_cols *= 2;
  shp.part_ld = lo->rank + 4;
  const int rows = M < LOW_BM ? M : LOW_BM;
  int smem = shp.stages * stage_bytes;
  if (smem < rows * shp.part_ld * 4) smem = rows * shp.part_ld * 4;
  smem += 1024;
  CUtensorMap tmX, tmA;
  {
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)M}, strides[1] = {(cuuint64_t)ldx * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)shp.x_rows};
    if (!low_tmap(&tmX, x, 2, dims, strides, box)) return -2;
  }
  {
    const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)lo->rank, (cuuint64_t)lo->adapters};
    const cuuint64_t strides[2] = {(cuuint64_t)K * 2, (cuuint64_t)K * 2 * lo->rank};
    const cuuint32_t box[3] = {64, (cuuint32_t)shp.npad, 1};
    if (!low_tmap(&tmA, lo->a, 3, dims, strides, box)) return -2;
  }
  // split K until two CTAs sit on every SM or a CTA is down to one k-block
  const int halves = lo->tile_rows / LOW_BM, num_kb = (K + LOW_BK - 1) / LOW_BK;
  int cs = 296 / (lo->max_planes * halves);
  cs = cs < 1 ? 1 : (cs > LOW_MAX_CLUSTER ? LOW_MAX_CLUSTER : cs);
  if (cs > num_kb) cs = num_kb;
  static unsigned long long done = 0;
  if (!smem_on_device(lora_low_kernel, 200 * 1024, done)) return -7;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs, halves, lo->max_planes);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cs, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, lora_low_kernel, tmX, tmA, M, K, *lo, shp, err) == cudaSuccess ? 0 : -5;
}

// Any number of rows, 128 a CTA.  N a multiple of 8 (32 with SwiGLU); out and
// bias on 8-byte boundaries.  K splits: as many CTAs (two a SM) as the feature
// tiles leave room for, up to a cluster of 6.
extern "C" int ll_lora_gemv(const bf16* x, int64_t ldx, const bf16* w, bf16* C, int64_t ldc, const bf16* bias, int M,
                            int N, int K, int swiglu, const LLLora* lo, int* err, cudaStream_t stream) {
  if (M <= 0 || lo->tile_rows != (M <= 128 ? 128 : 256)) return -3;
  if ((K % 8) || (N % 8) || (swiglu && (N % 32)) || (ldx % 8) || (ldc % 4)) return -3;
  const int bnx = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
  GemvMaps tm;
  const cuuint32_t box2w[2] = {64, 128}, box2x[2] = {64, (cuuint32_t)bnx}, box3[3] = {64, 128, 1};
  const cuuint64_t dw[2] = {(cuuint64_t)K, (cuuint64_t)N}, sw[1] = {(cuuint64_t)K * 2};
  const cuuint64_t dx[2] = {(cuuint64_t)K, (cuuint64_t)M}, sx[1] = {(cuuint64_t)ldx * 2};
  const cuuint64_t dl[2] = {(cuuint64_t)lo->ld(), (cuuint64_t)lo->max_planes * lo->halves() * lo->tile_rows};
  const cuuint64_t sl[1] = {(cuuint64_t)lo->ld() * 2};
  const cuuint64_t db[3] = {(cuuint64_t)lo->rank, (cuuint64_t)N, (cuuint64_t)lo->adapters};
  const cuuint64_t sb[2] = {(cuuint64_t)lo->rank * 2, (cuuint64_t)lo->rank * 2 * N};
  if (!low_tmap(&tm.w, w, 2, dw, sw, box2w) || !low_tmap(&tm.x, x, 2, dx, sx, box2x) ||
      !low_tmap(&tm.low, lo->low, 2, dl, sl, box2x) || !low_tmap(&tm.b, lo->b, 3, db, sb, box3))
    return -2;
  const int ntiles = (N + 127) / 128, mtiles = (M + bnx - 1) / bnx, num_kb = (K + LOW_BK - 1) / LOW_BK;
  if (ntiles > 65535 || mtiles > 65535) return -3;
  int cs = GEMV_PLACES / (ntiles * mtiles);
  if (cs > GEMV_MAX_CLUSTER) cs = GEMV_MAX_CLUSTER;
  // at least two k-blocks a CTA, the adapters' (at most that many) among them
  const int64_t blocks = num_kb + (int64_t)(mtiles == 1 ? lo->max_planes : 1) * lo->steps();
  if (cs > (blocks + 1) / 2) cs = (int)((blocks + 1) / 2);
  if (cs < 1) cs = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs, ntiles, mtiles);
  cfg.blockDim = dim3(192);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cs, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const bool x_ready = !by_rows(M, K, *lo);
  cudaError_t e;
#define LL_GEMV(BNX_, SW_)                                                                      \
  do {                                                                                          \
    auto kern = lora_gemv_kernel<BNX_, SW_>;                                                    \
    static unsigned long long done = 0;                                                         \
    if (!smem_on_device(kern, GemvCfg<BNX_>::SMEM, done)) return -7;                            \
    cfg.dynamicSmemBytes = GemvCfg<BNX_>::SMEM;                                                 \
    e = cudaLaunchKernelEx(&cfg, kern, tm, C, ldc, bias, M, N, K, *lo, x_ready, err);                    \
  } while (0)
#define LL_GEMV_SW(BNX_)              \
  do {                                \
    if (swiglu) LL_GEMV(BNX_, true);  \
    else LL_GEMV(BNX_, false);        \
  } while (0)
  switch (bnx) {
    case 16: LL_GEMV_SW(16); break;
    case 32: LL_GEMV_SW(32); break;
    case 64: LL_GEMV_SW(64); break;
    default: LL_GEMV_SW(128); break;
  }
#undef LL_GEMV_SW
#undef LL_GEMV
  return e == cudaSuccess ? 0 : -5;
}
