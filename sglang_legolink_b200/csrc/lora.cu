// The low-rank half of the adapter projection (lora.h): low = scale x A^T.
//
// Per plane (a row tile's adapter) and 128-row half of the tile: a 128 x rank
// product over K on tcgen05, x rows on the M side and the adapter's ranks on
// the N side, K split over the CTAs of a cluster.  It is bound by reading x
// (K / rank is large: 36 MB of x against 0.3 MB of A at 5087 rows x 3584,
// rank 48), so what counts is bytes in flight: the cluster split puts up to
// two CTAs with a ~96 KB ring on every SM whatever the number of row tiles.
// The CTAs' fp32 partials meet in distributed shared memory and are summed in
// CTA order, so a row's bits do not depend on timing.
//
// low is kept as two bf16 planes, hi = bf16(v) and lo = bf16(v - hi): the
// product that reads them takes bf16 operands, and one bf16 would put 2^-9 of
// every low-rank value into the result, as much again as rounding the result
// itself; hi + lo holds 16 bits and costs one more k-block a plane.
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
  pdl_trigger();

  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && lo.num_tickets > 0) {
    pdl_wait();  // the previous kernel may be the product of an earlier call on this scratch
    for (int i = tid; i < lo.num_tickets; i += blockDim.x) lo.tickets[i] = 0;
  }

  // which rows and which adapter: the same for every CTA of the cluster
  const int planes = lo.tile_ptr[lo.tiles];
  if (plane >= planes) return;
  const int t = lo.plane_tile[plane], adapter = lo.plane_adapter[plane];
  const int m0 = t * lo.tile_rows + blockIdx.y * LOW_BM;
  if (planes > lo.max_planes || t < 0 || t >= lo.tiles || adapter < 0 || adapter >= lo.adapters) {
    if (tid == 0) record_error(err, kErrBadIndex);
    return;
  }
  if (m0 >= M) return;
  const int rows = min(LOW_BM, M - m0), slot = plane - lo.tile_ptr[t];
  const bool mine = tid < rows && lo.row_slot[m0 + tid] == slot;
  bf16* low = lo.low + ((size_t)plane * 2 * lo.tile_rows + blockIdx.y * LOW_BM) * lo.rank;
  const size_t lo_plane = (size_t)lo.tile_rows * lo.rank;
  const int groups = lo.rank / 4;  // 4 ranks a thread
  if (!__syncthreads_or(mine)) {   // no row of this half uses the adapter
    pdl_wait();
    for (int i = crank * 128 + tid; i < rows * groups; i += cs * 128) {
      bf16* d = low + (size_t)(i / groups) * lo.rank + 4 * (i % groups);
      *reinterpret_cast<uint2*>(d) = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(d + lo_plane) = make_uint2(0, 0);
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
        if (c + i < lo.rank)
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
      if (lo.row_slot[m0 + row] == slot) {
        for (int r = 0; r < cs; ++r) {
          const float4 p = ld_cluster_f32x4(low_mapa(base + (uint32_t)(row * shp.part_ld + 4 * g) * 4, r));
          v.x += p.x;
          v.y += p.y;
          v.z += p.z;
          v.w += p.w;
        }
        v.x *= scale;
        v.y *= scale;
        v.z *= scale;
        v.w *= scale;
      }
      const uint32_t h0 = pack_bf16x2(v.x, v.y), h1 = pack_bf16x2(v.z, v.w);
      const float2 f0 = unpack_bf16x2(h0), f1 = unpack_bf16x2(h1);
      bf16* d = low + (size_t)row * lo.rank + 4 * g;
      *reinterpret_cast<uint2*>(d) = make_uint2(h0, h1);
      // an infinite value has no remainder
      const float r0 = v.x - f0.x, r1 = v.y - f0.y, r2 = v.z - f1.x, r3 = v.w - f1.y;
      auto rest = [](float r) { return r == r && fabsf(r) < 3.0e38f ? r : 0.f; };
      *reinterpret_cast<uint2*>(d + lo_plane) =
          make_uint2(pack_bf16x2(rest(r0), rest(r1)), pack_bf16x2(rest(r2), rest(r3)));
    }
  }
  low_cluster_sync();  // the partials live until every CTA has read them
  if (warp == 1) tmem_dealloc(tmem, shp.tmem_cols);
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

extern "C" int ll_lora_low(const bf16* x, int64_t ldx, int M, int K, const LLLora* lo, int* err, cudaStream_t stream) {
  if (M <= 0) return 0;
  if ((K % 8) || (ldx % 8) || lo->rank <= 0 || lo->rank > LL_LORA_MAX_RANK || (lo->rank % 8)) return -3;
  if (lo->max_planes < 1 || lo->max_planes > 65535) return -3;
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
