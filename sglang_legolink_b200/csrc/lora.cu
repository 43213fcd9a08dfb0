// The low-rank half of the adapter projection (lora.h): low = scale x A^T.
#include <cuda_runtime.h>

#include "common.cuh"
#include "lora.h"

namespace ll {

// One warp per (row, rank): a dot product over K.  The row's value goes to
// the plane of its adapter, zeros to the other planes of its tile.
__global__ void __launch_bounds__(256) lora_low_rows_kernel(const bf16* __restrict__ x, int64_t ldx, int M, int K,
                                                            const LLLora lo, int* err) {
  pdl_trigger();
  const int m = blockIdx.x, r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < lo.num_tickets; i += blockDim.x) lo.tickets[i] = 0;
  if (r >= lo.rank) return;
  const int t = m / lo.tile_rows;
  const int p0 = lo.tile_ptr[t], np = lo.tile_ptr[t + 1] - p0, slot = lo.row_slot[m];
  if (p0 < 0 || np < 0 || p0 + np > lo.max_planes || slot >= np) {
    if (lane == 0) record_error(err, kErrBadIndex);
    return;
  }
  float v = 0.f;
  if (slot >= 0) {
    const int a = lo.plane_adapter[p0 + slot];
    if (a < 0 || a >= lo.adapters) {
      if (lane == 0) record_error(err, kErrBadIndex);
    } else {
      const uint4* xr = reinterpret_cast<const uint4*>(x + m * ldx);
      const uint4* ar = reinterpret_cast<const uint4*>(lo.a + ((size_t)a * lo.rank + r) * K);
      float s = 0.f;
      for (int i = lane; i < K / 8; i += 32) {
        const uint4 xv = xr[i], av = ar[i];
        const uint32_t* xu = reinterpret_cast<const uint32_t*>(&xv);
        const uint32_t* au = reinterpret_cast<const uint32_t*>(&av);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = unpack_bf16x2(xu[j]), q = unpack_bf16x2(au[j]);
          s += p.x * q.x;
          s += p.y * q.y;
        }
      }
      v = warp_sum(s) * lo.scale[a];
    }
  }
  // bf16: the second product's operands are bf16; the rounding moves the
  // adapter's term by 2^-9 of itself per rank at most
  for (int j = lane; j < np; j += 32)
    lo.low[((size_t)(p0 + j) * lo.tile_rows + m % lo.tile_rows) * lo.rank + r] = __float2bfloat16(j == slot ? v : 0.f);
}

}  // namespace ll

using namespace ll;

extern "C" int ll_lora_low(const bf16* x, int64_t ldx, int M, int K, const LLLora* lo, int* err, cudaStream_t stream) {
  if (M <= 0) return 0;
  if ((K % 8) || (ldx % 8) || lo->rank <= 0 || lo->rank > LL_LORA_MAX_RANK || (lo->rank % 8)) return -3;
  return launch_pdl(lora_low_rows_kernel, dim3(M, (lo->rank + 7) / 8), dim3(256), 0, stream, x, ldx, M, K, *lo, err) ==
                 cudaSuccess
             ? 0
             : -5;
}
