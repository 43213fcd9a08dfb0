// Rows to 8 bits: e4m3 values with one fp32 scale a row,
//
//   scale = max(amax |y| / 448, 2^-126),  q = e4m3(y * (1 / scale)),
//
// of y = x, of y = rmsnorm(x) w, or of y = rmsnorm(x + residual) w with the sum
// stored as well.  448 is e4m3's largest number.  The floor 2^-126 keeps the
// scale and its reciprocal normal numbers: a row of zeros has zeros and that
// scale.  y is never rounded to bf16 on the way: its one rounding is e4m3's.  A
// row with an infinity or a NaN has the scale NaN (its magnitudes are compared
// as integers, where a NaN is the largest), so every product of that row is NaN.
//
// Bound by memory: each value is read once, kept in registers through the
// reductions, and written as one byte.  In a graph, of bytes that cannot be saved at
// 6551 GB/s: quantising 2048 x 18944 19.6 us of 17.8, the norm with the residual's
// addition of 5087 x 3584 20.3 of 19.5 (alone 13.7 of 8.4: two reductions and the
// weight between its loads and its stores); a few rows 1.1 to 2 us.  Persistent CTAs
// that fetch rows ahead into shared memory by bulk copies were slower (9.5 -> 10.4,
// 13.8 -> 14.9, 21.0 -> 23.4 us for 5087 x 3584), and so was one reduction for both the
// squares and the largest |x w| (13.7 -> 15.5: the weight is read twice).
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "q8.h"

namespace ll {

constexpr float kE4m3Max = 448.f;
constexpr float kQ8MinScale = 1.17549435e-38f;  // 2^-126

enum Q8Mode : int { kQ8Quantize = 0, kQ8Norm = 1, kQ8AddNorm = 2 };

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// The larger of two magnitudes, NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum, and largest magnitude (as an integer, where a NaN is the largest), over the
// row's threads: a warp's (WARP), else the CTA's.  The order is fixed, so a row's
// bits depend on K and the number of rows alone, never on other rows.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = warp_sum(lane < (blockDim.x >> 5) ? red[lane] : 0.f);
    __syncthreads();  // free again
  }
  return v;
}
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[warp] = __uint_as_float(v);
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < (blockDim.x >> 5) ? __float_as_uint(red[lane]) : 0u);
  }
  return v;
}

// WARP: a row a warp; else a row a CTA.  VPT vectors of 8 values a thread.
template <int VPT, int MODE, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
    q8_rows_kernel(const __grid_constant__ LLQ8Rows p) {
  __shared__ float red[32];
  pdl_trigger();
  pdl_wait();
  const int tid = WARP ? (threadIdx.x & 31) : threadIdx.x, step = WARP ? 32 : blockDim.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const int nvec = p.K / 8;
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
  // the row in fp32; a thread's vectors lie `step` apart
  float v[VPT][8];
  uint4 in[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + i * step;
    in[i] = j < nvec ? xr[j] : make_uint4(0, 0, 0, 0);
  }
  if constexpr (MODE == kQ8AddNorm) {
    const uint4* rr = reinterpret_cast<const uint4*>(p.residual + row * p.ldr);
    uint4* sr = reinterpret_cast<uint4*>(p.sum + row * p.lds);
    uint4 add[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = tid + i * step;
      add[i] = j < nvec ? rr[j] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t a[4] = {in[i].x, in[i].y, in[i].z, in[i].w}, b[4] = {add[i].x, add[i].y, add[i].z, add[i].w};
      uint32_t o[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 fa = unpack_bf16x2(a[c]), fb = unpack_bf16x2(b[c]);
        v[i][2 * c] = fa.x + fb.x;
        v[i][2 * c + 1] = fa.y + fb.y;
        o[c] = pack_bf16x2(v[i][2 * c], v[i][2 * c + 1]);
      }
      const int j = tid + i * step;
      if (j < nvec) sr[j] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t a[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 fa = unpack_bf16x2(a[c]);
        v[i][2 * c] = fa.x;
        v[i][2 * c + 1] = fa.y;
      }
    }
  }
  if constexpr (MODE != kQ8Quantize) {
    // few rows (up to two vectors a thread) have the weight loaded beside them: one
    // row of 3584 1.45 us for 1.64; for many it costs registers, and with them CTAs a
    // SM: 5087 rows 17.8 us for 13.7
    constexpr bool EARLY = VPT <= 2;
    const uint4* wr = reinterpret_cast<const uint4*>(p.w);
    uint4 early[VPT];
    auto load_w = [&](int i) {
      const int j = tid + i * step;
      return j < nvec ? wr[j] : make_uint4(0, 0, 0, 0);
    };
    if constexpr (EARLY) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) early[i] = load_w(i);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int c = 0; c < 8; ++c) ss = fmaf(v[i][c], v[i][c], ss);
    ss = row_sum<WARP>(ss, red);
    float rstd = rsqrtf(ss / (float)p.K + p.eps);
    if (!(ss < INFINITY)) {  // squares past fp32's range, or a value that is not finite: the same, 2^-80 as large
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float t = v[i][c] * 0x1p-80f;
          ss = fmaf(t, t, ss);
        }
      ss = row_sum<WARP>(ss, red);
      rstd = rsqrtf(ss / (float)p.K) * 0x1p-80f;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      uint4 w;
      if constexpr (EARLY) w = early[i];
      else w = load_w(i);
      const uint32_t wu[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 fw = unpack_bf16x2(wu[c]);
        v[i][2 * c] = v[i][2 * c] * rstd * fw.x;
        v[i][2 * c + 1] = v[i][2 * c + 1] * rstd * fw.y;
      }
    }
  }
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) big = max_nan(big, fabsf(v[i][c]));
  const uint32_t top = row_max<WARP>(__float_as_uint(big), red);
  const float amax = __uint_as_float(top);
  const float scale = amax < INFINITY ? fmaxf(amax / kE4m3Max, kQ8MinScale) : __uint_as_float(0x7fffffffu);
  const float inv = 1.f / scale;
  uint2* qr = reinterpret_cast<uint2*>(p.q + row * p.ldq);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + i * step;
    if (j < nvec)
      qr[j] = make_uint2(e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                         e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
  }
  if (tid == 0) p.scale[row] = scale;
}

template <int VPT, bool WARP>
static cudaError_t q8_rows_launch(const LLQ8Rows& p, int grid, int threads, cudaStream_t stream) {
  if (p.w == nullptr)
    return launch_pdl(q8_rows_kernel<VPT, kQ8Quantize, WARP>, dim3(grid), dim3(threads), 0, stream, p);
  if (p.residual == nullptr)
    return launch_pdl(q8_rows_kernel<VPT, kQ8Norm, WARP>, dim3(grid), dim3(threads), 0, stream, p);
  return launch_pdl(q8_rows_kernel<VPT, kQ8AddNorm, WARP>, dim3(grid), dim3(threads), 0, stream, p);
}

}  // namespace ll

using namespace ll;

extern "C" int ll_q8_rows(const LLQ8Rows* p, cudaStream_t stream) {
  if (p->rows <= 0) return 0;
  if (p->K <= 0 || (p->K % 16) || p->K > LL_Q8_MAX_K) return -3;
  const int nvec = p->K / 8;
  // A warp holds a row of up to 1024 values.  Longer ones are a CTA's: two vectors
  // a thread while every row has a place at once, four for more rows, so that more
  // bytes are on their way (us, 1 / 2 / 4 vectors: quantising 300 x 3584 1.8 / 2.2 /
  // 2.3, 5087 x 3584 13.9 / 9.7 / 10.1; with the norm 2.6 / 2.9 / 4.0 and 19.8 /
  // 15.0 / 14.2; a warp to a row there 15.1 and 22.0).
  const int vpt = nvec <= 32 ? 1 : (nvec <= 64 ? 2 : (nvec <= 128 || nvec > 2048 || p->rows > 600 ? 4 : 2));
  cudaError_t e;
  if (nvec <= 128) {
    const int warps = p->rows < 8 ? p->rows : 8, grid = (p->rows + warps - 1) / warps;
    if (vpt == 1) e = q8_rows_launch<1, true>(*p, grid, 32 * warps, stream);
    else if (vpt == 2) e = q8_rows_launch<2, true>(*p, grid, 32 * warps, stream);
    else e = q8_rows_launch<4, true>(*p, grid, 32 * warps, stream);
  } else {
    const int threads = ((nvec + vpt - 1) / vpt + 31) / 32 * 32;
    if (vpt == 2) e = q8_rows_launch<2, false>(*p, p->rows, threads, stream);
    else e = q8_rows_launch<4, false>(*p, p->rows, threads, stream);
  }
  return e == cudaSuccess ? 0 : -5;
}
