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
// reductions, and written as one byte.  In a graph over rows that L2 does not hold, of
// bytes that cannot be saved at 6551 GB/s: quantising 2048 x 18944 18.4 us of 17.8, the
// norm with the residual's addition of 5087 x 3584 21.4 of 19.5; a few rows 1.2 to 2 us.
// The norm alone, 13.9 us of 8.4, issues an instruction in 65 % of the cycles (with the
// addition 63 %, quantising 53 %), with products two and maxima three values an
// instruction (one each issued in 70 %, and 5087 x 18944 took 98 us for 60).
// Persistent CTAs that fetch rows ahead into shared memory by bulk copies were slower
// (quantising 5087 x 3584 10.4 us for 9.5, the norm 14.9 for 13.8), and so was one
// reduction for both the squares and the largest |x w| (15.5 for 13.7: the weight is
// read twice).
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

// The largest of three, NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two products, or two products and sums, an instruction: these kernels are bound by
// their instructions as soon as their bytes are on their way.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 a, b, r;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " mul.rn.f32x2 r, a, b;\n mov.b64 {%0, %1}, r;}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 a, b, c, r;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 r, a, b, c;\n mov.b64 {%0, %1}, r;}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
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

// WARP: a row a warp; else a row a CTA.  VPT vectors of 8 values a thread.  PACKED
// (quantising, long rows): they stay as they were loaded, so that more of the large CTAs
// fit a SM: 3000 x 25600 36.0 us for 47; short rows have places enough, and unpacking
// them behind the maximum costs 8192 x 2048 10.1 for 9.0.
// LOW: an eps below 2^-80, beside which squares below fp32's range count.  A kernel of its
// own, since its registers cost the norm 2 to 16 % (5087 x 3584 14.2 us for 13.9, 5087 x
// 1024 6.3 for 5.4).
template <int VPT, int MODE, bool WARP, bool PACKED, bool LOW>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
    q8_rows_kernel(const __grid_constant__ LLQ8Rows p) {
  __shared__ float red[3][32];
  pdl_trigger();
  pdl_wait();
  const int tid = WARP ? (threadIdx.x & 31) : threadIdx.x, step = WARP ? 32 : blockDim.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const int nvec = p.K / 8;
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
  // a thread's vectors lie `step` apart
  uint4 in[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + i * step;
    in[i] = j < nvec ? xr[j] : make_uint4(0, 0, 0, 0);
  }
  uint32_t top = 0;  // the largest magnitude's bits
  float up = 1.f;    // what is held of y is 1 / up of it
  float2 v[PACKED ? 1 : VPT][4];  // the row in fp32
  if constexpr (MODE == kQ8Quantize) {
    if constexpr (PACKED) {
      uint32_t big = 0;  // of pairs, as integers
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        constexpr uint32_t MAG = 0x7fff7fffu;
        big = __vimax3_u16x2(big, in[i].x & MAG, in[i].y & MAG);
        big = __vimax3_u16x2(big, in[i].z & MAG, in[i].w & MAG);
      }
      top = max(big << 16, big & 0xffff0000u);
    } else {
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t a[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v[i][c] = unpack_bf16x2(a[c]);
          big = max_nan(big, fabsf(v[i][c].x), fabsf(v[i][c].y));
        }
      }
      top = __float_as_uint(big);
    }
  } else {
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
          v[i][c] = make_float2(fa.x + fb.x, fa.y + fb.y);
          o[c] = pack_bf16x2(v[i][c].x, v[i][c].y);
        }
        const int j = tid + i * step;
        if (j < nvec) sr[j] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t a[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i][c] = unpack_bf16x2(a[c]);
      }
    }
    // few rows (up to two vectors a thread) have the weight loaded beside them: one
    // row of 3584 1.44 us for 1.64; for many it costs registers, and with them CTAs a
    // SM: 5087 rows 17.5 us for 12.7
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
    float2 sq = make_float2(0.f, 0.f), sq2 = sq;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        sq = fma2(v[i][c], v[i][c], sq);
        sq2 = fma2(v[i][c + 1], v[i][c + 1], sq2);
      }
    float ss = row_sum<WARP>((sq.x + sq.y) + (sq2.x + sq2.y), red[0]);
    float rstd = rsqrtf(ss / (float)p.K + p.eps);
    // squares past fp32's range, or a value that is not finite: the same, 2^-80 as large;
    // squares below it: 2^80 as large
    if (!(ss < INFINITY) || (LOW && ss < 0x1p-80f)) {
      const float f = LOW && ss < 1.f ? 0x1p80f : 0x1p-80f;
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float a = v[i][c].x * f, b = v[i][c].y * f;
          ss = fmaf(a, a, fmaf(b, b, ss));
        }
      ss = row_sum<WARP>(ss, red[2]);
      rstd = rsqrtf(ss / (float)p.K + (LOW ? p.eps * f * f : 0.f));
      if (LOW && rstd * f == INFINITY) up = f;  // itself past the range: until the row is quantised
      else rstd *= f;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      uint4 w;
      if constexpr (EARLY) w = early[i];
      else w = load_w(i);
      const uint32_t wu[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) v[i][c] = mul2(mul2(v[i][c], make_float2(rstd, rstd)), unpack_bf16x2(wu[c]));
    }
    float big = 0.f, big2 = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        big = max_nan(big, fabsf(v[i][c].x), fabsf(v[i][c].y));
        big2 = max_nan(big2, fabsf(v[i][c + 1].x), fabsf(v[i][c + 1].y));
      }
    top = __float_as_uint(max_nan(big, big2, 0.f));
  }
  const float amax = __uint_as_float(row_max<WARP>(top, red[1])) * (LOW ? up : 1.f);
  const float scale = amax < INFINITY ? fmaxf(amax / kE4m3Max, kQ8MinScale) : __uint_as_float(0x7fffffffu);
  float inv = 1.f / scale;
  if (LOW && up > 1.f) inv = inv * up == INFINITY ? 0x1p127f : inv * up;  // zeros stay zeros
  const float2 inv2 = make_float2(inv, inv);
  uint2* qr = reinterpret_cast<uint2*>(p.q + row * p.ldq);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float2 y[4];
    const uint32_t a[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = mul2(PACKED ? unpack_bf16x2(a[c]) : v[PACKED ? 0 : i][c], inv2);
    const int j = tid + i * step;
    if (j < nvec) qr[j] = make_uint2(e4m3x4(y[0].x, y[0].y, y[1].x, y[1].y), e4m3x4(y[2].x, y[2].y, y[3].x, y[3].y));
  }
  if (tid == 0) p.scale[row] = scale;
}

template <int VPT, bool WARP>
static cudaError_t q8_rows_launch(const LLQ8Rows& p, int grid, int threads, cudaStream_t stream) {
  const auto run = [&](auto kernel) { return launch_pdl(kernel, dim3(grid), dim3(threads), 0, stream, p); };
  if (p.w == nullptr) {
    if constexpr (!WARP && VPT == 4) {
      if (threads > 256) return run(q8_rows_kernel<VPT, kQ8Quantize, WARP, true, false>);
    }
    return run(q8_rows_kernel<VPT, kQ8Quantize, WARP, false, false>);
  }
  const bool low = p.eps < 0x1p-80f;
  if (p.residual == nullptr)
    return low ? run(q8_rows_kernel<VPT, kQ8Norm, WARP, false, true>)
               : run(q8_rows_kernel<VPT, kQ8Norm, WARP, false, false>);
  return low ? run(q8_rows_kernel<VPT, kQ8AddNorm, WARP, false, true>)
             : run(q8_rows_kernel<VPT, kQ8AddNorm, WARP, false, false>);
}

}  // namespace ll

using namespace ll;

extern "C" int ll_q8_rows(const LLQ8Rows* p, cudaStream_t stream) {
  if (p->rows <= 0) return 0;
  if (p->K <= 0 || (p->K % 16) || p->K > LL_Q8_MAX_K) return -3;
  const int nvec = p->K / 8;
  // A warp holds a row of up to 1024 values.  Longer ones are a CTA's: two vectors
  // a thread, four where the rows do not all have places at once (us, 2 / 4 vectors, 3584
  // values: quantising 600 rows 1.93 / 2.14, 1500 3.36 / 3.32, 5087 9.5 / 9.4; the norm
  // 600 2.50 / 3.91, 1200 4.24 / 4.06, 5087 15.1 / 12.6; with the addition 600 3.86 /
  // 4.47, 1000 6.40 / 6.01.  One vector a thread is slower but for some 300 to 450 rows.)
  const int64_t many = p->w == nullptr ? 600000 : (p->residual == nullptr ? 480000 : 380000);  // vectors
  const bool four = nvec <= 128 ? nvec > 64 : nvec > 2048 || p->rows * (int64_t)nvec > many;
  const int vpt = nvec <= 32 ? 1 : (four ? 4 : 2);
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
