// Matrices in 8 bits: e4m3 values with one fp32 scale a row (q8_rows.cu makes
// them, gemm_q8.cu multiplies two of them).
#pragma once

#include <stdint.h>

#include <cuda_bf16.h>

constexpr int LL_Q8_MAX_K = 32768;  // longest row that q8_rows.cu takes

// One row of y to 8 bits: y = x, or its RMSNorm (w), or that of x + residual.
struct LLQ8Rows {
  const __nv_bfloat16* x;         // [rows, K], rows ldx elements apart
  const __nv_bfloat16* residual;  // [rows, K] or null
  __nv_bfloat16* sum;             // [rows, K]: x + residual; may be residual itself
  const __nv_bfloat16* w;         // [K] or null: no norm
  uint8_t* q;                     // [rows, K]
  float* scale;                   // [rows]
  int64_t ldx, ldr, lds, ldq;
  int rows, K;
  float eps;
};

// C = act(xs ws (X . W^T) + bias) + residual
struct LLQ8Gemm {
  const uint8_t* x;   // [M, K] e4m3
  const float* xs;    // [M]
  const uint8_t* w;   // [N, K] e4m3
  const float* ws;    // [N]
  const __nv_bfloat16* bias;      // [N] or null
  const __nv_bfloat16* residual;  // [M, N] ([M, N / 2] with SwiGLU) or null; may be C itself
  __nv_bfloat16* C;
  int64_t ldx, ldw, ldr, ldc;
  int M, N, K;
};
