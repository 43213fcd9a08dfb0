// Low-rank adapters (LoRA) of many requests beside one shared projection:
//
//   y[m] = x[m] W^T + bias + scale[a] (x[m] A[a]^T) B[a]^T,   a = adapter of row m
//
// in two launches (lora.cu, gemm_tcgen05.cu):
//
//   1. low[plane][row] = scale[a] x[row] A[a]^T, one plane per adapter that a
//      tile of rows uses, with zeros in the rows of other adapters; each value
//      as the sum of two bf16, hi and lo;
//   2. the shared product, whose k-loop goes on over the planes:
//      [x | hi_0 | lo_0 | hi_1 | ...] . [W | B[a_0] | B[a_0] | B[a_1] | ...]^T.
//
// A k-block is 64 columns.  Up to rank 32 a plane's hi and lo are the halves of
// one block (low's rows are 64 wide, zero between), and the last two of the
// block's four MMA steps read B's first 32 columns once more.  Else hi and lo
// are blocks of their own.  In a graph, 61 rows of 32 adapters, rank 16, K =
// 8192, N = 5120: 26.8 us packed, 28.4 not; 16 rows of 8, rank 32, K = 3584, N =
// 37888 with SwiGLU: 48.4 and 51.0.
//
// Rows are cut into tiles of `tile_rows`; the planes of tile t are
// [tile_ptr[t], tile_ptr[t + 1]) and plane_adapter names their adapters.
#pragma once

#include <stdint.h>

#include <cuda_bf16.h>

struct LLLora {
  const __nv_bfloat16* a;   // [adapters, rank, K]
  const __nv_bfloat16* b;   // [adapters, N, rank]
  const float* scale;       // [adapters]
  const int* row_slot;      // [M] plane of the row within its tile, -1: no adapter
  const int* tile_ptr;      // [tiles + 1]
  const int* plane_adapter; // [max_planes]
  const int* plane_tile;    // [max_planes]
  __nv_bfloat16* low;       // [max_planes, 2 (hi, lo), tile_rows, rank]; packed [max_planes, tile_rows, 64]
  int adapters, rank, tiles, tile_rows, max_planes;

#ifdef __CUDACC__
#define LL_HD __host__ __device__
#else
#define LL_HD
#endif
  LL_HD bool packed() const { return rank <= 32; }
  LL_HD int halves() const { return packed() ? 1 : 2; }  // blocks of tile_rows rows in low per plane
  LL_HD int ld() const { return packed() ? 64 : rank; }  // of a row of low
  LL_HD int steps() const { return packed() ? 1 : 2 * ((rank + 63) / 64); }  // k-blocks of a plane
  LL_HD long long to_lo() const { return packed() ? 32 : (long long)tile_rows * rank; }  // from hi
#undef LL_HD
};

constexpr int LL_LORA_MAX_RANK = 256;
