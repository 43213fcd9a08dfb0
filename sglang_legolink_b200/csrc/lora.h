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
  __nv_bfloat16* low;       // [max_planes, 2 (hi, lo), tile_rows, rank]
  int adapters, rank, tiles, tile_rows, max_planes;
};

constexpr int LL_LORA_MAX_RANK = 256;
