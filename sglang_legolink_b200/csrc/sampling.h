// Arguments of the sampling kernel (sampling.cu).
#pragma once

#include <stdint.h>

constexpr int LL_SAMPLE_MAX_VOCAB = 1 << 19;

struct LLSample {
  const void* logits;        // [B, V], bf16 or fp32, rows `stride` elements apart
  int64_t stride;
  const double* u;           // [B] in [0, 1)
  const float* temperature;  // [B] or null (1); <= 0: the largest logit
  const int* top_k;          // [B] or null; <= 0 or >= V: all
  const float* top_p;        // [B] or null; >= 1: all
  const float* min_p;        // [B] or null; <= 0: all
  int* out;                  // [B] token, -1 where no logit is above -inf
  float* logprob;            // [B] or null: log of the token's share of what is kept
  int B, V, fp32;
};
