// Controls of many requests on their logits: parameters and launch of logits.cu.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace aipu {

struct LogitParams {
  const void* logits;         // [M, V] bf16 or fp32
  int64_t ld;                 // elements between rows
  int f32;                    // 1: fp32 logits
  int M, V;
  const int32_t* tokens;      // contexts, back to back or overlapping
  int64_t n_tokens;
  const int64_t* spans;       // [M, 3] begin, first generated, end (nullable)
  const float* penalties;     // [M, 3] repetition, presence, frequency (with spans)
  const int64_t* bias_begin;  // [M + 1] (nullable)
  const int32_t* bias_ids;
  const float* bias_vals;
  int64_t n_bias;
  const uint32_t* mask;       // [n_masks, ceil(V / 32)] bit v % 32 of word v / 32: token v is allowed (nullable)
  const int32_t* mask_rows;   // [M] mask of each row, negative: none
  int n_masks;
  float* out;                 // [M, V] fp32 (nullable)
  int64_t ldo;
  int32_t* token;             // [M] greedy token (nullable)
  int* status;
  int blocks;                 // set by the launch: blocks (256 bf16 or 128 fp32 tokens) of one CTA and window
};

int logits_launch(LogitParams p, int num_sms, cudaStream_t s, bool pdl);

}  // namespace aipu
