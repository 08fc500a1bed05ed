// Low-rank adapters of many requests beside a projection: parameters and launches of lora.cu.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace aipu {

enum AdType : int { AD_BF16 = 0, AD_F16 = 1 };

struct LoraParams {
  const void* a;         // [L, R, K] bf16 or fp16
  const void* b;         // [L, N, R]
  const float* scale;    // [L] or nullptr (1)
  const int32_t* ranks;  // [L] or nullptr (R)
  int adtype;            // AdType
  int L, R, K, N, M;
  const int32_t* ids;    // [M]
  const uint16_t* x;     // bf16 rows
  int64_t ldx;           // elements
  const void* y;         // rows added to: bf16 or fp32
  int64_t ldy;
  void* out;             // bf16, or fp32 when y is
  int64_t ldo;
  int y_f32, out_f32;
  int* status;           // device status word (nullable)
  // set by the launch
  int32_t* perm;         // rows ordered by adapter
  int4* tiles;           // {adapter or -1, first position in perm, rows, 0}
  int32_t* n_tiles;
  int skip_plain;        // 1: in-place, rows without an adapter are not touched
  int wa, wx, wb;        // widest aligned load of A rows, x rows, B rows (elements: 8, 2 or 1)
  int vy;                // 1: 16-byte loads and stores of y and out
  int wait_y;            // 1: y comes from the kernel launched just before (programmatic dependent launch)
};

// bytes of the row plan (0 when M rows need none)
size_t lora_plan_bytes(int64_t M, int64_t L);
// the plan of p.ids in `plan` (sets p's pointers to it; nothing to do for few rows)
int lora_plan_launch(LoraParams& p, void* plan, cudaStream_t s, bool pdl);
int lora_launch(LoraParams p, int num_sms, cudaStream_t s, bool pdl);

}  // namespace aipu
