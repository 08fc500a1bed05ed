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
  int yparts;            // shares of fp32 y to be summed, M * ldy elements apart (0: one; more need aligned, padded rows)
  int y_cols;            // columns of y that may be read (0: N; more where its rows are padded)
  int* status;           // device status word (nullable)
  int wait_y;            // 1: y comes from the kernel launched just before lora_finish's (programmatic launch)
  // set by lora_begin
  int32_t* perm;         // rows ordered by adapter (more rows than one launch takes: tiles is set)
  int4* tiles;           // {adapter or -1, first position in perm, rows, the adapter's rank}
  int32_t* n_tiles;
  float* sums;           // [ksplit][M][rp] shares of h by position
  int ksplit, nsplit;    // shares of K and of N
  int rp;                // padded rank: 16, 32, 64 or 128
  int skip_plain;        // 1: in-place, rows without an adapter are not touched
  int wa, wx, wb;        // widest aligned load of A rows, x rows, B rows (elements: 8, 2 or 1)
  int vy;                // columns of y that may be read in 16-byte pieces (0: rows not aligned)
  int vo;                // 2: 16-byte stores of out, 1: 4-byte stores
};

// bytes of the scratch of M rows (0 when the one launch takes them)
size_t lora_plan_bytes(int64_t M, int64_t L, int64_t R);
// what does not need y: the row plan and the first product of many rows. Then the rest.
int lora_begin(LoraParams& p, void* plan, cudaStream_t s, bool pdl);
int lora_finish(LoraParams& p, cudaStream_t s, bool pdl);

}  // namespace aipu
