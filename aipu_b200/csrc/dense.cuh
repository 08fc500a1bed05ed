// Projection of many rows through fp16 operands: parameters and launches of dense.cu.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace aipu {

// scratch of dense_gemm for N weight rows of type wt, K and M token rows
size_t dense_bytes(int wt, int64_t N, int64_t K, int64_t M);
// y32[M, N] (fp32) = x[M, K] (bf16) x W^T, W = N GGUF rows
int dense_gemm(int wt, const uint8_t* w, int N, int K, const uint16_t* x, int M, float* y32, void* scratch, int* status,
               cudaStream_t s);

}  // namespace aipu
