// Projection of many rows through fp16 operands: parameters and launches of dense.cu.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace aipu {

// token rows of one launch: 65535 tiles of 256
constexpr int64_t kDenseMaxRows = 65535 * 256;
// scratch of dense_gemm for N weight rows of type wt, K and M token rows
size_t dense_bytes(int wt, int64_t N, int64_t K, int64_t M);
// shares of K of the result of dense_gemm
int dense_parts(int64_t N, int64_t K, int64_t M);
// y32[parts][M, N] (fp32, rows ldy elements apart, to be summed over the parts) = x[M, K] (bf16) x W^T, W = N GGUF rows. pdl: x and W do
// not depend on the kernel launched before, whose dependents may be launched early; what follows dense_gemm
// in the stream then follows that kernel too
int dense_gemm(int wt, const uint8_t* w, int N, int K, const uint16_t* x, int M, float* y32, int64_t ldy, void* scratch,
               int* status, cudaStream_t s, bool pdl);

}  // namespace aipu
