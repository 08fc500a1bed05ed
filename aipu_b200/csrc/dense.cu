// Projection of many token rows on the 5th-generation tensor cores, for every weight type, sm_100a.
//
//   y32[m, n] = sum_k x[m, k] * w[n, k],  x bf16, w = GGUF rows (Q4_K, Q6_K, Q8_0, F16), fp32 out
//
// Two kernels: the weights and tokens as fp16 rows, and a GEMM of the two (TMA tiles with 128-byte swizzle,
// tcgen05.mma kind::f16, fp32 accumulators in TMEM). Dequantising once per call and not once per token tile is what makes
// this faster than a GEMM that dequantises its own tiles: 2048 rows of 6144 x 2048 Q4_K 99 us against 145. The operands take 20
// of them, the GEMM 79 (its two products 1.31 PFLOP/s, 0.80 of the measured bf16 peak; the tensor pipe is busy 82 % of the
// time on the 128 SMs that have a tile).
//
// Rounding: a token row is scaled by a power of two and is then exact in fp16 (bf16 has 8 bits; values below
// 2^-24 of the row's largest lose bits). A weight is dequantised in fp32 as ggml defines it, scaled by a
// power of two per row, and enters as two fp16 halves, 22 bits (2^-38 of the row's bound where it is small), whose
// products go to accumulators of their own and are added once. One half alone would round it by 2^-11 and change every
// tenth bf16 result (and the call of that case would take 79 us for 111). F16 weights are used as they are stored, in one
// product. Products are exact, sums fp32.
#include <algorithm>

#include "deq.cuh"
#include "dense.cuh"
#include "kernels.h"
#include "launch.h"
#include "tc.cuh"

namespace aipu {

// ------------------------------------------------------------------ operands
// s such that bound * 2^-s is in [2^top, 2^(top + 1)) (0 and not finite: some scale that is finite). Rows of magnitudes
// below 2^(top - 126) are scaled by 2^126 only: bf16 values are multiples of 2^-133, so those stay exact in fp16.
__device__ __forceinline__ int scale_shift(float bound, int top) {
  const int e = static_cast<int>((__float_as_uint(bound) >> 23) & 0xFFu);
  const int s = bound == 0.f ? 0 : e - 127 - top;
  return max(s, -126);  // (at most 128 - top: the factor 2^-s is a normal number)
}
// shift of a token row with an infinite value (top = 9): all its results are infinite or NaN by the upper halves alone (a
// lower half of 0 or of the other sign would make NaN of an infinity)
constexpr int kNotFinite = 255 - 127 - 9;

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// a and b as fp16 pairs hi + lo: hi rounded, lo the rest (exact in fp32) rounded, 2^-22 of the value together. A value
// that is not finite is hi alone.
__device__ __forceinline__ void two_halves(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = half2_bits(fabsf(f.x) < INFINITY ? __fsub_rn(a, f.x) : 0.f, fabsf(f.y) < INFINITY ? __fsub_rn(b, f.y) : 0.f);
}

// 8 bytes from a 2-byte aligned address
__device__ __forceinline__ uint2 ld8_a2(const uint8_t* p) {
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
  return make_uint2(__ldg(q) | (static_cast<uint32_t>(__ldg(q + 1)) << 16), __ldg(q + 2) | (static_cast<uint32_t>(__ldg(q + 3)) << 16));
}

// largest magnitude that the header of unit u (256 weights) of a row allows, from its scales
template <int WT>
__device__ __forceinline__ float unit_bound(const uint8_t* row, int u) {
  if (WT == WT_Q4K) {
    const uint32_t h = __ldg(reinterpret_cast<const uint32_t*>(row + 144 * u));
    return fabsf(f16_bits_to_f32(h)) * 945.f + fabsf(f16_bits_to_f32(h >> 16)) * 63.f;
  }
  if (WT == WT_Q6K) return fabsf(f16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(row + 210 * u + 208)))) * 4096.f;
  float m = 0.f;
  for (int b = 0; b < 8; ++b)
    m = fmaxf(m, fabsf(f16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(row + 272 * u + 34 * b)))) * 128.f);
  return m;
}

// weights 8 l .. 8 l + 7 of unit u, with the roundings of ggml's dequantisation
template <int WT>
__device__ __forceinline__ void unit_weights(const uint8_t* row, int u, int l, float (&w)[8]) {
  if (WT == WT_Q4K) {
    const uint8_t* b = row + 144 * u;
    const uint4 h = __ldg(reinterpret_cast<const uint4*>(b));  // d, dmin, 12 bytes of scales
    const int j = l >> 2, i = j & 3;
    const uint32_t near = h.y >> (8 * i), far = h.z >> (8 * i), both = h.w >> (8 * i);
    const uint32_t sc = j < 4 ? near & 63u : (both & 15u) | ((near >> 6 & 3u) << 4);
    const uint32_t mn = j < 4 ? far & 63u : (both >> 4 & 15u) | ((far >> 6 & 3u) << 4);
    const float d = __fmul_rn(f16_bits_to_f32(h.x), static_cast<float>(sc));
    const float m = __fmul_rn(f16_bits_to_f32(h.x >> 16), static_cast<float>(mn));
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(b + 16 + 32 * (j >> 1) + 8 * (l & 3)));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t code = (k < 4 ? q.x : q.y) >> (8 * (k & 3) + 4 * (j & 1)) & 15u;
      w[k] = __fsub_rn(__fmul_rn(d, static_cast<float>(code)), m);
    }
  } else if (WT == WT_Q6K) {
    const uint8_t* b = row + 210 * u;
    const int half = l >> 4, run = (l >> 2) & 3, n = 8 * (l & 3);
    const uint2 lo = ld8_a2(b + 64 * half + 32 * (run & 1) + n), hi = ld8_a2(b + 128 + 32 * half + n);
    const int sc = static_cast<int8_t>(__ldg(b + 192 + (l >> 1)));
    const float d = __fmul_rn(f16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(b + 208))), static_cast<float>(sc));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t nib = (k < 4 ? lo.x : lo.y) >> (8 * (k & 3) + 4 * (run >> 1)) & 15u;
      const uint32_t top = (k < 4 ? hi.x : hi.y) >> (8 * (k & 3) + 2 * run) & 3u;
      w[k] = __fmul_rn(d, static_cast<float>(static_cast<int>(nib | (top << 4)) - 32));
    }
  } else {
    const uint8_t* b = row + 272 * u + 34 * (l >> 2);
    const float d = f16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(b)));
    const uint2 q = ld8_a2(b + 2 + 8 * (l & 3));
#pragma unroll
    for (int k = 0; k < 8; ++k)
      w[k] = __fmul_rn(d, static_cast<float>(static_cast<int8_t>((k < 4 ? q.x : q.y) >> (8 * (k & 3)) & 255u)));
  }
}

// Both operands in one launch; four warps a row, two rows a CTA. The first CTAs take weight rows (their scale
// from the blocks' headers, then 256 weights a warp and step, 16 bytes a lane), the others token rows (their
// scale from the largest magnitude, into [2^9, 2^10)). It depends on nothing that the kernel before it
// writes and only ends after it, so both run at the same time.
template <int WT>
__global__ void __launch_bounds__(256) aipu_dense_operands_kernel(const uint8_t* __restrict__ w, int N, int K, int64_t row_bytes,
                                                                  uint16_t* __restrict__ w16, int* __restrict__ wshift,
                                                                  const uint16_t* __restrict__ x, int M,
                                                                  uint16_t* __restrict__ x16, int* __restrict__ xshift) {
  __shared__ float red[2][4];
  const int half = threadIdx.x >> 7, t = threadIdx.x & 127, warp = t >> 5, lane = t & 31;
  const int wblocks = WT == WT_F16 ? 0 : (N + 1) / 2;
  pdl_launch_dependents();  // (the GEMM waits for this grid before it reads)
  if (WT != WT_F16 && blockIdx.x < wblocks) {
    const int n = 2 * blockIdx.x + half;
    if (n < N) {
      const uint8_t* row = w + n * row_bytes;
      const int units = K / 256;
      float bound = 0.f;
      for (int u = lane; u < units; u += 32) bound = fmaxf(bound, unit_bound<WT>(row, u));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
      const int s = scale_shift(bound, 13);
      const float f = exp2i(-s);
      if (t == 0) wshift[n] = s;
      uint4* dst = reinterpret_cast<uint4*>(w16 + static_cast<int64_t>(n) * K) + lane;
      uint4* rest = reinterpret_cast<uint4*>(w16 + (static_cast<int64_t>(N) + n) * K) + lane;
#pragma unroll 2
      for (int u = warp; u < units; u += 4) {
        float v[8];
        unit_weights<WT>(row, u, lane, v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) two_halves(__fmul_rn(v[2 * k], f), __fmul_rn(v[2 * k + 1], f), hi[k], lo[k]);
        dst[32 * u] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        rest[32 * u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  } else {
    const int m = 2 * (blockIdx.x - wblocks) + half;
    if (m < M) {
      const uint4* src = reinterpret_cast<const uint4*>(x + static_cast<int64_t>(m) * K);
      const int nv = K / 8;
      float mx = 0.f;
#pragma unroll 4
      for (int v = t; v < nv; v += 128) {
        const uint4 q = __ldg(src + v);
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(u[i] << 16)), fabsf(__uint_as_float(u[i] & 0xFFFF0000u))));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (lane == 0) red[half][warp] = mx;
      named_bar_sync(1 + half, 128);
      mx = fmaxf(fmaxf(red[half][0], red[half][1]), fmaxf(red[half][2], red[half][3]));
      const int s = scale_shift(mx, 9);
      const float f = exp2i(-s);
      if (t == 0) xshift[m] = s;
      uint4* dst = reinterpret_cast<uint4*>(x16 + static_cast<int64_t>(m) * K);
#pragma unroll 4
      for (int v = t; v < nv; v += 128) {
        const uint4 q = __ldg(src + v);
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[i] = half2_bits(__fmul_rn(__uint_as_float(u[i] << 16), f), __fmul_rn(__uint_as_float(u[i] & 0xFFFF0000u), f));
        dst[v] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
  pdl_wait();
}

// ------------------------------------------------------------------ GEMM
struct DenseParams {
  alignas(64) CUtensorMap wmap;  // [N][K] fp16, behind it the lower halves' [N][K]; box 128 rows x 64 k, 128-byte swizzle
  alignas(64) CUtensorMap xmap;  // [M][K] fp16, box NT rows x 64 k
  const int* wshift;             // [N] or nullptr (0)
  const int* xshift;             // [M]
  float* y;                      // share of K z at y + z * M * ldy
  int64_t ldy;
  int N, K, M;
  int* status;
};

constexpr int kDenseThreads = 320;  // 8 epilogue warps, the copy warp, the MMA warp

// P: 2 where the weights are two halves, 1 where they are stored as fp16
template <int NT, int P>
struct DenseCfg {
  static constexpr int A = 128 * 128, B = NT * 128;  // bytes of a stage: 64 k of 128 weight rows (P times) and NT token rows
  static constexpr int STAGE = P * A + B;
  static constexpr int S = std::min(8, 196608 / STAGE);  // stages in 192 KB: 3 to 8
  static constexpr int TOTAL = S * STAGE + 1024;     // (tiles start on 1024 bytes)
};

struct DenseBars {
  uint64_t full[8], empty[8], done;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// One 128 x NT tile of (weight rows, token rows) and share of K a CTA. Copy warp: a stage is one TMA box of each operand.
// MMA warp: four K = 16 steps a stage, one thread; a commit releases the stage. Epilogue: TMEM lane =
// weight row, so a warp's store is 32 neighbouring results of a token. Every wait is bounded: on expiry the
// status word is set, the roles leave, copies and MMAs in flight are waited for (bounded), TMEM is freed.
template <int NT, int P>
__global__ void __launch_bounds__(kDenseThreads, 1) aipu_dense_gemm_kernel(const __grid_constant__ DenseParams p) {
  using C = DenseCfg<NT, P>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DenseBars bars;
  __shared__ int xs[NT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int n0 = blockIdx.x * 128, m0 = blockIdx.y * NT;
  if (tid == 0) {
    for (int i = 0; i < C::S; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.done, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(&bars.tmem, P * NT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  pdl_wait();
  pdl_launch_dependents();
  const int all = p.K / 64;
  const int k0 = static_cast<int>(static_cast<int64_t>(all) * blockIdx.z / gridDim.z);
  const int steps = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.z + 1) / gridDim.z) - k0;
  volatile int* abort = &bars.abort;
  if (warp == 8) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < steps && !*abort; ++i, ++issued) {
        const int s = i % C::S;
        if (i >= C::S && !mbar_wait_bounded(&bars.empty[s], (i / C::S + 1) & 1, p.status, ST_TIMEOUT_EMPTY)) {
          *abort = 1;
          break;
        }
        mbar_arrive_expect_tx(&bars.full[s], C::STAGE);
#pragma unroll
        for (int h = 0; h < P; ++h)  // (rows past N are of the other half or 0: their results are not stored)
          tma_load_2d(base + s * C::STAGE + h * C::A, &p.wmap, 64 * (k0 + i), h * p.N + n0, &bars.full[s]);
        tma_load_2d(base + s * C::STAGE + P * C::A, &p.xmap, 64 * (k0 + i), m0, &bars.full[s]);
      }
      // no copy may land after the CTA has ended: the MMAs have read them all, or (abort) they are waited for
      mbar_wait_bounded(&bars.done, 0, p.status, ST_TIMEOUT_FULL);
      if (*abort)
        for (int i = max(0, issued - C::S); i < issued; ++i)
          mbar_wait_bounded(&bars.full[i % C::S], (i / C::S) & 1, p.status, ST_TIMEOUT_FULL, 200000000LL);
    }
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_f16(128, NT);
      for (int i = 0; i < steps; ++i) {
        const int s = i % C::S;
        if (*abort || !mbar_wait_bounded(&bars.full[s], (i / C::S) & 1, p.status, ST_TIMEOUT_FULL)) {
          *abort = 1;
          break;
        }
        tc_fence_after();
        const uint32_t a = base + s * C::STAGE, b = a + P * C::A;
#pragma unroll
        for (int h = 0; h < P; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem + h * NT, umma_desc_sw128(a + h * C::A + 32 * k, 1024), umma_desc_sw128(b + 32 * k, 1024), idesc,
                     (i | k) ? 1u : 0u);
        umma_commit(&bars.empty[s]);
      }
      umma_commit(&bars.done);
    }
  } else {
    for (int i = tid; i < NT; i += 256) xs[i] = m0 + i < p.M ? p.xshift[m0 + i] : 0;
    named_bar_sync(1, 256);
    const int q = warp & 3, n = n0 + 32 * q + lane;
    // (the weights' factor first: finite ones have shifts of -32 to 13, so nothing is lost or overflows before the result does)
    const float wf = exp2i((p.wshift && n < p.N) ? p.wshift[n] : 0);
    const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.done, 0, p.status, ST_TIMEOUT_FULL)) && !*abort;
    if (ok) {
      tc_fence_after();
      const int cols = min(NT, p.M - m0);
#pragma unroll 1
      for (int c0 = (warp >> 2) * 16; c0 < cols; c0 += 32) {
        float v[16], lo[16];
        tmem_ld16(tmem + (static_cast<uint32_t>(32 * q) << 16) + c0, v);
        if (P == 2) {
          tmem_ld16(tmem + (static_cast<uint32_t>(32 * q) << 16) + NT + c0, lo);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < cols && xs[c0 + j] < kNotFinite) v[j] = __fadd_rn(v[j], lo[j]);
        }
        if (n < p.N) {
          float* dst = p.y + (static_cast<int64_t>(blockIdx.z) * p.M + m0 + c0) * p.ldy + n;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < cols) dst[j * p.ldy] = __fmul_rn(__fmul_rn(v[j], wf), exp2i(xs[c0 + j]));
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    mbar_wait_bounded(&bars.done, 0, p.status, ST_TIMEOUT_FULL, 200000000LL);  // the MMAs in flight (after an abort too)
    tc_fence_after();
    tmem_dealloc(tmem, P * NT);
    tmem_relinquish();
  }
}

// ------------------------------------------------------------------ host
static size_t al1k(size_t v) { return (v + 1023) & ~static_cast<size_t>(1023); }

size_t dense_bytes(int wt, int64_t N, int64_t K, int64_t M) {
  const size_t w = wt == WT_F16 ? 0 : al1k(static_cast<size_t>(4) * N * K) + al1k(4 * N);
  return w + al1k(static_cast<size_t>(2) * M * K) + al1k(4 * M);
}

static int rows_map(CUtensorMap* map, const void* base, int64_t rows, int K, int box) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(K) * 2};
  const cuuint32_t bx[2] = {64, static_cast<cuuint32_t>(box)};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, bx, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int NT, int P>
static int dense_launch_p(DenseParams& p, int parts, cudaStream_t s) {
  using C = DenseCfg<NT, P>;
  const void* kern = reinterpret_cast<const void*>(aipu_dense_gemm_kernel<NT, P>);
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(kern, C::TOTAL, attr, "cudaFuncSetAttribute(dense)");
  if (rc) return rc;
  return launch_kernel(kern, dim3((p.N + 127) / 128, (p.M + NT - 1) / NT, parts), dim3(kDenseThreads), C::TOTAL, s, true, &p);
}
template <int NT>
static int dense_launch(DenseParams& p, int parts, cudaStream_t s) {
  return p.wshift ? dense_launch_p<NT, 2>(p, parts, s) : dense_launch_p<NT, 1>(p, parts, s);
}

static int token_tile(int64_t M) { return M <= 64 ? 64 : M <= 128 ? 128 : 256; }

int dense_parts(int64_t N, int64_t K, int64_t M) {
  // As many shares of K as still leave a CTA an SM (a B200's 148: the workspace is sized without a context), of eight
  // steps of 64 at least; of sixteen above 256 rows, where the last kernel pays more for adding shares than a short GEMM
  // gains. F16 in us, a call, shares of at least 4 / 8 / 16 / 32 steps: 300 rows, 512 x 1024 29.3 / 29.4 / 26.4 / 26.4,
  // 1003 x 4096 46.5 / 46.5 / 37.2 / 40.8, 2048 x 6144 41.8 / 41.5 / 41.5 / 44.1. Fewer rows, 4 / 8 steps: 64 rows of 1024 x
  // 2048 14.9 / 12.0, 256 rows of 512 x 1024 19.7 / 16.0, but 64 rows of 64 x 1024 10.1 / 11.1.
  const int64_t tiles = ((N + 127) / 128) * ((M + token_tile(M) - 1) / token_tile(M));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(8, K / (M > 256 ? 1024 : 512)), 148 / tiles)));
}

template <int WT>
static int operands_launch(const uint8_t* w, int N, int K, uint16_t* w16, int* wshift, const uint16_t* x, int M, uint16_t* x16,
                           int* xshift, cudaStream_t s, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((WT == WT_F16 ? 0 : (N + 1) / 2) + (M + 1) / 2);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  return set_cuda_error(cudaLaunchKernelEx(&cfg, aipu_dense_operands_kernel<WT>, w, N, K, row_bytes_of(WT, K), w16, wshift, x, M,
                                           x16, xshift),
                        "aipu_dense_operands_kernel");
}

int dense_gemm(int wt, const uint8_t* w, int N, int K, const uint16_t* x, int M, float* y32, int64_t ldy, void* scratch,
               int* status, cudaStream_t s, bool pdl) {
  if (K % 256 || K <= 0 || N <= 0 || M <= 0) return set_error(EINVAL_, "dense: K must be a multiple of 256");
  uint8_t* b = static_cast<uint8_t*>(scratch);
  uint16_t* w16 = nullptr;
  int* wshift = nullptr;
  if (wt != WT_F16) {
    w16 = reinterpret_cast<uint16_t*>(b);
    b += al1k(static_cast<size_t>(4) * N * K);
    wshift = reinterpret_cast<int*>(b);
    b += al1k(4 * static_cast<size_t>(N));
  }
  uint16_t* x16 = reinterpret_cast<uint16_t*>(b);
  b += al1k(static_cast<size_t>(2) * M * K);
  int* xshift = reinterpret_cast<int*>(b);
  int rc;
  switch (wt) {
    case WT_Q4K: rc = operands_launch<WT_Q4K>(w, N, K, w16, wshift, x, M, x16, xshift, s, pdl); break;
    case WT_Q6K: rc = operands_launch<WT_Q6K>(w, N, K, w16, wshift, x, M, x16, xshift, s, pdl); break;
    case WT_Q80: rc = operands_launch<WT_Q80>(w, N, K, w16, wshift, x, M, x16, xshift, s, pdl); break;
    default: rc = operands_launch<WT_F16>(w, N, K, w16, wshift, x, M, x16, xshift, s, pdl);
  }
  if (rc) return rc;
  const int nt = token_tile(M), parts = dense_parts(N, K, M);
  DenseParams p = {};
  rc = wt == WT_F16 ? rows_map(&p.wmap, w, N, K, 128) : rows_map(&p.wmap, w16, 2 * static_cast<int64_t>(N), K, 128);
  if (!rc) rc = rows_map(&p.xmap, x16, M, K, nt);
  if (rc) return rc;
  p.wshift = wshift;
  p.xshift = xshift;
  p.y = y32;
  p.ldy = ldy;
  p.N = N;
  p.K = K;
  p.M = M;
  p.status = status;
  return nt == 64 ? dense_launch<64>(p, parts, s) : nt == 128 ? dense_launch<128>(p, parts, s) : dense_launch<256>(p, parts, s);
}

}  // namespace aipu
