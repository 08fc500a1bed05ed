// Low-rank adapters of many requests beside a shared projection, sm_100a.
//
//   h[m, r]   = sum_k x[m, k] A[id][r, k]                      id = ids[m], r < rank[id], fp32
//   out[m, n] = round( y[m, n] + sum_r (scale[id] h[m, r]) B[id][n, r] )
//
// Bound: 2 T flops per byte pair of an adapter for a tile of T rows, and A, B, x, y and out are each
// read or written once, so the operator is limited by latency (one row) or by memory (many rows) long
// before the tensor pipe; mma.sync, whose fragments come straight from global memory, feeds it without
// a trip through shared memory or TMEM.
//
// Few rows (lora_direct): ONE launch. A cluster of CTAs takes a tile of up to 8 rows that share an adapter
// (found by comparing the ids).
//   1. CTA c and its 8 warps each take a share of K. Rank rows are the 16 MMA rows, token rows the 8
//      MMA columns; a lane loads 8 consecutive k of its rows (16 bytes) and uses them as two MMA steps
//      whose k order is permuted the same way on both sides.
//   2. The partial sums are added over the warps in shared memory and over the CTAs through distributed
//      shared memory, always in the same order (no atomics: equal calls give equal bits).
//   3. CTA c and its warps each take 64-column blocks of N. The MMA's rows are columns of y, ordered so
//      that a lane ends with 8 consecutive columns of a row: y is read and written 16 bytes at a time.
//   h never leaves the chip, and the reads of B and y do not wait for the sums of A.
//   (4096 x 4096, device time in a graph: 1 row of rank 16 5.8 us, 64 rows of 32 adapters of rank 16 to 64 9.1 us.)
// More rows: a plan (rows ordered by adapter, tiles of up to 64 of them), the first product (a tile and a
// share of K a CTA: x and A stream through a ring of asynchronous copies in shared memory, partial sums to
// global memory), the second product (a tile and a share of N a CTA: step 3 above, 32 columns a warp). 4096 rows of
// eight adapters of rank 32, 6144 x 2048: 33 us, 88 MB at 2.7 TB/s; as one cluster kernel 119 us, because its
// phases followed one another with one CTA an SM.
//
// Rounding: bf16 x and A products are exact in the MMA, sums are fp32: the MMA's own, which are cut off, over 64 k (and 32
// ranks, fp32 results), then rounded adds. h enters the second product as 2 (bf16 result) or 3 (fp32 result) bf16 pieces, 16 and
// 24 bits: for a bf16 result 2^-16 of h is 2^-8 of its own rounding, and a third piece would take Q6_K 2048 x 6144, 8
// rows, from 19.4 to 21.9 us and 4096 rows of rank 128, 4096 x 4096, from 82 to 128. fp16 adapters enter as two bf16 pieces
// (11 bits: exact).
#include <algorithm>
#include <cstdint>

#include "cluster.cuh"
#include "common.cuh"
#include "kernels.h"
#include "launch.h"
#include "lora.cuh"

namespace aipu {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kDirectRows = 256;     // rows of the one-launch kernel (a thread each) at most
constexpr int kDirectCtas = 8;       // CTAs of its clusters
constexpr int kMaxAdapters = 32768;  // counters of the plan kernel in shared memory

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 consecutive 16-bit values at p, of which `valid` (from the first) are wanted and the others come as 0. VEC: p is
// 16-byte aligned and valid is 0 or 8. Else from the one or two aligned 16-byte pieces that hold wanted values
// (the tensors are readable to such boundaries), moved into place by selects and a funnel shift: a quarter of
// the loads that one value at a time takes, and far less code (1 row of aligned 4096 x 4096 got 1.8 us faster too).
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int valid) {
  if (valid <= 0) return make_uint4(0, 0, 0, 0);
  if (VEC) return __ldg(reinterpret_cast<const uint4*>(p));
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint4* base = reinterpret_cast<const uint4*>(a & ~static_cast<uintptr_t>(15));
  const int off = static_cast<int>(a & 15u);  // even
  const uint4 u = __ldg(base);
  const uint4 v = off + 2 * min(valid, 8) > 16 ? __ldg(base + 1) : make_uint4(0, 0, 0, 0);
  const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  uint32_t s8[6], s4[5], o[4];
#pragma unroll
  for (int i = 0; i < 6; ++i) s8[i] = (off & 8) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) s4[i] = (off & 4) ? s8[i + 1] : s8[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (off & 2) ? __funnelshift_r(s4[i], s4[i + 1], 16) : s4[i];
  if (valid < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i >= valid) o[i] = 0;
      else if (2 * i + 1 >= valid) o[i] &= 0xFFFFu;
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// v as bf16 pieces: hi = v cut off (to the next value towards 0 where nothing would be left) and the rest, which is exact.
// So no piece of a value other than 0 is 0 or has another sign, and infinity = the largest number + infinity: pieces
// times an infinite or NaN factor sum to what the value times it is. (Below 2^-110 a rest may be too small for the type.)
__device__ __forceinline__ uint32_t upper(float v) { return (__float_as_uint(v) - (v != 0.f ? 1u : 0u)) & 0xFFFF0000u; }
__device__ __forceinline__ uint32_t piece(float v, float& rest) {
  const uint32_t hi = upper(v);
  rest = __fsub_rn(v, __uint_as_float(hi));
  return hi >> 16;
}
// packed pair of fp16 -> packed bf16 hi and lo (11 bits: lo is exact too)
__device__ __forceinline__ void split_f16(uint32_t w, uint32_t& hi, uint32_t& lo) {
  const float a = f16_bits_to_f32(w), b = f16_bits_to_f32(w >> 16);
  const uint32_t ua = upper(a), ub = upper(b);
  hi = prmt(ua, ub, 0x7632u);
  const float ra = __fsub_rn(a, __uint_as_float(ua)), rb = __fsub_rn(b, __uint_as_float(ub));
  lo = prmt(__float_as_uint(ra), __float_as_uint(rb), 0x7632u);
}

// acc += (16 rank or output rows: va rows g, vb rows g + 8) x (8 columns: x), two MMA steps of 16
__device__ __forceinline__ void mma_pair(float (&acc)[4], const uint4& va, const uint4& vb, const uint4& x) {
  mma_bf16_16816(acc, va.x, vb.x, va.y, vb.y, x.x, x.y);
  mma_bf16_16816(acc, va.z, vb.z, va.w, vb.w, x.z, x.w);
}
__device__ __forceinline__ void split4_f16(const uint4& v, uint4& hi, uint4& lo) {
  split_f16(v.x, hi.x, lo.x);
  split_f16(v.y, hi.y, lo.y);
  split_f16(v.z, hi.z, lo.z);
  split_f16(v.w, hi.w, lo.w);
}

constexpr int kDirectTile = 8;  // rows of a tile of the one-launch kernel
static_assert(kDirectRows <= kLoraThreads, "a thread a row");
template <int MT>
struct LoraCfg {
  static constexpr int TM = kDirectTile;
  static constexpr int RP = 16 * MT;                 // rank rows
  static constexpr int RF = RP < 32 ? 32 : RP;       // rank columns of the second product (steps of 32)
  static constexpr int HPITCH = RF + 8;              // bf16 pitch of a token's h (16-byte rows, banks spread)
  static constexpr int PITCH = RP + 4;               // fp32 pitch of a token's sums (banks spread)
  static constexpr int OFF_HP = 0;                   // fp32 [TM][PITCH]: this CTA's sums
  static constexpr int OFF_HF = OFF_HP + TM * PITCH * 4;  // bf16 [3][TM][HPITCH]: scale * h
  static constexpr int OFF_RED = OFF_HF + 3 * TM * HPITCH * 2;
  static constexpr int TOTAL = OFF_RED + kLoraWarps * TM * PITCH * 4;
};

struct LoraTile {
  int id, rows, rank;
  float scale;
};

// ------------------------------------------------------------------ first product: this warp's k range
// The MMA's own sums are cut off and not rounded, so it sums 64 k at most, the small pieces first, and the rest is rounded
// adds, as in the first product of many rows (no slower: 256 rows of rank 64 13.9 -> 13.7 us).
template <int MT, int AT, bool VEC>
__device__ __forceinline__ void shrink(const LoraParams& p, const int* tok, const LoraTile& tl, int c0, int c1, int lane,
                                       float (&acc)[MT][4]) {
  constexpr int U = MT == 1 ? 4 : MT == 2 ? 2 : 1;  // k chunks loaded ahead
  const int g = lane >> 2, t = lane & 3;
  const uint16_t* abase = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(tl.id) * p.R * p.K;
  const uint16_t* xrow = p.x + static_cast<int64_t>(tok[g]) * p.ldx;
  for (int c = c0; c < c1; c += U) {
    uint4 va[U][MT][2], vx[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c + u) * 32 + 8 * t;
      const int valid = (c + u < c1) ? p.K - k : 0;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * i + 8 * h + g;
          va[u][i][h] = load8<VEC>(abase + static_cast<int64_t>(r) * p.K + k, r < tl.rank ? valid : 0);
        }
      vx[u] = load8<VEC>(xrow + k, g < tl.rows ? valid : 0);
    }
    constexpr int V = U < 2 ? U : 2;  // chunks that the MMA sums
#pragma unroll
    for (int u0 = 0; u0 < U; u0 += V)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (16 * i >= tl.rank) continue;  // warp-uniform
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = u0; u < u0 + V; ++u) {
          if (AT == AD_F16) {
            uint4 ah, al, bh, bl;
            split4_f16(va[u][i][0], ah, al);
            split4_f16(va[u][i][1], bh, bl);
            mma_pair(sum, al, bl, vx[u]);
            mma_pair(sum, ah, bh, vx[u]);
          } else {
            mma_pair(sum, va[u][i][0], va[u][i][1], vx[u]);
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][q] = __fadd_rn(acc[i][q], sum[q]);
      }
  }
}

// ------------------------------------------------------------------ second product and the result rows
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // rounded to the nearest, ties to even
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A warp's block of y is 16 Q columns: MMA q's rows g and g + 8 are its columns 2 Q g + 2 q and + 2 q + 1, so a
// lane holds 2 Q neighbouring columns of rows 2 t and 2 t + 1 of the 8 token columns of an MMA. Those values of y:
template <int Q, bool Y32>
struct YRows {
  static constexpr int W = Q * (Y32 ? 2 : 1);  // 32-bit words a row
  uint32_t w[2][W];
  __device__ __forceinline__ void put(int e, const void* src) {
    if constexpr (W == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(src);
      w[e][0] = v.x;
      w[e][1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 v = reinterpret_cast<const uint4*>(src)[i / 4];
        w[e][i] = v.x;
        w[e][i + 1] = v.y;
        w[e][i + 2] = v.z;
        w[e][i + 3] = v.w;
      }
    }
  }
  // rows 8 j + 2 t (+ 1) of the tile from global memory, columns n on (where whole 16-byte pieces may be read)
  __device__ __forceinline__ void load(const LoraParams& p, const int* tok, int rows, int n, int j, int t) {
    if (n + 2 * Q > p.vy) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = 8 * j + 2 * t + e;
      if (m >= rows) continue;
      put(e, static_cast<const uint8_t*>(p.y) + (static_cast<int64_t>(tok[m]) * p.ldy + n) * (Y32 ? 4 : 2));
      if (Y32 && p.yparts > 1) {
        const float* o = static_cast<const float*>(p.y) + static_cast<int64_t>(tok[m]) * p.ldy + n;
        const int64_t share = static_cast<int64_t>(p.M) * p.ldy;
        for (int s = 1; s < p.yparts; s += 4) {  // the loads of four shares are in flight together
          float4 v[4][W / 4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (s + u < p.yparts)
#pragma unroll
              for (int i = 0; i < W / 4; ++i) v[u][i] = *reinterpret_cast<const float4*>(o + (s + u) * share + 4 * i);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (s + u >= p.yparts) break;
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
              const float d[4] = {v[u][i].x, v[u][i].y, v[u][i].z, v[u][i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) w[e][4 * i + k] = __float_as_uint(__fadd_rn(__uint_as_float(w[e][4 * i + k]), d[k]));
            }
          }
        }
      }
    }
  }
  __device__ __forceinline__ float get(int e, int i) const {
    if (Y32) return __uint_as_float(w[e][Y32 ? i : 0]);
    return __uint_as_float((i & 1) ? w[e][i >> 1] & 0xFFFF0000u : w[e][i >> 1] << 16);
  }
};

// out rows 8 j + 2 t (+ 1) of the tile, columns n on: y + acc, rounded once (y: loaded, or read here a column at a time)
template <int Q, bool Y32, bool O32>
__device__ __forceinline__ void finish_rows(const LoraParams& p, const int* tok, int rows, int n, int j, int t,
                                            const float (&acc)[Q][4], const YRows<Q, Y32>& y, bool loaded) {
  constexpr int C = 2 * Q;
  const int cols = p.N - n;
  if (cols <= 0) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int m = 8 * j + 2 * t + e;
    if (m >= rows) continue;
    const int64_t row = tok[m];
    float d[C];
#pragma unroll
    for (int i = 0; i < C; ++i) d[i] = acc[i >> 1][e + 2 * (i & 1)];
    if (loaded) {
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] = __fadd_rn(y.get(e, i), d[i]);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (i >= cols) break;
        d[i] = __fadd_rn(Y32 ? static_cast<const float*>(p.y)[row * p.ldy + n + i]
                             : bf16_bits_to_f32(static_cast<const uint16_t*>(p.y)[row * p.ldy + n + i]),
                         d[i]);
      }
    }
    if (O32) {
      float* op = static_cast<float*>(p.out) + row * p.ldo + n;
      if (p.vo == 2 && cols >= C) {
#pragma unroll
        for (int i = 0; i < C; i += 4) *reinterpret_cast<float4*>(op + i) = make_float4(d[i], d[i + 1], d[i + 2], d[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (i < cols) op[i] = d[i];
      }
    } else {
      uint16_t* op = static_cast<uint16_t*>(p.out) + row * p.ldo + n;
      uint32_t o[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i) o[i] = pack_bf16(d[2 * i], d[2 * i + 1]);
      if (p.vo == 2 && cols >= C) {
        if constexpr (Q == 2) *reinterpret_cast<uint2*>(op) = make_uint2(o[0], o[1]);
        else *reinterpret_cast<uint4*>(op) = make_uint4(o[0], o[1], o[2], o[3]);
      } else if (p.vo == 1 && cols >= C) {
#pragma unroll
        for (int i = 0; i < Q; ++i) reinterpret_cast<uint32_t*>(op)[i] = o[i];
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (i < cols) op[i] = static_cast<uint16_t>(o[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// scale * h of one token and two ranks as packed bf16 pieces
template <int NS>
__device__ __forceinline__ void pieces(float2 v, uint32_t (&w)[NS]) {
  float r0, r1, q0, q1;
  w[0] = piece(v.x, r0) | (piece(v.y, r1) << 16);
  if constexpr (NS == 2) {
    w[1] = pack_bf16(r0, r1);
  } else {
    w[1] = piece(r0, q0) | (piece(r1, q1) << 16);
    w[2] = (__float_as_uint(q0) >> 16) | (__float_as_uint(q1) & 0xFFFF0000u);
  }
}

// B rows n .. n + 2 Q - 1 (a lane's columns), rank columns r .. r + 7 (past the rank: 0, whatever is stored)
template <int Q>
__device__ __forceinline__ void load_b(const LoraParams& p, const LoraTile& tl, int n, int r, uint4 (&vb)[2 * Q]) {
  const uint16_t* row = static_cast<const uint16_t*>(p.b) + (static_cast<int64_t>(tl.id) * p.N + n) * p.R + r;
  const int valid = tl.rank - r, rows = p.N - n;
  if (p.wb == 8) {  // R is a multiple of 8: whole vectors are in the row, the columns past the rank are cleared
#pragma unroll
    for (int i = 0; i < 2 * Q; ++i)
      vb[i] = (i < rows && valid > 0) ? __ldg(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(i) * p.R)) : make_uint4(0, 0, 0, 0);
    if (valid < 8) {
#pragma unroll
      for (int i = 0; i < 2 * Q; ++i) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&vb[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (2 * q >= valid) w[q] = 0;
          else if (2 * q + 1 >= valid) w[q] &= 0xFFFFu;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2 * Q; ++i) vb[i] = load8<false>(row + static_cast<int64_t>(i) * p.R, i < rows ? valid : 0);
  }
}

// acc[q][j] += B rows x h of the tile's rows 8 (j0 + j) .. + 7, rank columns 32 rc .. 32 rc + 31
template <int Q, int NT, int AT, int NS>
__device__ __forceinline__ void expand_step(float (&acc)[NT][Q][4], const uint4 (&vb)[2 * Q], const uint16_t* hf, int hpitch,
                                            int hsplit, int j0, int rows, int rc, int lane) {
  const int g = lane >> 2, t = lane & 3;
  // (fp16 adapters: a pair of B rows at a time is split into its two pieces, and h read again for it)
#pragma unroll
  for (int q0 = 0; q0 < Q; q0 += AT == AD_F16 ? 1 : Q) {
    uint4 h0, l0, h1, l1;
    if (AT == AD_F16) {
      split4_f16(vb[2 * q0], h0, l0);
      split4_f16(vb[2 * q0 + 1], h1, l1);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (8 * (j0 + j) >= rows) continue;  // warp-uniform
      const uint16_t* hrow = hf + (8 * (j0 + j) + g) * hpitch + 32 * rc + 8 * t;
      constexpr int QN = AT == AD_F16 ? 1 : Q;
      // fp32 results: the MMA's own sums are cut off and not rounded, so it sums 32 ranks only, the small pieces
      // first, and the rest is rounded adds
      float sum[QN][4];
#pragma unroll
      for (int q = 0; q < QN; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[q][i] = NS == 3 ? 0.f : acc[j][q0 + q][i];
#pragma unroll
      for (int s = NS - 1; s >= 0; --s) {
        const uint4 h = *reinterpret_cast<const uint4*>(hrow + s * hsplit);
        if (AT == AD_F16) {
          mma_pair(sum[0], l0, l1, h);
          mma_pair(sum[0], h0, h1, h);
        } else {
#pragma unroll
          for (int q = 0; q < QN; ++q) mma_pair(sum[q], vb[2 * q], vb[2 * q + 1], h);
        }
      }
#pragma unroll
      for (int q = 0; q < QN; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][q0 + q][i] = NS == 3 ? __fadd_rn(acc[j][q0 + q][i], sum[q][i]) : sum[q][i];
    }
  }
}

// Adapter, rank and factor of a tile (id < 0: none)
__device__ __forceinline__ LoraTile lora_tile(const LoraParams& p, int id, int rows) {
  LoraTile tl = {id, rows, 0, 1.f};
  if (id >= 0) {
    tl.rank = p.ranks ? min(max(p.ranks[id], 0), p.R) : p.R;
    if (p.scale) tl.scale = p.scale[id];
  }
  return tl;
}

template <int MT, int AT, bool VEC, bool Y32, bool O32>
__global__ void __cluster_dims__(kDirectCtas) __launch_bounds__(kLoraThreads, 2) aipu_lora_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraCfg<MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int tok[C::TM];
  float* hp = reinterpret_cast<float*>(smem + C::OFF_HP);
  uint16_t* hf = reinterpret_cast<uint16_t*>(smem + C::OFF_HF);
  float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t crank = cluster_rank(), csize = cluster_size();
  constexpr int NS = O32 ? 3 : 2;  // pieces of h
  constexpr int HS = C::TM * C::HPITCH;  // elements of one piece
  // x (and the ids) may come from the kernel before the one that writes y, so they wait too unless the
  // launch says that only y does
  if (!p.wait_y) pdl_wait();

  // A row leads a tile if the number of earlier rows with its id is a multiple of a tile's rows; the tile is
  // that row and the following ones of the id, and this cluster's is the one of the cluster's number.
  __shared__ __align__(16) int key[kDirectRows];  // (read four at a time)
  __shared__ uint32_t lead_bits[kDirectRows / 32];
  int mine = -2, prior = 0;  // this thread's row: its id and the earlier rows with it
  if (tid < p.M) {
    const int v = p.ids[tid];
    if (v >= p.L && blockIdx.x == 0 && p.status) atomicOr(p.status, ST_BAD_ARGS);
    mine = (v < 0 || v >= p.L) ? -1 : v;
  }
  key[tid] = mine;
  __syncthreads();
  if (32 * warp < p.M) {
    prior = __popc(__match_any_sync(0xffffffffu, mine) & ((1u << lane) - 1));
    for (int i = 0; i < 32 * warp; i += 4) {
      const int4 k = *reinterpret_cast<const int4*>(key + i);
      prior += (k.x == mine) + (k.y == mine) + (k.z == mine) + (k.w == mine);
    }
  }
  const uint32_t bits = __ballot_sync(0xffffffffu, (mine >= 0 || (mine == -1 && !p.skip_plain)) && prior % C::TM == 0);
  if (lane == 0) lead_bits[warp] = bits;
  __syncthreads();
  int lead = -1;
  for (int i = 0, skip = blockIdx.x / csize; i < kDirectRows / 32 && lead < 0; ++i) {
    uint32_t word = lead_bits[i];
    const int n = __popc(word);
    if (skip >= n) {
      skip -= n;
      continue;
    }
    for (; skip > 0; --skip) word &= word - 1;
    lead = 32 * i + __ffs(word) - 1;
  }
  if (lead < 0) {  // (the same for every thread of the cluster)
    pdl_launch_dependents();
    if (p.wait_y) pdl_wait();  // a cluster without a tile may not end before what it depends on
    return;
  }
  const int id = key[lead];
  LoraTile tl = lora_tile(p, id, 0);
  __shared__ int lead_prior, count;
  if (tid < C::TM) tok[tid] = 0;
  if (tid == lead) lead_prior = prior;
  if (tid == 0) count = 0;
  __syncthreads();
  const int place = prior - lead_prior;
  if (mine == id && place >= 0 && place < C::TM) {
    tok[place] = tid;
    atomicAdd(&count, 1);
  }
  if (C::RF > C::RP)  // rank columns that the second product reads and the first does not give
    for (int i = tid; i < 3 * C::TM * (C::HPITCH - C::RP); i += kLoraThreads)
      hf[(i / (C::HPITCH - C::RP)) * C::HPITCH + C::RP + i % (C::HPITCH - C::RP)] = 0;
  __syncthreads();
  tl.rows = count;

  const int nblk = (p.N + 63) / 64;
  const int gw = crank * kLoraWarps + warp, nw = csize * kLoraWarps;
  const int c8 = 8 * g;  // this lane's columns of a block
  uint4 vb[8];
  YRows<4, Y32> yt;
  if (!p.wait_y && gw < nblk) yt.load(p, tok, tl.rows, gw * 64 + c8, 0, t);
  bool pending = false;
  if (tl.rank > 0) {
    // ---- first product: this warp's share of K
    float acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
    const int chunks = (p.K + 31) / 32;
    const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * gw / nw);
    const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (gw + 1) / nw);
    shrink<MT, AT, VEC>(p, tok, tl, c0, c1, lane, acc);
    // the first block's B rows are on the way while the sums are joined
    if (gw < nblk) load_b<4>(p, tl, gw * 64 + c8, 8 * t, vb);
    // ---- sums over the warps of the CTA, in warp order
    float* mine = red + warp * C::TM * C::PITCH;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) mine[(2 * t + (q & 1)) * C::PITCH + 16 * i + g + 8 * (q >> 1)] = acc[i][q];
    __syncthreads();
    for (int e = tid; e < C::TM * C::PITCH; e += kLoraThreads) {
      float v = red[e];
#pragma unroll
      for (int w = 1; w < kLoraWarps; ++w) v = __fadd_rn(v, red[w * C::TM * C::PITCH + e]);
      hp[e] = v;
    }
    // ---- sums over the CTAs of the cluster, in rank order; h as bf16 pieces in every CTA
    cluster_arrive();
    cluster_wait();
    const uint32_t hpa = smem_u32(hp);
    for (int e = tid; e < tl.rows * C::RP / 2; e += kLoraThreads) {
      const int m = (2 * e) / C::RP, r = 2 * e - m * C::RP;
      float2 v = make_float2(0.f, 0.f);
      for (uint32_t c = 0; c < csize; ++c) {
        const float2 o = ld_cluster_f2(map_rank(hpa + 4 * (m * C::PITCH + r), c));
        v.x = __fadd_rn(v.x, o.x);
        v.y = __fadd_rn(v.y, o.y);
      }
      // past the rank the sums are 0, or NaN where x is not finite: they count for nothing
      v.x = r < tl.rank ? __fmul_rn(v.x, tl.scale) : 0.f;
      v.y = r + 1 < tl.rank ? __fmul_rn(v.y, tl.scale) : 0.f;
      uint32_t w[NS];
      pieces<NS>(v, w);
#pragma unroll
      for (int s = 0; s < NS; ++s) reinterpret_cast<uint32_t*>(hf)[(s * HS + m * C::HPITCH + r) >> 1] = w[s];
    }
    cluster_arrive();  // no CTA ends before the others have read its sums
    pending = true;
    __syncthreads();
  }
  if (p.wait_y) {
    pdl_wait();
    if (gw < nblk) yt.load(p, tok, tl.rows, gw * 64 + c8, 0, t);
  }
  // ---- second product: 64-column blocks
  const int rchunks = (tl.rank + 31) / 32;
  for (int nb = gw; nb < nblk; nb += nw) {
    float acc[1][4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][q][i] = -0.f;  // y + -0 is y, also for y = -0
    if (nb != gw) yt.load(p, tok, tl.rows, nb * 64 + c8, 0, t);
    for (int rc = 0; rc < rchunks; ++rc) {
      if (nb != gw || rc != 0) load_b<4>(p, tl, nb * 64 + c8, 32 * rc + 8 * t, vb);
      expand_step<4, 1, AT, NS>(acc, vb, hf, C::HPITCH, HS, 0, tl.rows, rc, lane);
    }
    finish_rows<4, Y32, O32>(p, tok, tl.rows, nb * 64 + c8, 0, t, acc[0], yt, nb * 64 + c8 + 8 <= p.vy);
  }
  pdl_launch_dependents();
  if (pending) cluster_wait();
}

// ------------------------------------------------------------------ many rows: first product
constexpr int kTile = 64;    // rows of a tile
// ring of 64-wide k chunks: two CTAs' rings of 80 to 96 KB fill an SM's shared memory
template <int MT>
constexpr int kStages = MT == 1 ? 8 : MT == 2 ? 7 : MT == 4 ? 6 : 4;
constexpr int kMaxSplit = 8; // shares of K

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// 8 values (those below `valid`, the rest 0) of a row to a 16-byte place in shared memory
template <bool VEC>
__device__ __forceinline__ void stage8(uint32_t dst, const uint16_t* src, int valid, int w) {
  if (VEC) {
    cp_async16(dst, src, valid >= 8 ? 16 : 0);
  } else if (w >= 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = valid - 2 * i;  // (a row of even length: its last pair is whole)
      cp_async4(dst + 4 * i, n > 0 ? src + 2 * i : src, n > 0 ? 4 : 0);
    }
  } else {
    const uint4 v = load8<false>(src, valid);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
  }
}

// CTA (tile, share of K): scaled sums[share][position][rank], positions in the plan's order. Warp w takes 16 rows
// and half the rank; operands by ldmatrix from rows of 128 bytes whose 16-byte chunks are XORed with the row.
template <int MT, int AT, bool VEC>
__global__ void __launch_bounds__(kLoraThreads) aipu_lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  constexpr int RP = 16 * MT, STAGE = (kTile + RP) * 128, S = kStages<MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();  // (the second product reads the plan, which is complete, before it waits for this)
  const int ti = blockIdx.x / p.ksplit, ks = blockIdx.x - ti * p.ksplit;
  const int4 tile = p.tiles[ti];  // (only tiles below n_tiles are written, but there is room for every ti)
  if (ti >= *p.n_tiles || tile.x < 0) return;
  const LoraTile tl = {tile.x, tile.z, tile.w, 1.f};
  const float scale = p.scale ? p.scale[tile.x] : 1.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunks = (p.K + 63) / 64;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * ks / p.ksplit);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (ks + 1) / p.ksplit);
  // this thread copies chunk tid % 8 of rows tid / 8 and + 32 of x and + 32 i of A
  const int cc = tid & 7, cr = tid >> 3;
  const uint16_t* xs[2];
  int xok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = cr + 32 * i;
    xok[i] = m < tl.rows;
    xs[i] = p.x + static_cast<int64_t>(xok[i] ? p.perm[tile.y + m] : 0) * p.ldx + 8 * cc;
  }
  const uint16_t* as = static_cast<const uint16_t*>(p.a) + (static_cast<int64_t>(tl.id) * p.R + cr) * p.K + 8 * cc;
  constexpr int AI = (RP + 31) / 32;
  const bool arow = RP % 32 == 0 || cr < RP;
  const uint32_t base = smem_u32(smem), at = cr * 128 + ((cc ^ (cr & 7)) << 4);  // (32 rows on: the same chunk)
  int slot = 0;
  auto issue = [&](int c) {
    if (c < c1) {
      const uint32_t st = base + slot * STAGE + at;
      const int k = 64 * c;
      if (VEC && k + 64 <= p.K) {
#pragma unroll
        for (int i = 0; i < 2; ++i) cp_async16(st + 4096 * i, xs[i] + k, xok[i] ? 16 : 0);
#pragma unroll
        for (int i = 0; i < AI; ++i) {
          const bool in = cr + 32 * i < tl.rank;
          if (arow) cp_async16(st + kTile * 128 + 4096 * i, in ? as + static_cast<int64_t>(32 * i) * p.K + k : as, in ? 16 : 0);
        }
      } else {
        const int valid = p.K - k - 8 * cc;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool in = xok[i] && valid > 0;
          stage8<VEC>(st + 4096 * i, in ? xs[i] + k : p.x, in ? valid : 0, p.wx);
        }
#pragma unroll
        for (int i = 0; i < AI; ++i) {
          const bool in = cr + 32 * i < tl.rank && valid > 0;
          if (arow)
            stage8<VEC>(st + kTile * 128 + 4096 * i,
                        in ? as + static_cast<int64_t>(32 * i) * p.K + k : static_cast<const uint16_t*>(p.a), in ? valid : 0, p.wa);
        }
      }
    }
    if (++slot == S) slot = 0;
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(c0 + i);
  float acc[MT][4];  // 8-rank groups of this warp's half
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][q] = 0.f;
  const int tg = 16 * (warp & 3), r0 = 8 * MT * (warp >> 2);
  const int xr = tg + (lane & 15), xh = lane >> 4;  // x row and k half that this lane addresses
  // A: two groups of 8 ranks and their k halves (one group only: its lines are addressed twice)
  const int ar = r0 + (MT == 1 ? (lane & 7) : (lane & 7) + ((lane >> 4) << 3)), ah = (lane >> 3) & 1;
  uint32_t xo[4], ao[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    xo[k] = base + xr * 128 + (((2 * k + xh) ^ (xr & 7)) << 4);
    ao[k] = base + (kTile + ar) * 128 + (((2 * k + ah) ^ (ar & 7)) << 4);
  }
  int use = 0;
  for (int c = c0; c < c1; ++c) {
    cp_wait<S - 2>();
    __syncthreads();
    issue(c + S - 1);
    const uint32_t st = use * STAGE;
    if (++use == S) use = 0;
    float sum[MT][4];  // (rounded adds from chunk to chunk: the MMA's own sums are cut off)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[i][q] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t x[4];
      ldsm4(st + xo[k], x);
#pragma unroll
      for (int i = 0; i < MT; i += 2) {
        uint32_t w[4];
        ldsm4(st + ao[k] + 1024 * i, w);
#pragma unroll
        for (int h = 0; h < (MT == 1 ? 1 : 2); ++h) {
          if (AT == AD_F16) {
            uint32_t h0, l0, h1, l1;
            split_f16(w[2 * h], h0, l0);
            split_f16(w[2 * h + 1], h1, l1);
            mma_bf16_16816(sum[i + h], x[0], x[1], x[2], x[3], l0, l1);
            mma_bf16_16816(sum[i + h], x[0], x[1], x[2], x[3], h0, h1);
          } else {
            mma_bf16_16816(sum[i + h], x[0], x[1], x[2], x[3], w[2 * h], w[2 * h + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][q] = __fadd_rn(acc[i][q], sum[i][q]);
  }
  cp_wait<0>();
  const int g = lane >> 2, t = lane & 3;
  float* dst = p.sums + (static_cast<int64_t>(ks) * p.M + tile.y) * RP;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int m = tg + g + 8 * h;
      if (m < tl.rows)
        *reinterpret_cast<float2*>(dst + static_cast<int64_t>(m) * RP + r0 + 8 * i + 2 * t) =
            make_float2(__fmul_rn(acc[i][2 * h], scale), __fmul_rn(acc[i][2 * h + 1], scale));
    }
}

// ------------------------------------------------------------------ many rows: second product
// CTA (tile, 512 columns of N, 256 where y is fp32): a warp takes 32 columns and all rows of the tile (half of them
// where there are few columns), so every value of B is read and, where it has to be, split or moved into place once. The
// tile's part of y, its rows and its B rows do not depend on the first product: they are on their way (y by
// asynchronous copies) while that runs, so what follows it is the sums of the shares of K in order, the MMAs and
// the stores. All of y passes through shared memory, also where its rows are not aligned or end inside 16 bytes (512 rows
// of 1003 columns, 4 shares of y: 19 us; 67 when the last columns were read by the threads that add to them). Behind a
// GEMM the loads of the shares are what this waits for: several pieces and shares are in flight a thread (28 tiles of
// 502 columns, 2 shares: 18 us; 47 with one after the other). The next B is not fetched ahead: with this many
// accumulators it spills (4096 rows of rank 128, 4096 x 4096: 84 us without, 99 with).
template <bool Y32>
struct ExpandCfg {
  static constexpr int COLS = Y32 ? 256 : 512;
  static constexpr int YPITCH = COLS * (Y32 ? 4 : 2) + 16;  // bytes; rows 2t of a quarter warp on distinct banks
  static constexpr int YBYTES = kTile * YPITCH;
};

template <int AT, bool Y32, bool O32>
__global__ void __launch_bounds__(kLoraThreads, 2) aipu_lora_expand_kernel(const __grid_constant__ LoraParams p) {
  using C = ExpandCfg<Y32>;
  constexpr int NT = kTile / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int tok[kTile];
  uint16_t* hf = reinterpret_cast<uint16_t*>(smem + C::YBYTES);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int ti = blockIdx.x / p.nsplit, np = blockIdx.x - ti * p.nsplit;
  const int4 tile = p.tiles[ti];  // (only tiles below n_tiles are written, but there is room for every ti)
  if (ti >= *p.n_tiles || (tile.x < 0 && p.skip_plain)) {
    pdl_wait();
    return;
  }
  const LoraTile tl = {tile.x, tile.z, tile.w, 1.f};
  if (tid < kTile) tok[tid] = tid < tl.rows ? p.perm[tile.y + tid] : 0;
  __syncthreads();
  constexpr int NS = O32 ? 3 : 2;  // pieces of h
  const int rchunks = (tl.rank + 31) / 32;
  const int hpitch = 32 * ((p.rp + 31) / 32) + 8, hs = kTile * hpitch;
  const int col0 = np * C::COLS, blocks = (min(C::COLS, p.N - col0) + 31) / 32;
  // this warp's first block and rows 8 j0 .. 8 j1 - 1 of the tile
  const bool halves = blocks <= kLoraWarps / 2 && tl.rows > kTile / 2;
  const int first = halves ? warp % (kLoraWarps / 2) : warp, step = halves ? kLoraWarps / 2 : kLoraWarps;
  const int j0 = halves && warp >= kLoraWarps / 2 ? NT / 2 : 0;
  const int rows = halves && warp < kLoraWarps / 2 ? kTile / 2 : tl.rows;
  auto load_y = [&]() {
    constexpr int each = Y32 ? 4 : 8, esz = Y32 ? 4 : 2;  // columns of a 16-byte piece
    const int cols = min(C::COLS, p.N - col0);
    // columns read in whole pieces (all of them where the rows are padded), and the pieces of a row, as a power of two
    const int whole = min((cols + each - 1) / each * each, max(0, p.vy - col0) / each * each);
    const int lg = whole > each ? 32 - __clz(whole / each - 1) : 0, per = 1 << lg;
    const int pieces = whole > 0 ? tl.rows << lg : 0;
    auto at = [&](int i) { return (i & (per - 1)) * each; };
    auto source = [&](int i) {
      return static_cast<const uint8_t*>(p.y) + (static_cast<int64_t>(tok[i >> lg]) * p.ldy + col0 + at(i)) * esz;
    };
    auto place = [&](int i) { return smem + (i >> lg) * C::YPITCH + at(i) * esz; };
    if (Y32 && p.yparts > 1) {
      const int64_t share = static_cast<int64_t>(p.M) * p.ldy;
      for (int i0 = tid; i0 < pieces; i0 += 2 * kLoraThreads) {
        float4 sum[2];
        for (int s0 = 0; s0 < p.yparts; s0 += 4) {  // the loads of four shares of two pieces are in flight together
          float4 v[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int i = i0 + u * kLoraThreads;
            const bool in = i < pieces && at(i) < whole;
#pragma unroll
            for (int s = 0; s < 4; ++s)
              if (in && s0 + s < p.yparts) v[u][s] = *reinterpret_cast<const float4*>(source(i) + 4 * (s0 + s) * share);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              if (s0 + s >= p.yparts) break;
              const float4 o = v[u][s];
              sum[u] = s0 + s == 0 ? o
                                   : make_float4(__fadd_rn(sum[u].x, o.x), __fadd_rn(sum[u].y, o.y), __fadd_rn(sum[u].z, o.z),
                                                 __fadd_rn(sum[u].w, o.w));
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = i0 + u * kLoraThreads;
          if (i < pieces && at(i) < whole) *reinterpret_cast<float4*>(place(i)) = sum[u];
        }
      }
    } else {
      for (int i = tid; i < pieces; i += kLoraThreads)
        if (at(i) < whole) cp_async16(smem_u32(place(i)), source(i), 16);
      // the other columns one at a time, neighbours on neighbouring threads
      const int left = max(0, cols - whole);
#pragma unroll 4
      for (int i = tid; i < tl.rows * left; i += kLoraThreads) {
        const int m = i / left, c = whole + i - m * left;
        const int64_t from = static_cast<int64_t>(tok[m]) * p.ldy + col0 + c;
        if (Y32) *reinterpret_cast<uint32_t*>(smem + m * C::YPITCH + 4 * c) = static_cast<const uint32_t*>(p.y)[from];
        else *reinterpret_cast<uint16_t*>(smem + m * C::YPITCH + 2 * c) = static_cast<const uint16_t*>(p.y)[from];
      }
    }
    cp_commit();
  };
  if (!p.wait_y) load_y();
  uint4 vb[4];
  if (first < blocks && rchunks > 0) load_b<2>(p, tl, col0 + 32 * first + 4 * g, 8 * t, vb);
  pdl_wait();
  if (p.wait_y) load_y();
  // four ranks a thread and step, two steps at a time: their loads of all shares are in flight together
  const int quads = 8 * rchunks, all = tl.rows * quads;
  for (int e0 = tid; e0 < all; e0 += 2 * kLoraThreads) {
    float4 v[2];
    int m[2], r[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = e0 + u * kLoraThreads;
      m[u] = e / quads;
      r[u] = 4 * (e - m[u] * quads);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 4
    for (int s = 0; s < p.ksplit; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (e0 + u * kLoraThreads < all && r[u] < p.rp) {
          const float4 o = *reinterpret_cast<const float4*>(p.sums + (static_cast<int64_t>(s) * p.M + tile.y + m[u]) * p.rp + r[u]);
          v[u] = make_float4(__fadd_rn(v[u].x, o.x), __fadd_rn(v[u].y, o.y), __fadd_rn(v[u].z, o.z), __fadd_rn(v[u].w, o.w));
        }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (e0 + u * kLoraThreads >= all) break;
      // past the rank the sums are 0, or NaN where x is not finite: they count for nothing
      const int left = tl.rank - r[u];
      uint32_t w0[NS], w1[NS];
      pieces<NS>(make_float2(left > 0 ? v[u].x : 0.f, left > 1 ? v[u].y : 0.f), w0);
      pieces<NS>(make_float2(left > 2 ? v[u].z : 0.f, left > 3 ? v[u].w : 0.f), w1);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        *reinterpret_cast<uint2*>(hf + s * hs + m[u] * hpitch + r[u]) = make_uint2(w0[s], w1[s]);
    }
  }
  cp_wait<0>();
  __syncthreads();
  pdl_launch_dependents();
  for (int bk = first; bk < blocks; bk += step) {
    const int c = 32 * bk + 4 * g, n = col0 + c;
    float acc[NT][2][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][q][i] = -0.f;  // y + -0 is y, also for y = -0
    for (int rc = 0; rc < rchunks; ++rc) {
      if (bk != first || rc) load_b<2>(p, tl, n, 32 * rc + 8 * t, vb);
      expand_step<2, NT, AT, NS>(acc, vb, hf, hpitch, hs, j0, rows, rc, lane);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (8 * (j0 + j) >= rows) break;
      YRows<2, Y32> y;
#pragma unroll
      for (int e = 0; e < 2; ++e) y.put(e, smem + (8 * (j0 + j) + 2 * t + e) * C::YPITCH + c * (Y32 ? 4 : 2));
      finish_rows<2, Y32, O32>(p, tok, rows, n, j0 + j, t, acc[j], y, true);
    }
  }
}

// ------------------------------------------------------------------ plan: rows ordered by adapter
// Counting sort of the rows by id in one CTA: perm (rows of an adapter together), and tiles of at most
// kTile of them (with the adapter's rank). Rows of a warp that share an id take one atomic (the rows of a prompt all do). The order
// inside an adapter follows the atomics; a row's result does not depend on its place in a tile.
__global__ void __launch_bounds__(1024) aipu_lora_plan_kernel(const int32_t* __restrict__ ids,
                                                              const int32_t* __restrict__ ranks, int M, int L, int R,
                                                              int32_t* __restrict__ perm, int4* __restrict__ tiles,
                                                              int32_t* __restrict__ n_tiles, int* status) {
  extern __shared__ int cnt[];  // [L + 1]; L = rows without an adapter
  __shared__ int wsum[32], wtile[32];
  constexpr int kHeld = 4;  // ids a thread keeps between the passes
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int held[kHeld];
  auto key = [&](int m) {
    const int v = m < M ? ids[m] : -1;
    if (v >= L && status) atomicOr(status, ST_BAD_ARGS);
    return (v < 0 || v >= L) ? L : v;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = key(tid + 1024 * i);
  for (int i = tid; i <= L; i += 1024) cnt[i] = 0;
  __syncthreads();
  // adds the rows of this warp's lanes to their counters: the lane's place in its counter
  auto add = [&](int k, bool in) {
    const uint32_t same = __match_any_sync(0xffffffffu, in ? k : -1);
    const int first = __ffs(same) - 1;
    int at = 0;
    if (in && lane == first) at = atomicAdd(&cnt[k], __popc(same));
    return __shfl_sync(0xffffffffu, at, first) + __popc(same & ((1u << lane) - 1));
  };
  const int steps = (M + 1023) / 1024;
  for (int i = 0; i < steps; ++i) {
    const int m = tid + 1024 * i;
    int k = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j == i) k = held[j];
    if (i >= kHeld) k = key(m);
    add(k, m < M);
  }
  __syncthreads();
  // exclusive sums over the keys of rows and of tiles; every thread takes a run of keys
  const int per = (L + 1 + 1023) / 1024;
  const int k0 = min(L + 1, tid * per), k1 = min(L + 1, k0 + per);
  int rows = 0, tl = 0;
  for (int k = k0; k < k1; ++k) {
    rows += cnt[k];
    tl += (cnt[k] + kTile - 1) / kTile;
  }
  int ir = rows, it = tl;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, ir, o), b = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) {
      ir += a;
      it += b;
    }
  }
  if (lane == 31) {
    wsum[warp] = ir;
    wtile[warp] = it;
  }
  __syncthreads();
  if (warp == 0) {
    int a = wsum[lane], b = wtile[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int c = __shfl_up_sync(0xffffffffu, a, o), d = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) {
        a += c;
        b += d;
      }
    }
    wsum[lane] = a;
    wtile[lane] = b;
    if (lane == 31) *n_tiles = b;
  }
  __syncthreads();
  int r0 = ir - rows + (warp ? wsum[warp - 1] : 0), t0 = it - tl + (warp ? wtile[warp - 1] : 0);
  for (int k = k0; k < k1; ++k) {
    const int n = cnt[k];
    cnt[k] = r0;
    const int rank = (k == L || n == 0) ? 0 : ranks ? min(max(ranks[k], 0), R) : R;
    for (int i = 0; i < n; i += kTile) tiles[t0++] = make_int4(k == L ? -1 : k, r0 + i, min(kTile, n - i), rank);
    r0 += n;
  }
  __syncthreads();
  for (int i = 0; i < steps; ++i) {
    const int m = tid + 1024 * i;
    int k = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j == i) k = held[j];
    if (i >= kHeld && m < M) {
      const int v = ids[m];
      k = (v < 0 || v >= L) ? L : v;
    }
    const int at = add(k, m < M);
    if (m < M) perm[at] = m;
  }
  pdl_launch_dependents();
}

// ------------------------------------------------------------------ host
static size_t al256l(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
static int64_t max_tiles(int64_t M, int64_t L) { return M / kTile + std::min<int64_t>(L + 1, M); }
static int padded_rank(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }
// shares of K: about two CTAs an SM over the tiles that M rows and L adapters make (a B200's 148 SMs: the workspace is
// sized without a context)
static int k_split(int64_t M, int64_t L) {
  const int64_t tiles = std::max<int64_t>(1, M / kTile + std::min<int64_t>(L, M) / 2);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxSplit, 296 / tiles)));
}

// The one launch: up to 256 rows (a thread each finds the tiles), whose adapters it reads once for every 8 rows.
// 4096 x 4096 in us, against the plan: rank 16, 128 rows on 1 / 8 / 64 adapters 7.6 / 7.5 / 15.6 (17.1 / 12.9 / 25.7), 256
// rows 9.5 / 11.4 / 19.8 (17.2 / 14.4 / 26.2); rank 64, 256 rows 12.5 / 13.7 / 24.5 (22.4 / 17.6 / 32.2); rank 128, 256 rows
// 17.0 / 17.9 / 42 (32.6 / 24.7 / 51), fp16 with fp32 results 29 / 29 / 64 (50 / 40 / 140).
static bool lora_direct(int64_t M) { return M <= kDirectRows; }

size_t lora_plan_bytes(int64_t M, int64_t L, int64_t R) {
  if (lora_direct(M)) return 0;
  return 256 + al256l(4 * M) + al256l(16 * max_tiles(M, L)) +
         al256l(static_cast<size_t>(4) * M * padded_rank(R) * k_split(M, L));
}

static int launch(const void* kern, int grid, int block, size_t smem, cudaStream_t s, bool pdl, void** args,
                  const char* what) {
  if (!pdl) return set_cuda_error(cudaLaunchKernel(kern, dim3(grid), dim3(block), args, smem, s), what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return set_cuda_error(cudaLaunchKernelExC(&cfg, kern, args), what);
}

template <int MT, int AT, bool VEC, bool Y32, bool O32>
static int direct_launch(LoraParams& p, cudaStream_t s, bool pdl) {
  const void* kern = reinterpret_cast<const void*>(aipu_lora_kernel<MT, AT, VEC, Y32, O32>);
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(kern, LoraCfg<MT>::TOTAL, attr, "cudaFuncSetAttribute(lora)");
  if (rc) return rc;
  void* args[1] = {&p};
  // a cluster for every tile that there may be
  const int tiles = std::min(p.M, p.M / kDirectTile + std::min(p.L + 1, p.M));
  return launch(kern, tiles * kDirectCtas, kLoraThreads, LoraCfg<MT>::TOTAL, s, pdl, args, "aipu_lora_kernel");
}
template <int MT, int AT, bool VEC>
static int direct_launch_y(LoraParams& p, cudaStream_t s, bool pdl) {
  if (!p.y_f32) return direct_launch<MT, AT, VEC, false, false>(p, s, pdl);
  return p.out_f32 ? direct_launch<MT, AT, VEC, true, true>(p, s, pdl) : direct_launch<MT, AT, VEC, true, false>(p, s, pdl);
}
template <int MT>
static int direct_launch_t(LoraParams& p, bool vec, cudaStream_t s, bool pdl) {
  if (p.adtype == AD_F16) return vec ? direct_launch_y<MT, AD_F16, true>(p, s, pdl) : direct_launch_y<MT, AD_F16, false>(p, s, pdl);
  return vec ? direct_launch_y<MT, AD_BF16, true>(p, s, pdl) : direct_launch_y<MT, AD_BF16, false>(p, s, pdl);
}

template <int MT, int AT, bool VEC>
static int shrink_launch(LoraParams& p, cudaStream_t s) {
  constexpr int smem = kStages<MT> * (kTile + 16 * MT) * 128;
  const void* kern = reinterpret_cast<const void*>(aipu_lora_shrink_kernel<MT, AT, VEC>);
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(kern, smem, attr, "cudaFuncSetAttribute(lora shrink)");
  if (rc) return rc;
  void* args[1] = {&p};
  return launch(kern, static_cast<int>(max_tiles(p.M, p.L)) * p.ksplit, kLoraThreads, smem, s, true, args,
                "aipu_lora_shrink_kernel");
}
template <int MT>
static int shrink_launch_t(LoraParams& p, bool vec, cudaStream_t s) {
  if (p.adtype == AD_F16) return vec ? shrink_launch<MT, AD_F16, true>(p, s) : shrink_launch<MT, AD_F16, false>(p, s);
  return vec ? shrink_launch<MT, AD_BF16, true>(p, s) : shrink_launch<MT, AD_BF16, false>(p, s);
}

template <int AT, bool Y32, bool O32>
static int expand_launch(LoraParams& p, cudaStream_t s, bool pdl) {
  constexpr int pieces = O32 ? 3 : 2;
  const int smem = ExpandCfg<Y32>::YBYTES + pieces * kTile * (32 * ((p.rp + 31) / 32) + 8) * 2;
  const void* kern = reinterpret_cast<const void*>(aipu_lora_expand_kernel<AT, Y32, O32>);
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(kern, ExpandCfg<Y32>::YBYTES + pieces * kTile * 136 * 2, attr, "cudaFuncSetAttribute(lora expand)");
  if (rc) return rc;
  void* args[1] = {&p};
  return launch(kern, static_cast<int>(max_tiles(p.M, p.L)) * p.nsplit, kLoraThreads, smem, s, pdl, args,
                "aipu_lora_expand_kernel");
}
template <int AT>
static int expand_launch_t(LoraParams& p, cudaStream_t s, bool pdl) {
  if (!p.y_f32) return expand_launch<AT, false, false>(p, s, pdl);
  return p.out_f32 ? expand_launch<AT, true, true>(p, s, pdl) : expand_launch<AT, true, false>(p, s, pdl);
}

// widest load (elements of 16 bits) of rows `ld` elements apart from `ptr`
static int load_width(const void* ptr, int64_t ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
  return (a % 16 == 0 && ld % 8 == 0) ? 8 : (a % 4 == 0 && ld % 2 == 0) ? 2 : 1;
}

int lora_begin(LoraParams& p, void* plan, cudaStream_t s, bool pdl) {
  if (p.L > kMaxAdapters || p.R > 128) return set_error(EINVAL_, "lora: at most 32768 adapters of rank 128");
  if (max_tiles(p.M, p.L) * std::max<int64_t>(kMaxSplit, (p.N + 255) / 256) > INT32_MAX)
    return set_error(EINVAL_, "lora: too many rows and columns for one launch");
  p.skip_plain = (p.out == p.y && p.out_f32 == p.y_f32) ? 1 : 0;
  p.rp = padded_rank(p.R);
  // (an even row length is what the pairwise copies of the first product need of A and x)
  p.wa = load_width(p.a, p.K);
  p.wx = p.K % 2 ? 1 : load_width(p.x, p.ldx);
  p.wb = load_width(p.b, p.R);
  auto rows16 = [](const void* q, int64_t ld, int esz) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld * esz % 16 == 0;
  };
  p.vy = rows16(p.y, p.ldy, p.y_f32 ? 4 : 2) ? (p.y_cols ? p.y_cols : p.N) : 0;
  p.vo = rows16(p.out, p.ldo, p.out_f32 ? 4 : 2) ? 2 : (!p.out_f32 && load_width(p.out, p.ldo) >= 2) ? 1 : 0;
  p.tiles = nullptr;
  if (lora_direct(p.M)) return OK;
  uint8_t* b = static_cast<uint8_t*>(plan);
  p.n_tiles = reinterpret_cast<int32_t*>(b);
  p.perm = reinterpret_cast<int32_t*>(b + 256);
  b += 256 + al256l(4 * static_cast<size_t>(p.M));
  p.tiles = reinterpret_cast<int4*>(b);
  p.sums = reinterpret_cast<float*>(b + al256l(16 * max_tiles(p.M, p.L)));
  p.ksplit = std::min(k_split(p.M, p.L), std::max(1, p.K / 256));  // (of four chunks at least)
  p.nsplit = p.y_f32 ? (p.N + ExpandCfg<true>::COLS - 1) / ExpandCfg<true>::COLS : (p.N + ExpandCfg<false>::COLS - 1) / ExpandCfg<false>::COLS;
  const void* kern = reinterpret_cast<const void*>(aipu_lora_plan_kernel);
  static bool attr[64] = {false};
  int rc = set_smem_attr_once(kern, (kMaxAdapters + 1) * 4, attr, "cudaFuncSetAttribute(lora plan)");
  if (rc) return rc;
  void* args[9] = {&p.ids, &p.ranks, &p.M, &p.L, &p.R, &p.perm, &p.tiles, &p.n_tiles, &p.status};
  if ((rc = launch(kern, 1, 1024, static_cast<size_t>(p.L + 1) * 4, s, pdl, args, "aipu_lora_plan_kernel"))) return rc;
  const bool vec = p.wa == 8 && p.wx == 8;
  switch (p.rp) {
    case 16: return shrink_launch_t<1>(p, vec, s);
    case 32: return shrink_launch_t<2>(p, vec, s);
    case 64: return shrink_launch_t<4>(p, vec, s);
    default: return shrink_launch_t<8>(p, vec, s);
  }
}

int lora_finish(LoraParams& p, cudaStream_t s, bool pdl) {
  if (!p.tiles) {
    const bool vec = p.wa == 8 && p.wx == 8;
    switch (p.rp) {
      case 16: return direct_launch_t<1>(p, vec, s, pdl);
      case 32: return direct_launch_t<2>(p, vec, s, pdl);
      case 64: return direct_launch_t<4>(p, vec, s, pdl);
      default: return direct_launch_t<8>(p, vec, s, pdl);
    }
  }
  return p.adtype == AD_F16 ? expand_launch_t<AD_F16>(p, s, pdl) : expand_launch_t<AD_BF16>(p, s, pdl);
}

}  // namespace aipu
