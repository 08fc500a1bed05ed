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
// One cluster of CTAs takes one tile: up to 8 * NT rows that share an adapter.
//   1. CTA c and its 8 warps each take a share of K. Rank rows are the 16 MMA rows, token rows the 8
//      MMA columns; a lane loads 8 consecutive k of its rows (16 bytes) and uses them as two MMA steps
//      whose k order is permuted the same way on both sides.
//   2. The partial sums are added over the warps in shared memory and over the CTAs through distributed
//      shared memory, always in the same order (no atomics: equal calls give equal bits).
//   3. CTA c and its warps each take 64-column blocks of N. The MMA's rows are columns of y, ordered so
//      that a lane ends with 8 consecutive columns of a row: y is read and written 16 bytes at a time.
// So a call is one launch (and a plan of the rows by adapter when there are more than kDirectRows), h
// never leaves the chip, and the reads of B do not wait for the sums of A.
//
// Rounding: bf16 x and A products are exact in the MMA, sums are fp32. h is not rounded to 16 bits: it
// enters the second product as 2 (bf16 result) or 3 (fp32 result) bf16 pieces, 16 and 24 bits. fp16
// adapters enter as two bf16 pieces (11 bits: exact).
#include <algorithm>

#include "cluster.cuh"
#include "common.cuh"
#include "kernels.h"
#include "launch.h"
#include "lora.cuh"

namespace aipu {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kDirectRows = 64;      // rows for which every cluster finds its tile itself
constexpr int kMaxAdapters = 32768;  // counters of the plan kernel in shared memory

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 consecutive 16-bit values at p (only `valid` of them are read, the others are 0), as four packed
// words. w: widest load that the row's alignment allows (8, 2 or 1 elements).
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int valid, int w) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (VEC) {
    if (valid >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
  }
  if (valid <= 0) return v;
  uint32_t h[4] = {0, 0, 0, 0};
  if (w >= 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i + 1 < valid) h[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
      else if (2 * i < valid) h[i] = __ldg(p + 2 * i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) h[i >> 1] |= static_cast<uint32_t>(__ldg(p + i)) << (16 * (i & 1));
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

// Two floats as packed bf16 pieces: hi truncated (never overflows), lo = the exact rest rounded or
// truncated. A value that is not finite has no rest.
__device__ __forceinline__ bool not_finite(float v) { return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u; }
__device__ __forceinline__ uint32_t piece(float v, float& rest) {
  if (not_finite(v)) {
    rest = 0.f;
    // a NaN keeps a bit that the upper half shows
    return (v != v) ? 0x7FC0u : __float_as_uint(v) >> 16;
  }
  const uint32_t hi = __float_as_uint(v) & 0xFFFF0000u;
  rest = __fsub_rn(v, __uint_as_float(hi));
  return hi >> 16;
}
// packed pair of fp16 -> packed bf16 hi and lo (exact: 11 bits)
__device__ __forceinline__ void split_f16(uint32_t w, uint32_t& hi, uint32_t& lo) {
  float r0, r1;
  const uint32_t h0 = piece(f16_bits_to_f32(w), r0), h1 = piece(f16_bits_to_f32(w >> 16), r1);
  hi = h0 | (h1 << 16);
  lo = (__float_as_uint(r0) >> 16) | (__float_as_uint(r1) & 0xFFFF0000u);
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

template <int MT, int NT>
struct LoraCfg {
  static constexpr int TM = 8 * NT;                  // rows of a tile
  static constexpr int RP = 16 * MT;                 // rank rows
  static constexpr int RF = RP < 32 ? 32 : RP;       // rank columns of the second product (steps of 32)
  static constexpr int HPITCH = RF + 8;              // bf16 pitch of a token's h (16-byte rows, banks spread)
  static constexpr int COPIES = NT == 1 ? kLoraWarps : kLoraWarps / 2;
  static constexpr int OFF_HP = 0;                   // fp32 [TM][RP]: this CTA's sums
  static constexpr int OFF_HF = OFF_HP + TM * RP * 4;  // bf16 [3][TM][HPITCH]: scale * h
  static constexpr int OFF_RED = OFF_HF + 3 * TM * HPITCH * 2;
  static constexpr int TOTAL = OFF_RED + COPIES * TM * RP * 4;
};

struct LoraTile {
  int id, rows, rank;
  float scale;
};

// ------------------------------------------------------------------ first product: this warp's k range
template <int MT, int NT, int AT, bool VEC>
__device__ __forceinline__ void shrink(const LoraParams& p, const int* tok, const LoraTile& tl, int c0, int c1, int lane,
                                       float (&acc)[MT][NT][4]) {
  constexpr int U = NT > 1 ? 1 : (MT == 1 ? 4 : MT == 2 ? 2 : 1);  // k chunks loaded ahead
  const int g = lane >> 2, t = lane & 3;
  const uint16_t* abase = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(tl.id) * p.R * p.K;
  for (int c = c0; c < c1; c += U) {
    uint4 va[U][MT][2], vx[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c + u) * 32 + 8 * t;
      const int valid = (c + u < c1) ? p.K - k : 0;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * i + 8 * h + g;
          va[u][i][h] = load8<VEC>(abase + static_cast<int64_t>(r) * p.K + k, r < tl.rank ? valid : 0, p.wa);
        }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int m = 8 * j + g;
        vx[u][j] = load8<VEC>(p.x + static_cast<int64_t>(tok[m]) * p.ldx + k, m < tl.rows ? valid : 0, p.wx);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (16 * i >= tl.rank) continue;  // warp-uniform
        if (AT == AD_F16) {
          uint4 ah, al, bh, bl;
          split4_f16(va[u][i][0], ah, al);
          split4_f16(va[u][i][1], bh, bl);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (NT > 1 && 8 * j >= tl.rows) continue;
            mma_pair(acc[i][j], ah, bh, vx[u][j]);
            mma_pair(acc[i][j], al, bl, vx[u][j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (NT > 1 && 8 * j >= tl.rows) continue;
            mma_pair(acc[i][j], va[u][i][0], va[u][i][1], vx[u][j]);
          }
        }
      }
  }
}

// ------------------------------------------------------------------ second product and the result rows
// acc2[j][nt]: MMA j's rows g and g + 8 are columns n0 + 8 g + 2 j and + 2 j + 1 of y
template <int NT>
__device__ __forceinline__ void store_rows(const LoraParams& p, const int* tok, int rows, int n0, int lane,
                                           const float (&acc)[4][NT][4], int nt0) {
  const int g = lane >> 2, t = lane & 3;
  const int n = n0 + 8 * g;
  if (n >= p.N) return;
  const int cols = min(8, p.N - n);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = 8 * (nt0 + j) + 2 * t + e;
      if (m >= rows) continue;
      const int64_t row = tok[m];
      float d[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        d[2 * q] = acc[q][j][e];
        d[2 * q + 1] = acc[q][j][2 + e];
      }
      if (p.vy && cols == 8) {
        if (p.y_f32) {
          const float4* yp = reinterpret_cast<const float4*>(static_cast<const float*>(p.y) + row * p.ldy + n);
          const float4 v0 = yp[0], v1 = yp[1];
          d[0] = __fadd_rn(v0.x, d[0]); d[1] = __fadd_rn(v0.y, d[1]); d[2] = __fadd_rn(v0.z, d[2]); d[3] = __fadd_rn(v0.w, d[3]);
          d[4] = __fadd_rn(v1.x, d[4]); d[5] = __fadd_rn(v1.y, d[5]); d[6] = __fadd_rn(v1.z, d[6]); d[7] = __fadd_rn(v1.w, d[7]);
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.y) + row * p.ldy + n);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d[2 * i] = __fadd_rn(__uint_as_float(w[i] << 16), d[2 * i]);
            d[2 * i + 1] = __fadd_rn(__uint_as_float(w[i] & 0xFFFF0000u), d[2 * i + 1]);
          }
        }
        if (p.out_f32) {
          float4* op = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.ldo + n);
          op[0] = make_float4(d[0], d[1], d[2], d[3]);
          op[1] = make_float4(d[4], d[5], d[6], d[7]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = bf16_rne_bits(d[2 * i]) | (static_cast<uint32_t>(bf16_rne_bits(d[2 * i + 1])) << 16);
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.ldo + n) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i >= cols) break;
          const float y = p.y_f32 ? static_cast<const float*>(p.y)[row * p.ldy + n + i]
                                  : bf16_bits_to_f32(static_cast<const uint16_t*>(p.y)[row * p.ldy + n + i]);
          const float v = __fadd_rn(y, d[i]);
          if (p.out_f32) static_cast<float*>(p.out)[row * p.ldo + n + i] = v;
          else static_cast<uint16_t*>(p.out)[row * p.ldo + n + i] = bf16_rne_bits(v);
        }
      }
    }
}

// B rows n0 + 8 g + 2 j (+ 1) for j = 0..3, rank columns r .. r + 7 (past the rank: 0, whatever is stored)
template <bool VEC>
__device__ __forceinline__ void load_b(const LoraParams& p, const LoraTile& tl, int n0, int r, int g, uint4 (&vb)[8]) {
  const uint16_t* bbase = static_cast<const uint16_t*>(p.b) + static_cast<int64_t>(tl.id) * p.N * p.R;
  const int valid = tl.rank - r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + 8 * g + i;
    const uint16_t* row = bbase + static_cast<int64_t>(n) * p.R + r;
    if (VEC) {  // R is a multiple of 8: whole vectors are in the row, the columns past the rank are cleared
      uint4 v = make_uint4(0, 0, 0, 0);
      if (n < p.N && valid > 0) v = __ldg(reinterpret_cast<const uint4*>(row));
      if (valid < 8) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (2 * q >= valid) w[q] = 0;
          else if (2 * q + 1 >= valid) w[q] &= 0xFFFFu;
        }
      }
      vb[i] = v;
    } else {
      vb[i] = load8<false>(row, n < p.N ? valid : 0, p.wb);
    }
  }
}

template <int NTG, int AT>
__device__ __forceinline__ void expand_step(float (&acc)[4][NTG][4], const uint4 (&vb)[8], const uint16_t* hf, int hpitch,
                                            int hsplit, int ns, int nt0, int rows, int rc, int lane) {
  const int g = lane >> 2, t = lane & 3;
  uint4 bh[8], bl[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (AT == AD_F16) split4_f16(vb[i], bh[i], bl[i]);
    else bh[i] = vb[i];
  }
#pragma unroll
  for (int j = 0; j < NTG; ++j) {
    if (8 * (nt0 + j) >= rows) continue;  // warp-uniform
    const uint16_t* hrow = hf + (8 * (nt0 + j) + g) * hpitch + 32 * rc + 8 * t;
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      if (s >= ns) break;  // uniform
      const uint4 h = *reinterpret_cast<const uint4*>(hrow + s * hsplit);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mma_pair(acc[q][j], bh[2 * q], bh[2 * q + 1], h);
        if (AT == AD_F16) mma_pair(acc[q][j], bl[2 * q], bl[2 * q + 1], h);
      }
    }
  }
}

template <int MT, int NT, int AT, bool VEC>
__global__ void __launch_bounds__(kLoraThreads) aipu_lora_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraCfg<MT, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int tok[C::TM];
  float* hp = reinterpret_cast<float*>(smem + C::OFF_HP);
  uint16_t* hf = reinterpret_cast<uint16_t*>(smem + C::OFF_HF);
  float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const int n_clusters = gridDim.x / csize, cl = blockIdx.x / csize;
  const int ns = p.out_f32 ? 3 : 2;
  constexpr int HS = C::TM * C::HPITCH;  // elements of one piece
  // x (and the ids) may come from the kernel before the one that writes y, so they wait too unless the
  // launch says that only y does
  if (!p.wait_y) pdl_wait();
  for (int i = tid; i < 3 * HS / 2; i += kLoraThreads) reinterpret_cast<uint32_t*>(hf)[i] = 0;

  const int total = p.tiles ? *p.n_tiles : p.M;
  bool pending = false;  // a cluster_arrive whose wait is still due
  for (int ti = cl; ti < total; ti += n_clusters) {
    // ---- the tile: rows that share an adapter
    LoraTile tl;
    if (p.tiles) {
      const int4 v = p.tiles[ti];
      tl.id = v.x;
      tl.rows = v.z;
      __syncthreads();  // the last tile's readers of tok are done
      for (int i = tid; i < C::TM; i += kLoraThreads) tok[i] = i < v.z ? p.perm[v.y + i] : 0;
    } else {
      // row ti leads a tile if the number of earlier rows with its id is a multiple of the tile's rows;
      // the tile is that row and the following ones of the id (at most kDirectRows rows in all)
      const int n0 = lane < p.M ? p.ids[lane] : -2, n1 = lane + 32 < p.M ? p.ids[lane + 32] : -2;
      const int mine = p.ids[ti];
      int id = mine;
      if (id < 0 || id >= p.L) {
        if (id >= p.L && crank == 0 && tid == 0 && p.status) atomicOr(p.status, ST_BAD_ARGS);
        id = -1;
      }
      auto same = [&](int v, int row) { return row < p.M && (id < 0 ? (v < 0 || v >= p.L) : v == id); };
      const uint32_t b0 = __ballot_sync(0xffffffffu, same(n0, lane));
      const uint32_t b1 = __ballot_sync(0xffffffffu, same(n1, lane + 32));
      const uint64_t all = static_cast<uint64_t>(b1) << 32 | b0;
      const uint64_t below = (1ull << ti) - 1;
      if (__popcll(all & below) % C::TM != 0) continue;  // the same for every thread of the cluster
      tl.id = id;
      const uint64_t rest = all & ~below;
      tl.rows = min(C::TM, __popcll(rest));
      __syncthreads();
      if (warp == 0) {
        for (int i = lane; i < C::TM; i += 32) tok[i] = 0;
        __syncwarp();
        for (int h = 0; h < 2; ++h) {
          const int row = lane + 32 * h;
          if ((rest >> row) & 1) {
            const int at = __popcll(rest & ((1ull << row) - 1));
            if (at < C::TM) tok[at] = row;
          }
        }
      }
    }
    __syncthreads();
    if (tl.id < 0 && p.skip_plain) continue;  // uniform over the cluster
    tl.rank = 0;
    tl.scale = 1.f;
    if (tl.id >= 0) {
      tl.rank = p.ranks ? min(max(p.ranks[tl.id], 0), p.R) : p.R;
      if (p.scale) tl.scale = p.scale[tl.id];
    }

    const int nblk = (p.N + 63) / 64;
    const int gw = crank * kLoraWarps + warp, nw = csize * kLoraWarps;
    uint4 vb[8];
    if (tl.rank > 0) {
      // ---- first product: this warp's share of K
      float acc[MT][NT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.f;
      const int chunks = (p.K + 31) / 32;
      const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * gw / nw);
      const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (gw + 1) / nw);
      shrink<MT, NT, AT, VEC>(p, tok, tl, c0, c1, lane, acc);
      // the first block's B rows are on the way while the sums are joined
      if (NT == 1 && gw < nblk) load_b<VEC>(p, tl, gw * 64, 8 * t, g, vb);

      // ---- sums over the warps of the CTA, in warp order (fixed tree for the large tile)
      auto put = [&](float* dst) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              dst[(8 * j + 2 * t + (q & 1)) * C::RP + 16 * i + g + 8 * (q >> 1)] = acc[i][j][q];
      };
      if (pending) {  // the other CTAs have read the last tile's sums
        cluster_wait();
        pending = false;
      }
      if (NT == 1) {
        put(red + warp * C::TM * C::RP);
        __syncthreads();
        for (int e = tid; e < C::TM * C::RP; e += kLoraThreads) {
          float v = red[e];
#pragma unroll
          for (int w = 1; w < kLoraWarps; ++w) v = __fadd_rn(v, red[w * C::TM * C::RP + e]);
          hp[e] = v;
        }
      } else {
#pragma unroll
        for (int half = kLoraWarps / 2; half >= 1; half >>= 1) {
          if (warp >= half && warp < 2 * half) put(red + (warp - half) * C::TM * C::RP);
          __syncthreads();
          if (warp < half) {
            const float* src = red + warp * C::TM * C::RP;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  acc[i][j][q] = __fadd_rn(acc[i][j][q],
                                           src[(8 * j + 2 * t + (q & 1)) * C::RP + 16 * i + g + 8 * (q >> 1)]);
          }
          __syncthreads();
        }
        if (warp == 0) put(hp);
      }
      // ---- sums over the CTAs of the cluster, in rank order; h as bf16 pieces in every CTA
      cluster_arrive();
      cluster_wait();
      const uint32_t hpa = smem_u32(hp), hfa = smem_u32(hf);
      const int pairs = tl.rows * C::RP / 2;
      const bool all = pairs <= 2 * kLoraThreads;  // few: every CTA sums all of them (one barrier less)
      const int e0 = all ? 0 : static_cast<int>(pairs * crank / csize);
      const int e1 = all ? pairs : static_cast<int>(pairs * (crank + 1) / csize);
      for (int e = e0 + tid; e < e1; e += kLoraThreads) {
        float2 v = make_float2(0.f, 0.f);
        for (uint32_t c = 0; c < csize; ++c) {
          const float2 o = ld_cluster_f2(map_rank(hpa + 8 * e, c));
          v.x = __fadd_rn(v.x, o.x);
          v.y = __fadd_rn(v.y, o.y);
        }
        const int m = (2 * e) / C::RP, r = 2 * e - m * C::RP;
        // past the rank the sums are 0, or NaN where x is not finite: they count for nothing
        v.x = r < tl.rank ? __fmul_rn(v.x, tl.scale) : 0.f;
        v.y = r + 1 < tl.rank ? __fmul_rn(v.y, tl.scale) : 0.f;
        float r0, r1, q0, q1;
        uint32_t w[3];
        w[0] = piece(v.x, r0) | (piece(v.y, r1) << 16);
        if (ns == 2) {
          w[1] = bf16_rne_bits(r0) | (static_cast<uint32_t>(bf16_rne_bits(r1)) << 16);
        } else {
          w[1] = piece(r0, q0) | (piece(r1, q1) << 16);
          w[2] = (__float_as_uint(q0) >> 16) | (__float_as_uint(q1) & 0xFFFF0000u);
        }
        for (int s = 0; s < ns; ++s) {
          const uint32_t at = hfa + 2 * (s * HS + m * C::HPITCH + r);
          if (all) reinterpret_cast<uint32_t*>(hf)[(s * HS + m * C::HPITCH + r) >> 1] = w[s];
          else
            for (uint32_t c = 0; c < csize; ++c) st_cluster_u32(map_rank(at, c), w[s]);
        }
      }
      cluster_arrive();
      pending = true;
      if (all) {
        __syncthreads();
      } else {
        cluster_wait();
        pending = false;
      }
    }
    if (p.wait_y) pdl_wait();
    // ---- second product: 64-column blocks
    // items: 64-column blocks times groups of NTG token tiles (one pass over the accumulators each)
    constexpr int NTG = NT > 4 ? 4 : NT;
    const int rchunks = (tl.rank + 31) / 32;
    const int items = nblk * ((tl.rows + 8 * NTG - 1) / (8 * NTG));
    for (int it = gw; it < items; it += nw) {
      const int nb = NT > NTG ? it % nblk : it, nt0 = NT > NTG ? (it / nblk) * NTG : 0;
      float acc[4][NTG][4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < NTG; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[q][j][i] = -0.f;  // y + -0 is y, also for y = -0
      for (int rc = 0; rc < rchunks; ++rc) {
        if (NT != 1 || it != gw || rc != 0) load_b<VEC>(p, tl, nb * 64, 32 * rc + 8 * t, g, vb);
        expand_step<NTG, AT>(acc, vb, hf, C::HPITCH, HS, ns, nt0, tl.rows, rc, lane);
      }
      store_rows<NTG>(p, tok, tl.rows, nb * 64, lane, acc, nt0);
    }
    if (!p.tiles) break;  // a cluster per row: this was its only tile
  }
  pdl_launch_dependents();
  if (p.wait_y) pdl_wait();  // a cluster without a tile may not end before what it depends on
  if (pending) cluster_wait();
}

// ------------------------------------------------------------------ plan: rows ordered by adapter
// Counting sort of the rows by id in one CTA: perm (rows of an adapter together), and tiles of at most
// tm of them. The order inside an adapter follows the atomics; a row's result does not depend on its
// place in a tile.
__global__ void __launch_bounds__(1024) aipu_lora_plan_kernel(const int32_t* __restrict__ ids, int M, int L, int tm,
                                                              int32_t* __restrict__ perm, int4* __restrict__ tiles,
                                                              int32_t* __restrict__ n_tiles, int* status) {
  extern __shared__ int cnt[];  // [L + 1]; L = rows without an adapter
  __shared__ int wsum[32], wtile[32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= L; i += 1024) cnt[i] = 0;
  __syncthreads();
  auto key = [&](int m) {
    const int v = ids[m];
    if (v >= L && status) atomicOr(status, ST_BAD_ARGS);
    return (v < 0 || v >= L) ? L : v;
  };
  for (int m = tid; m < M; m += 1024) atomicAdd(&cnt[key(m)], 1);
  __syncthreads();
  // exclusive sums over the keys of rows and of tiles; every thread takes a run of keys
  const int per = (L + 1 + 1023) / 1024;
  const int k0 = min(L + 1, tid * per), k1 = min(L + 1, k0 + per);
  int rows = 0, tl = 0;
  for (int k = k0; k < k1; ++k) {
    rows += cnt[k];
    tl += (cnt[k] + tm - 1) / tm;
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
    for (int i = 0; i < n; i += tm) tiles[t0++] = make_int4(k == L ? -1 : k, r0 + i, min(tm, n - i), 0);
    r0 += n;
  }
  __syncthreads();
  for (int m = tid; m < M; m += 1024) {
    const int v = ids[m];
    perm[atomicAdd(&cnt[(v < 0 || v >= L) ? L : v], 1)] = m;
  }
  pdl_launch_dependents();
}

// ------------------------------------------------------------------ host
static size_t al256l(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
// tiles of 8 rows at least: never more than this
static int64_t plan_max_tiles(int64_t M, int64_t L, int tm) { return M / tm + std::min<int64_t>(L + 1, M); }

size_t lora_plan_bytes(int64_t M, int64_t L) {
  if (M <= kDirectRows) return 0;
  return 256 + al256l(4 * M) + al256l(16 * plan_max_tiles(M, L, 8));
}

template <int MT, int NT, int AT, bool VEC>
static int lora_launch_one(const LoraParams& p, int clusters, int csize, cudaStream_t s, bool pdl) {
  using C = LoraCfg<MT, NT>;
  auto kern = aipu_lora_kernel<MT, NT, AT, VEC>;
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(reinterpret_cast<const void*>(kern), C::TOTAL, attr, "cudaFuncSetAttribute(lora)");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * csize);
  cfg.blockDim = dim3(kLoraThreads);
  cfg.dynamicSmemBytes = C::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = csize;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 2 : 1;
  return set_cuda_error(cudaLaunchKernelEx(&cfg, kern, p), "aipu_lora_kernel");
}

template <int MT, int NT>
static int lora_launch_t(const LoraParams& p, bool vec, int clusters, int csize, cudaStream_t s, bool pdl) {
  if (p.adtype == AD_F16)
    return vec ? lora_launch_one<MT, NT, AD_F16, true>(p, clusters, csize, s, pdl)
               : lora_launch_one<MT, NT, AD_F16, false>(p, clusters, csize, s, pdl);
  return vec ? lora_launch_one<MT, NT, AD_BF16, true>(p, clusters, csize, s, pdl)
             : lora_launch_one<MT, NT, AD_BF16, false>(p, clusters, csize, s, pdl);
}

// widest load (elements of 16 bits) of rows `ld` elements apart from `ptr`
static int load_width(const void* ptr, int64_t ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
  return (a % 16 == 0 && ld % 8 == 0) ? 8 : (a % 4 == 0 && ld % 2 == 0) ? 2 : 1;
}

// Shape of the row tiles. Tiles of 8 rows where the rows of an adapter are few on average, else of 64
// (32 for ranks above 64, whose sums take twice the registers).
struct LoraShape {
  int mt, tm;
  bool wide;
};
static LoraShape lora_shape(const LoraParams& p) {
  LoraShape sh;
  sh.mt = p.R <= 16 ? 1 : p.R <= 32 ? 2 : p.R <= 64 ? 4 : 8;
  sh.wide = p.M > kDirectRows && p.M / std::min(p.L, p.M) > 8;
  sh.tm = !sh.wide ? 8 : sh.mt == 8 ? 32 : 64;
  return sh;
}

int lora_plan_launch(LoraParams& p, void* plan, cudaStream_t s, bool pdl) {
  p.tiles = nullptr;
  if (p.M <= kDirectRows) return OK;
  uint8_t* b = static_cast<uint8_t*>(plan);
  p.n_tiles = reinterpret_cast<int32_t*>(b);
  p.perm = reinterpret_cast<int32_t*>(b + 256);
  p.tiles = reinterpret_cast<int4*>(b + 256 + al256l(4 * static_cast<size_t>(p.M)));
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(reinterpret_cast<const void*>(aipu_lora_plan_kernel), (kMaxAdapters + 1) * 4, attr,
                                    "cudaFuncSetAttribute(lora plan)");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.L + 1) * 4;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  return set_cuda_error(cudaLaunchKernelEx(&cfg, aipu_lora_plan_kernel, p.ids, p.M, p.L, lora_shape(p).tm, p.perm, p.tiles,
                                           p.n_tiles, p.status),
                        "aipu_lora_plan_kernel");
}

int lora_launch(LoraParams p, int num_sms, cudaStream_t s, bool pdl) {
  if (p.M <= 0 || p.N <= 0) return OK;
  if (p.L > kMaxAdapters || p.R > 128) return set_error(EINVAL_, "lora: at most 32768 adapters of rank 128");
  p.skip_plain = (p.out == p.y && p.out_f32 == p.y_f32) ? 1 : 0;
  p.wa = load_width(p.a, p.K);
  p.wx = load_width(p.x, p.ldx);
  p.wb = load_width(p.b, p.R);
  const bool vec = p.wa == 8 && p.wx == 8 && p.wb == 8;
  auto rows16 = [](const void* q, int64_t ld, int esz) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld * esz % 16 == 0;
  };
  p.vy = rows16(p.y, p.ldy, p.y_f32 ? 4 : 2) && rows16(p.out, p.ldo, p.out_f32 ? 4 : 2);
  const LoraShape sh = lora_shape(p);
  int clusters = p.M, csize = 8;
  if (p.tiles) {
    const int64_t tiles = plan_max_tiles(p.M, p.L, sh.tm);
    csize = tiles >= 2 * num_sms ? 2 : tiles >= num_sms / 2 ? 4 : 8;
    clusters = static_cast<int>(std::min<int64_t>(tiles, 4 * num_sms / csize));
  }
  if (sh.wide) {
    switch (sh.mt) {
      case 1: return lora_launch_t<1, 8>(p, vec, clusters, csize, s, pdl);
      case 2: return lora_launch_t<2, 8>(p, vec, clusters, csize, s, pdl);
      case 4: return lora_launch_t<4, 8>(p, vec, clusters, csize, s, pdl);
      default: return lora_launch_t<8, 4>(p, vec, clusters, csize, s, pdl);
    }
  }
  switch (sh.mt) {
    case 1: return lora_launch_t<1, 1>(p, vec, clusters, csize, s, pdl);
    case 2: return lora_launch_t<2, 1>(p, vec, clusters, csize, s, pdl);
    case 4: return lora_launch_t<4, 1>(p, vec, clusters, csize, s, pdl);
    default: return lora_launch_t<8, 1>(p, vec, clusters, csize, s, pdl);
  }
}

}  // namespace aipu
