// Penalties, biases and masks of many requests on their logits, and the greedy token, sm_100a.
//
//   z = fp32(logit)
//   z = z > 0 ? z / repetition : z * repetition     if v occurs in the row's context
//   z = z - frequency * count;  z = z - presence    if v occurs count > 0 times in its generated part
//   z = z + bias                                    every entry of the row's list for v, in list order
//   z = -inf                                        if the row's mask does not allow v
//   token = lowest v of the largest z; -1 if no z is above -inf
//
// Every step is rounded to fp32 by itself, so the values (and so the token) are those of any program
// that takes the same steps. NaN is never the largest.
//
// Bound: each logit is read once and each result written once; the rest (contexts, masks, biases) is
// small, so the operator should be bound by memory for many rows and by latency for one. Measured (device time in
// a graph): 64 bf16 rows of 128000 14.7 us without controls (3.3 TB/s), 31 us with contexts of 4000 to 8000
// tokens, biases and masks; 256 fp32 rows of 50001 30 and 40 us; one row of 32000 3.6 and 6.9 us.
//
// One cluster of CTAs takes one row; blocks of tokens go to its CTAs in turn (frequent tokens are
// neighbours, and their counting should not fall to one CTA). The counts of a CTA's blocks are built in its
// shared memory from the row's context, which each CTA scans whole (from L2 after the first): no table of
// counts in global memory, nothing to reset or to keep from call to call, and rows may share a context (the
// rows of a verify pass do). (Sharing the scan out and counting by atomics in distributed shared memory was no
// faster: 64 rows with contexts of 4000 to 8000 tokens 34.5 us against 32.4. A remote atomic costs about what the
// compares that it saves do.) Integer atomics only, so the order changes nothing.
// The tokens that a penalty changes are few among the vocabulary: the pass over it stores a lane's tokens as
// they are and then finishes those with a count one by one (a branch for each would be taken by most warps
// for the sake of a lane). Tokens with a bias are finished by the entries of the bias list after that.
// A warp takes a block, a lane the neighbouring tokens of one 16-byte load: 4 of fp32, 8 of bf16. (8 of fp32,
// in two loads that each skip every other 16 bytes, lean on an L1 cache that the counts leave little of: 256
// rows took twice as long.) Rows of odd length start at any element, so the blocks are laid from the row's
// last 16-byte boundary on. A warp's loads are issued a batch of blocks ahead, the first before the context
// is counted. The token is reduced over the cluster through distributed shared memory.
#include <algorithm>
#include <climits>

#include "cluster.cuh"
#include "common.cuh"
#include "launch.h"
#include "logits.cuh"

namespace aipu {

// tokens of a lane's group and of a warp's block
__host__ __device__ constexpr int group_tokens(bool f32) { return f32 ? 4 : 8; }
constexpr int block_tokens(bool f32) { return 32 * group_tokens(f32); }
constexpr int kMaxFields = 40960;  // tokens of a CTA and window: 80 KB of counts, two CTAs an SM
// A token's field takes 16 bits, 32 in rows that generated more than 14 bits count (their windows are half
// as long): the count, a bit for a token with a bias, and the upper bit for one of the prompt.
constexpr int kMaxCount16 = 0x3FFF;

// Tokens with several bias entries that are kept apart: the entries of the others need not look through the row's list. (In a
// list with more of them each entry does: 20000 entries of 32000 tokens, one repeated, took 55 ms so and take 1.7. Looking
// through by whole warps brings 0.2 and costs registers: 256 fp32 rows with biases 40.3 -> 43.9 us.)
constexpr int kMaxTwice = 64;

struct Best {
  float z;
  int v;
};
// larger value, then lower token; NaN never wins
__device__ __forceinline__ void take(Best& b, float z, int v) {
  if (z > b.z || (z == b.z && v < b.v && z > -INFINITY)) {
    b.z = z;
    b.v = v;
  }
}

__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float z = __shfl_xor_sync(0xffffffffu, b.z, d);
    const int v = __shfl_xor_sync(0xffffffffu, b.v, d);
    take(b, z, v);
  }
  return b;
}

struct RowPenalty {
  float rep, pres, freq;
};
// n: how often the token was generated; it occurs in the context
__device__ __forceinline__ float penalise(float z, uint32_t n, const RowPenalty& r) {
  z = z > 0.f ? __fdiv_rn(z, r.rep) : __fmul_rn(z, r.rep);
  if (n) {
    z = __fsub_rn(z, __fmul_rn(r.freq, static_cast<float>(n)));
    z = __fsub_rn(z, r.pres);
  }
  return z;
}

template <bool F32>
__device__ __forceinline__ float load_logit(const uint8_t* row, int v) {
  if (F32) return reinterpret_cast<const float*>(row)[v];
  return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[v]);
}

// the G logits from v0 on of a row of V (v0 may be below 0 or V - v0 below G: those values are 0) and their
// mask bits (of tokens 0 .. V - 1 only)
template <bool F32>
struct Group {
  static constexpr int G = group_tokens(F32);
  uint32_t q[4];
  uint32_t ok;
  static __device__ __forceinline__ uint32_t inside(int v0, int V) {
    if (v0 >= 0 && v0 + G <= V) return (1u << G) - 1;
    uint32_t in = 0;
#pragma unroll
    for (int j = 0; j < G; ++j) in |= static_cast<uint32_t>(v0 + j >= 0 && v0 + j < V) << j;
    return in;
  }
  __device__ __forceinline__ void load(const uint8_t* row, const uint32_t* mask, int v0, int V) {
    ok = inside(v0, V);
    if (ok == (1u << G) - 1) {
      const uint4 t = __ldcs(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(v0) * (F32 ? 4 : 2)));
      q[0] = t.x; q[1] = t.y; q[2] = t.z; q[3] = t.w;
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const float z = (ok >> j & 1u) ? load_logit<F32>(row, v0 + j) : 0.f;
        if (F32) q[j & 3] = __float_as_uint(z);
        else if (j & 1) q[j >> 1] |= __float_as_uint(z) & 0xFFFF0000u;
        else q[j >> 1] = __float_as_uint(z) >> 16;
      }
    }
    if (mask && ok) {
      const int at = max(v0, 0), last = min(v0 + G, V) - 1;  // the tokens of the group that there are
      const uint32_t lo = __ldg(mask + (at >> 5));
      const uint32_t hi = (at >> 5) < (last >> 5) ? __ldg(mask + (last >> 5)) : 0u;
      ok &= __funnelshift_r(lo, hi, at & 31) << (at - v0);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if (F32) return __uint_as_float(q[j & 3]);
    return __uint_as_float((j & 1) ? q[j >> 1] & 0xFFFF0000u : q[j >> 1] << 16);
  }
};

template <bool F32, int T>
__global__ void __launch_bounds__(T, T == 256 ? 4 : 1) aipu_logits_kernel(const __grid_constant__ LogitParams p) {
  extern __shared__ __align__(16) uint32_t smem_u[];
  constexpr int G = group_tokens(F32), kBlock = block_tokens(F32), kShift = F32 ? 7 : 8;
  constexpr uint32_t kAll = (1u << G) - 1;
  uint32_t* cnt = smem_u;     // [blocks][kBlock] fields (with spans or biases)
  __shared__ Best wbest[32];
  __shared__ Best cbest[16];  // per CTA of the cluster, in the CTA of rank 0
  __shared__ int n_twice, twice[kMaxTwice];  // tokens with two or more entries in the bias list (one too many: any may be)
  constexpr int nt = T, nw = T / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t crank = cluster_rank(), csize = cluster_size();  // a power of two
  const int cshift = 31 - __clz(csize);
  const int m = blockIdx.x >> cshift;
  auto clear = [&]() {
    if (p.spans || p.bias_begin) {
      for (int i = tid; i < p.blocks * (kBlock / 8); i += nt) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) n_twice = 0;
    }
  };
  clear();
  cluster_arrive();  // waited for before the first store to another CTA: all have started by then
  pdl_wait();

  const uint8_t* row = static_cast<const uint8_t*>(p.logits) + m * p.ld * (F32 ? 4 : 2);
  float* out = p.out ? p.out + m * p.ldo : nullptr;
  // token v is element v + o of the blocks, which start at a 16-byte boundary
  const int o = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15u) / (F32 ? 4 : 2);
  const bool ovec = (reinterpret_cast<uintptr_t>(out - o) & 15u) == 0;
  const int nblocks = (p.V + o + kBlock - 1) / kBlock;
  // group of this lane in local block lb of the window that starts at block b0: its first token
  auto first = [&](int b0, int lb) { return (b0 + (lb << cshift) + static_cast<int>(crank)) * kBlock + G * lane - o; };

  bool bad = false;
  // ---- the row's controls
  RowPenalty pen = {1.f, 0.f, 0.f};
  int cb = 0, cg = 0, ce = 0;  // (fewer than 2^30 tokens: a count fits below the marks of a 32-bit field)
  if (p.spans) {
    const int64_t b = p.spans[3 * m], g = p.spans[3 * m + 1], e = p.spans[3 * m + 2];
    cb = static_cast<int>(min(max(b, static_cast<int64_t>(0)), p.n_tokens));
    ce = static_cast<int>(min(max(e, static_cast<int64_t>(cb)), p.n_tokens));
    cg = static_cast<int>(min(max(g, static_cast<int64_t>(cb)), static_cast<int64_t>(ce)));
    bad = cb != b || cg != g || ce != e;
    pen = {p.penalties[3 * m], p.penalties[3 * m + 1], p.penalties[3 * m + 2]};
  }
  const bool penal = ce > cb && !(pen.rep == 1.f && pen.pres == 0.f && pen.freq == 0.f);
  int64_t bb = 0, be = 0;
  if (p.bias_begin) {
    const int64_t b = p.bias_begin[m], e = p.bias_begin[m + 1];
    bb = min(max(b, static_cast<int64_t>(0)), p.n_bias);
    be = min(max(e, bb), p.n_bias);
    bad = bad || bb != b || be != e;
  }
  const bool some = be > bb;
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int r = p.mask_rows[m];
    if (r >= p.n_masks) bad = true;
    else if (r >= 0) mask = p.mask + static_cast<int64_t>(r) * ((p.V + 31) / 32);
  }
  if (bad && tid == 0 && crank == 0 && p.status) atomicOr(p.status, ST_BAD_ARGS);
  // the first bias entry of this thread, on its way while the context is counted
  int bid = 0;
  float bval = 0.f;
  if (bb + tid < be) {
    bid = p.bias_ids[bb + tid];
    bval = p.bias_vals[bb + tid];
  }
  const bool wide = penal && ce - cg > kMaxCount16;
  const int cbits = wide ? 32 : 16;
  const uint32_t seen = 1u << (cbits - 1), biased = seen >> 1;
  const int blocks = wide ? p.blocks / 2 : p.blocks;  // p.blocks is even where a window does not hold the row

  Best best = {-INFINITY, INT_MAX};
  const int window = blocks << cshift;
  for (int b0 = 0; b0 < nblocks; b0 += window) {
    // this CTA's blocks of the window
    const int mine = min(blocks, (nblocks - b0 - static_cast<int>(crank) + static_cast<int>(csize) - 1) >> cshift);
    // word and shift of token v's field; false if another CTA or window has it
    auto place = [&](int32_t v, uint32_t& word, int& sh) {
      const uint32_t u = static_cast<uint32_t>(v) + static_cast<uint32_t>(o);
      const uint32_t b = (u >> kShift) - static_cast<uint32_t>(b0);  // (b0 is a multiple of the cluster's size)
      if ((b & (csize - 1)) != crank || static_cast<uint32_t>(v) >= static_cast<uint32_t>(p.V) ||
          b >= static_cast<uint32_t>(window))
        return false;
      const uint32_t i = (b >> cshift << kShift) + (u & (kBlock - 1));
      word = wide ? i : i >> 1;
      sh = wide ? 0 : 16 * (i & 1);
      return true;
    };
    auto allowed = [&](int v) { return !mask || (__ldg(mask + (v >> 5)) >> (v & 31) & 1u); };
    if (b0 > 0) {
      __syncthreads();  // the last window's fields are read
      clear();
    }
    constexpr int D = 2;  // blocks of a batch
    Group<F32> cur[D], nxt[D];
    auto fetch = [&](Group<F32>(&g)[D], int lb) {
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (lb + d * nw < mine) g[d].load(row, mask, first(b0, lb + d * nw), p.V);
    };
    fetch(cur, warp);
    if (penal || some) __syncthreads();
    // ---- counts, and marks of the tokens with a bias
    if (some)
      for (int64_t i = bb + tid; i < be; i += nt) {
        uint32_t word;
        int sh;
        const int v = i == bb + tid ? bid : p.bias_ids[i];
        if (place(v, word, sh) && (atomicOr(&cnt[word], biased << sh) >> sh & biased)) {
          const int k = atomicAdd(&n_twice, 1);
          if (k < kMaxTwice) twice[k] = v;
        }
      }
    if (penal) {
      auto count = [&](int32_t t, int at) {
        uint32_t word;
        int sh;
        if (!place(t, word, sh)) return;
        if (at >= cg) atomicAdd(&cnt[word], 1u << sh);
        else atomicOr(&cnt[word], seen << sh);
      };
      // 16-byte loads of the context between its unaligned ends
      const int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p.tokens + cb) & 15u)) & 15u) / 4;
      const int a0 = min(ce - cb, head) + cb, nv = (ce - a0) / 4, t0 = a0 + 4 * nv;
      const int4* tv = reinterpret_cast<const int4*>(p.tokens + a0);
      for (int i = tid; i < nv; i += 4 * nt) {
        int4 q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (u * nt < nv - i) q[u] = __ldg(tv + i + u * nt);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u * nt >= nv - i) break;
          const int at = a0 + 4 * (i + u * nt);
          count(q[u].x, at);
          count(q[u].y, at + 1);
          count(q[u].z, at + 2);
          count(q[u].w, at + 3);
        }
      }
      if (tid < a0 - cb) count(p.tokens[cb + tid], cb + tid);
      if (tid < ce - t0) count(p.tokens[t0 + tid], t0 + tid);
    }
    if (penal || some) __syncthreads();
    // ---- the pass
    for (int lb0 = warp; lb0 < mine; lb0 += D * nw) {
      fetch(nxt, lb0 + D * nw);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int lb = lb0 + d * nw;
        if (lb >= mine) break;
        const int v0 = first(b0, lb);
        const uint32_t in = Group<F32>::inside(v0, p.V), ok = cur[d].ok;
        float z[G];
#pragma unroll
        for (int j = 0; j < G; ++j) z[j] = cur[d].get(j);
        if (ok != kAll) {
#pragma unroll
          for (int j = 0; j < G; ++j)
            if (!(ok >> j & 1u)) z[j] = -INFINITY;
        }
        if (out) {
          if (in == kAll && ovec) {
#pragma unroll
            for (int j = 0; j < G; j += 4) *reinterpret_cast<float4*>(out + v0 + j) = make_float4(z[j], z[j + 1], z[j + 2], z[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < G; ++j)
              if (in >> j & 1u) out[v0 + j] = z[j];
          }
        }
        if (penal || some) {
          // the group's fields: two of 16 bits a word, or one of 32
          uint32_t w[G];
          const uint32_t* f = cnt + (lb * 32 + lane) * (wide ? G : G / 2);
          if (wide) {
#pragma unroll
            for (int j = 0; j < G; j += 4) {
              const uint4 c = *reinterpret_cast<const uint4*>(f + j);
              w[j] = c.x; w[j + 1] = c.y; w[j + 2] = c.z; w[j + 3] = c.w;
            }
          } else {
            uint32_t h[G / 2];
            if constexpr (F32) {
              const uint2 c = *reinterpret_cast<const uint2*>(f);
              h[0] = c.x; h[1] = c.y;
            } else {
              const uint4 c = *reinterpret_cast<const uint4*>(f);
              h[0] = c.x; h[1] = c.y; h[G / 2 - 2] = c.z; h[G / 2 - 1] = c.w;
            }
#pragma unroll
            for (int j = 0; j < G; ++j) w[j] = (j & 1) ? h[j >> 1] >> 16 : h[j >> 1] & 0xFFFFu;
          }
          uint32_t any = 0;
#pragma unroll
          for (int j = 0; j < G; ++j) any |= w[j];
          if (any) {
            // finished one by one, or (with a bias) after the pass; masked ones and those past the row are finished
            uint32_t todo = 0;
            float keep[G];
#pragma unroll
            for (int j = 0; j < G; ++j) {
              keep[j] = z[j];
              if (w[j]) {
                todo |= (w[j] & biased) ? 0u : 1u << j;
                z[j] = -INFINITY;
              }
            }
            todo &= ok;
#pragma unroll 1
            while (todo) {
              const int j = __ffs(todo) - 1;
              todo &= todo - 1;
              float v = keep[0];
#pragma unroll
              for (int i = 1; i < G; ++i) v = i == j ? keep[i] : v;
              const uint32_t n = (wide ? f[j] : f[j >> 1] >> (16 * (j & 1)) & 0xFFFFu) & (biased - 1);
              v = penalise(v, n, pen);
              take(best, v, v0 + j);
              if (out) out[v0 + j] = v;
            }
          }
        }
        // (the larger of a number and NaN is the number; what is outside the row is -inf)
        float top = z[0];
#pragma unroll
        for (int j = 1; j < G; ++j) top = fmaxf(top, z[j]);
        if (top >= best.z && top > -INFINITY) {
#pragma unroll
          for (int j = G - 1; j >= 0; --j)
            if (z[j] == top) take(best, top, v0 + j);
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d) cur[d] = nxt[d];
    }
    // ---- tokens with a bias
    if (some) {
      __syncthreads();  // the pass has stored them as they are (in place too: or as -inf, where the mask says so)
      for (int64_t i = bb + tid; i < be; i += nt) {
        const int v = i == bb + tid ? bid : p.bias_ids[i];
        uint32_t word;
        int sh;
        if (!place(v, word, sh)) continue;
        float z = load_logit<F32>(row, v);
        const uint32_t w = cnt[word] >> sh & (seen | (biased - 1));
        if (w) z = penalise(z, w & (biased - 1), pen);
        bool several = n_twice > kMaxTwice;
        for (int k = 0; k < min(n_twice, kMaxTwice) && !several; ++k) several = twice[k] == v;
        if (!several) {
          z = __fadd_rn(z, i == bb + tid ? bval : p.bias_vals[i]);
        } else {  // all entries of the token, in list order, by the thread of the first one
          bool lead = true;
          for (int64_t j = bb; j < be && lead; ++j)
            if (p.bias_ids[j] == v) {
              if (j < i) lead = false;
              else z = __fadd_rn(z, p.bias_vals[j]);
            }
          if (!lead) continue;
        }
        if (!allowed(v)) z = -INFINITY;
        take(best, z, v);
        if (out) out[v] = z;
      }
    }
  }
  if (!p.token) {
    cluster_wait();
    return;
  }
  // ---- the greedy token of the row
  best = warp_best(best);
  cluster_wait();
  // the warps' tokens, then (in the CTA of rank 0) the CTAs': a lane each
  if (lane == 0) wbest[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = lane < nw ? wbest[lane] : Best{-INFINITY, INT_MAX};
    best = warp_best(best);
    if (lane == 0) {
      const uint32_t at = map_rank(smem_u32(&cbest[crank]), 0);
      st_cluster_u32(at, __float_as_uint(best.z));
      st_cluster_u32(at + 4, static_cast<uint32_t>(best.v));
    }
    __syncwarp();
  }
  cluster_arrive();
  cluster_wait();
  if (crank == 0 && warp == 0) {
    best = warp_best(lane < csize ? cbest[lane] : Best{-INFINITY, INT_MAX});
    if (lane == 0) p.token[m] = best.v == INT_MAX ? -1 : best.v;
  }
}

template <bool F32, int T>
static int logits_launch_t(const LogitParams& p, int csize, int smem, cudaStream_t s, bool pdl) {
  auto kern = aipu_logits_kernel<F32, T>;
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(reinterpret_cast<const void*>(kern), kMaxFields * 2, attr,
                                    "cudaFuncSetAttribute(logits)");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.M * csize);
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = csize;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 2 : 1;
  return set_cuda_error(cudaLaunchKernelEx(&cfg, kern, p), "aipu_logits_kernel");
}

int logits_launch(LogitParams p, int num_sms, cudaStream_t s, bool pdl) {
  if (p.M <= 0 || p.V <= 0) return OK;
  const int bt = block_tokens(p.f32 != 0);
  // (a row's blocks start up to a group before it)
  const int row_blocks = (p.V + group_tokens(p.f32 != 0) - 1 + bt - 1) / bt;
  // CTAs of a row: 8, fewer where there are rows enough to fill the SMs (three CTAs each) with fewer, as long as
  // a CTA's counts leave room for four. Few rows: 512 threads, so that a row's loads are in flight at once; else
  // 256, whose CTAs overlap one another's phases.
  int csize = 8;
  while (csize > 1 && static_cast<int64_t>(p.M) * csize / 2 >= 3 * num_sms && (row_blocks + csize / 2 - 1) / (csize / 2) * bt <= 25600)
    csize /= 2;
  const bool few = static_cast<int64_t>(p.M) * csize <= num_sms;
  p.blocks = std::min(kMaxFields / bt, ((row_blocks + csize - 1) / csize + 1) / 2 * 2);
  const int smem = (p.spans || p.bias_begin) ? p.blocks * bt * 2 : 0;
  if (p.f32)
    return few ? logits_launch_t<true, 512>(p, csize, smem, s, pdl) : logits_launch_t<true, 256>(p, csize, smem, s, pdl);
  return few ? logits_launch_t<false, 512>(p, csize, smem, s, pdl) : logits_launch_t<false, 256>(p, csize, smem, s, pdl);
}

}  // namespace aipu
