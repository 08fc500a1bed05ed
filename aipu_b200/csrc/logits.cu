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
// small, so the operator is bound by memory for many rows and by latency for one.
//
// One cluster of CTAs takes one row; every CTA a slice of the vocabulary. The counts of the slice are
// built in shared memory from the row's context, which each CTA scans whole (from L2 after the first):
// no table of counts in global memory, nothing to reset or to keep from call to call, and rows may share
// a context (the rows of a verify pass do). Integer atomics only, so the order changes nothing. A warp
// takes 32 neighbouring tokens: its mask is one word. Tokens with a bias are few: they are finished
// first, marked in a bitmap and left out of the pass over the slice. The token is reduced over the
// cluster through distributed shared memory.
#include <algorithm>
#include <climits>

#include "cluster.cuh"
#include "common.cuh"
#include "launch.h"
#include "logits.cuh"

namespace aipu {

constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the other bits count the generated part
constexpr int kMaxSlice = 24576;         // tokens: 96 KB of counts, two CTAs an SM

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

struct RowPenalty {
  float rep, pres, freq;
};
__device__ __forceinline__ float penalise(float z, uint32_t w, const RowPenalty& r) {
  if (w == 0) return z;
  z = z > 0.f ? __fdiv_rn(z, r.rep) : __fmul_rn(z, r.rep);
  const uint32_t n = w & ~kSeen;
  if (n) {
    z = __fsub_rn(z, __fmul_rn(r.freq, static_cast<float>(n)));
    z = __fsub_rn(z, r.pres);
  }
  return z;
}

template <bool F32>
__device__ __forceinline__ float load_logit(const void* row, int v) {
  if (F32) return static_cast<const float*>(row)[v];
  return bf16_bits_to_f32(static_cast<const uint16_t*>(row)[v]);
}

template <bool F32>
__global__ void __launch_bounds__(1024) aipu_logits_kernel(const __grid_constant__ LogitParams p) {
  extern __shared__ __align__(16) uint32_t smem_u[];
  uint32_t* cnt = smem_u;                                          // [slice] (with spans)
  uint32_t* biased = smem_u + (p.spans ? p.slice : 0);              // [slice / 32] (with biases)
  __shared__ Best wbest[32];
  __shared__ Best cbest[16];  // per CTA of the cluster, in the CTA of rank 0
  __shared__ int twice;       // a token has two entries in the bias list
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  const uint32_t crank = cluster_rank(), csize = cluster_size();
  cluster_arrive();  // waited for before the first store to another CTA: all have started by then
  const int m = blockIdx.x / csize;
  pdl_wait();

  const uint8_t* row = static_cast<const uint8_t*>(p.logits) + m * p.ld * (F32 ? 4 : 2);
  float* out = p.out ? p.out + m * p.ldo : nullptr;
  bool bad = false;
  // ---- the row's controls
  RowPenalty pen = {1.f, 0.f, 0.f};
  int64_t cb = 0, cg = 0, ce = 0;
  if (p.spans) {
    const int64_t b = p.spans[3 * m], g = p.spans[3 * m + 1], e = p.spans[3 * m + 2];
    cb = min(max(b, static_cast<int64_t>(0)), p.n_tokens);
    ce = min(max(e, cb), p.n_tokens);
    cg = min(max(g, cb), ce);
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
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int r = p.mask_rows[m];
    if (r >= p.n_masks) bad = true;
    else if (r >= 0) mask = p.mask + static_cast<int64_t>(r) * ((p.V + 31) / 32);
  }
  if (bad && tid == 0 && crank == 0 && p.status) atomicOr(p.status, ST_BAD_ARGS);

  Best best = {-INFINITY, INT_MAX};
  const int window = p.slice * csize;
  for (int w0 = 0; w0 < p.V; w0 += window) {
    const int s0 = min(p.V, w0 + static_cast<int>(crank) * p.slice), s1 = min(p.V, s0 + p.slice);
    const int len = s1 - s0;
    if (w0 > 0) __syncthreads();  // the last window's counts are read
    // ---- counts of the slice
    if (penal)
      for (int i = tid; i < len; i += nt) cnt[i] = 0;
    if (be > bb) {
      for (int i = tid; i < (len + 31) / 32; i += nt) biased[i] = 0;
      if (tid == 0) twice = 0;
    }
    if (penal || be > bb) __syncthreads();
    if (penal) {
      auto count = [&](int32_t t, int64_t at) {
        const uint32_t i = static_cast<uint32_t>(t) - static_cast<uint32_t>(s0);
        if (i < static_cast<uint32_t>(len)) {
          if (at >= cg) atomicAdd(&cnt[i], 1u);
          else atomicOr(&cnt[i], kSeen);
        }
      };
      // 16-byte loads of the context between its unaligned ends
      const int64_t a0 = min(ce, cb + static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p.tokens + cb) & 15u)) & 15u) / 4);
      const int64_t nv = (ce - a0) / 4;
      if (tid < a0 - cb) count(p.tokens[cb + tid], cb + tid);
      const int4* tv = reinterpret_cast<const int4*>(p.tokens + a0);
      for (int64_t i = tid; i < nv; i += 4 * nt) {
        int4 q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = (i + u * nt < nv) ? __ldg(tv + i + u * nt) : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t at = a0 + 4 * (i + u * nt);
          count(q[u].x, at);
          count(q[u].y, at + 1);
          count(q[u].z, at + 2);
          count(q[u].w, at + 3);
        }
      }
      const int64_t t0 = a0 + 4 * nv;
      if (tid < ce - t0) count(p.tokens[t0 + tid], t0 + tid);
    }
    // ---- tokens with a bias: marked, then finished here
    if (be > bb) {
      for (int64_t i = bb + tid; i < be; i += nt) {
        const uint32_t at = static_cast<uint32_t>(p.bias_ids[i]) - static_cast<uint32_t>(s0);
        if (at < static_cast<uint32_t>(len) && (atomicOr(&biased[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u)) twice = 1;
      }
    }
    if (penal || be > bb) __syncthreads();
    if (be > bb) {
      for (int64_t i = bb + tid; i < be; i += nt) {
        const int v = p.bias_ids[i];
        const uint32_t at = static_cast<uint32_t>(v) - static_cast<uint32_t>(s0);
        if (at >= static_cast<uint32_t>(len)) continue;
        float z = load_logit<F32>(row, v);
        if (penal) z = penalise(z, cnt[at], pen);
        if (!twice) {
          z = __fadd_rn(z, p.bias_vals[i]);
        } else {  // all entries of the token, in list order, by the thread of the first one
          bool first = true;
          for (int64_t j = bb; j < be && first; ++j)
            if (p.bias_ids[j] == v) {
              if (j < i) first = false;
              else z = __fadd_rn(z, p.bias_vals[j]);
            }
          if (!first) continue;
        }
        if (mask && !(mask[v >> 5] >> (v & 31) & 1u)) z = -INFINITY;
        take(best, z, v);
        if (out) out[v] = z;
      }
    }
    // ---- the pass over the slice: a warp takes 32 neighbouring tokens
    constexpr int U = 8;
    for (int g0 = s0 + 32 * warp; g0 < s1; g0 += 32 * nw * U) {
      float l[U];
      uint32_t ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = g0 + 32 * nw * u + lane;
        l[u] = v < s1 ? load_logit<F32>(row, v) : 0.f;
        ok[u] = (mask && v < s1) ? __ldg(mask + (v >> 5)) : 0xFFFFFFFFu;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = g0 + 32 * nw * u + lane;
        if (v >= s1) break;
        if (be > bb && (biased[(v - s0) >> 5] >> (v & 31) & 1u)) continue;  // s0 is a multiple of 32
        float z = l[u];
        if (penal) z = penalise(z, cnt[v - s0], pen);
        if (!(ok[u] >> (v & 31) & 1u)) z = -INFINITY;
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
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float z = __shfl_xor_sync(0xffffffffu, best.z, o);
    const int v = __shfl_xor_sync(0xffffffffu, best.v, o);
    take(best, z, v);
  }
  if (lane == 0) wbest[warp] = best;
  __syncthreads();
  cluster_wait();
  if (tid == 0) {
    for (int w = 1; w < nw; ++w) take(best, wbest[w].z, wbest[w].v);
    const uint32_t at = map_rank(smem_u32(&cbest[crank]), 0);
    st_cluster_u32(at, __float_as_uint(best.z));
    st_cluster_u32(at + 4, static_cast<uint32_t>(best.v));
  }
  cluster_arrive();
  cluster_wait();
  if (crank == 0 && tid == 0) {
    for (uint32_t c = 1; c < csize; ++c) take(best, cbest[c].z, cbest[c].v);
    p.token[m] = best.v == INT_MAX ? -1 : best.v;
  }
}

template <bool F32>
static int logits_launch_t(const LogitParams& p, int csize, int threads, int smem, cudaStream_t s, bool pdl) {
  auto kern = aipu_logits_kernel<F32>;
  static bool attr[64] = {false};
  const int rc = set_smem_attr_once(reinterpret_cast<const void*>(kern), kMaxSlice * 4 + kMaxSlice / 8, attr,
                                    "cudaFuncSetAttribute(logits)");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.M * csize);
  cfg.blockDim = dim3(threads);
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
  const int csize = 8;
  // few rows: as many threads as an SM takes, so that a row's loads are in flight at once
  const int threads = p.M * csize <= num_sms ? 1024 : 512;
  p.slice = std::min(kMaxSlice, ((p.V + csize - 1) / csize + 31) / 32 * 32);
  const int smem = (p.spans ? p.slice * 4 : 0) + (p.bias_begin ? p.slice / 8 : 0);
  return p.f32 ? logits_launch_t<true>(p, csize, threads, smem, s, pdl) : logits_launch_t<false>(p, csize, threads, smem, s, pdl);
}

}  // namespace aipu
