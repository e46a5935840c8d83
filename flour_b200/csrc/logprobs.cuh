// Log probabilities of given tokens, entropy and top alternatives of logits rows.
//
// With m = max x and Z = sum e^(x - m) over a row's logits x:
//   log p(t) = x_t - m - ln Z,   H = -sum p ln p = ln Z - (1/Z) sum e^(x - m) (x - m),
// and the k tokens of highest logit, ties to the lower index. A logit of -inf is a token that a
// mask took out: it has probability 0, adds nothing, and is not listed.
//
// One pass over the row. A row is one cluster of 1 to 8 CTAs (more for few rows), each takes a
// contiguous part, and rank 0 joins the parts over distributed shared memory: no workspace, no
// atomics, one launch, and one order of every sum.
//
// A thread holds a tile of 32 logits in registers (16-byte loads, all in flight together), then
// takes the tile's maximum, rescales its running Z and W = sum e^(x - m)(x - m) only where the
// maximum grew, and adds the tile.
//
// Top k. Each warp keeps the best 32 it has seen as sorted 64-bit keys (ordered float bits, then
// the complement of the index), one to a lane. From the first tile's 32 lane maxima it takes the
// k-th largest: at least k logits are no smaller, so it bounds the k-th largest from below, and
// only about 1.5 k of the tile's 1024 logits pass. Passing logits are gathered 32 at a time, sorted
// and merged across the lanes; the list's k-th key is the bound of the next tile.
#pragma once

#include <cooperative_groups.h>

#include "fa_common.cuh"

namespace fa {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpTile = 32;       // logits per thread and tile
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxCluster = 8;

struct LogprobParams {
  const void *logits;        // row r at r * row_stride elements
  int64_t row_stride;
  const int32_t *token_ids;  // [rows] or nullptr; -1: no token
  float *logprobs;           // [rows], given with token_ids
  float *entropy;            // [rows] or nullptr
  int32_t *top_ids;          // [rows, top_k]
  float *top_logprobs;       // [rows, top_k]
  int32_t vocab;
  int32_t top_k;
};

__device__ __forceinline__ uint64_t lp_key(float x, int idx) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 ties with 0
  const uint32_t o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return (uint64_t(o) << 32) | (0xffffffffu - uint32_t(idx));
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = uint32_t(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  return __shfl_xor_sync(0xffffffffu, v, m);
}

// Bitonic sort of one key per lane, largest first.
__device__ __forceinline__ uint64_t warp_sort(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint64_t w = shfl_xor64(v, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);  // this lane keeps the larger
      v = (v > w) == larger ? v : w;
    }
  }
  return v;
}

// The 32 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x & 31;
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  uint64_t v = a > r ? a : r;  // bitonic
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const uint64_t w = shfl_xor64(v, j);
    v = (v > w) == ((lane & j) == 0) ? v : w;
  }
  return v;
}

// Largest 32 floats of a warp (one a lane) in order; used for the first bound alone.
__device__ __forceinline__ float warp_sort_f(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, v, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);
      v = larger ? fmaxf(v, w) : fminf(v, w);
    }
  }
  return v;
}

// (m, Z, W) of two parts of a row. m = -inf marks a part without a finite logit.
struct LpState {
  float m, z, w;
};
__device__ __forceinline__ void lp_shift(LpState &a, float m) {
  // e^(x - m') = e^(x - m) e^(m - m'): Z' = c Z, W' = c (W + (m - m') Z).
  const float d = a.m - m;
  const float c = ex2(d * kLog2e);
  if (a.m != neg_inf()) {
    const float w = c * fmaf(d, a.z, a.w);
    a.z *= c;
    a.w = c > 0.f ? w : a.z;  // c = 0: nothing is left of the part, and d Z may have overflowed
  }
  a.m = m;
}
__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  const float m = fmaxf(a.m, b.m);
  if (m == neg_inf()) return LpState{m, a.z + b.z, a.w + b.w};
  lp_shift(a, m);
  lp_shift(b, m);
  return LpState{m, a.z + b.z, a.w + b.w};
}

struct LpPart {
  LpState s;
  uint64_t top[kLpMaxTop];
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 3) token_logprobs_kernel(const LogprobParams p) {
  namespace cg = cooperative_groups;
  constexpr int VE = 16 / sizeof(T);      // logits per 16-byte vector
  constexpr int NV = kLpTile / VE;        // vectors per thread and tile
  __shared__ LpState s_state[kLpWarps];
  __shared__ uint64_t s_top[kLpWarps][32];
  __shared__ uint64_t s_new[kLpWarps][64];  // gathered candidates of a warp
  __shared__ LpPart s_part;
  __shared__ LpPart s_parts[kLpMaxCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / ranks;
  const int V = p.vocab, K = p.top_k;
  if (tid == 0) pdl_trigger();
  pdl_wait();

  // The row as 16-byte vectors from the aligned address at or below its start: vector v holds
  // logits v * VE - off .. + VE, the first and last may hold others' too and are read by element.
  const T *x = static_cast<const T *>(p.logits) + row * p.row_stride;
  const int off = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint4 *xv = reinterpret_cast<const uint4 *>(x - off);
  const int64_t nv = (int64_t(V) + off + VE - 1) / VE;
  const int64_t per = (nv + ranks - 1) / ranks;
  const int64_t v0 = rank * per, v1 = min(nv, v0 + per);

  LpState st{neg_inf(), 0.f, 0.f};
  uint64_t list = 0;           // this lane's entry of the warp's best 32
  uint64_t bound = 0;          // only larger keys may enter the best k
  float fbound = neg_inf();    // its value
  int n_new = 0;               // gathered candidates (warp-uniform)
  uint64_t *const cand = s_new[warp];

  auto flush = [&](int n) {  // merge the first n (<= 32) gathered candidates
    __syncwarp();
    const uint64_t c = warp_sort(lane < n ? cand[lane] : 0);
    list = warp_merge(list, c);
    bound = max(bound, __shfl_sync(0xffffffffu, list, K - 1));
    fbound = bound ? lp_value(bound) : neg_inf();
    __syncwarp();
  };

  bool first = true;
  for (int64_t vt = v0; vt < v1; vt += int64_t(kLpThreads) * NV) {
    // ---- load a tile: vector vt + i * 256 + tid -----------------------------------------------
    uint4 raw[NV];
    float f[kLpTile];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t v = vt + i * kLpThreads + tid;
      const int64_t e0 = v * VE - off;
      if (v < v1 && e0 >= 0 && e0 + VE <= V) {
        raw[i] = __ldcs(xv + v);
      } else {
        // Outside the part, or an edge vector of the row: element by element, -inf elsewhere.
        T e[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j)
          e[j] = (v < v1 && e0 + j >= 0 && e0 + j < V) ? x[e0 + j] : Elem<T>::from_f(neg_inf());
        raw[i] = *reinterpret_cast<const uint4 *>(e);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          f[i * VE + j] = __uint_as_float(w[j]);
        } else {
          const float2 t2 = unpack2<T>(w[j]);
          f[i * VE + 2 * j] = t2.x;
          f[i * VE + 2 * j + 1] = t2.y;
        }
      }
    }
    // ---- softmax sums ---------------------------------------------------------------------------
    float tm = f[0];
#pragma unroll
    for (int j = 1; j < kLpTile; ++j) tm = fmaxf(tm, f[j]);
    if (tm > st.m) lp_shift(st, tm);
    const float m = st.m == neg_inf() ? 0.f : st.m;
#pragma unroll
    for (int j = 0; j < kLpTile; ++j) {
      const float d = f[j] - m;
      const float e = ex2(d * kLog2e);
      st.z += e;
      st.w = fmaf(e, fmaxf(d, -1e30f), st.w);  // e = 0 where d = -inf, and 0 * -inf is not 0
    }
    // ---- candidates -------------------------------------------------------------------------------
    if (K > 0) {
      if (first) {
        // At least K of the lane maxima, so at least K logits, are >= their K-th largest. Equal
        // ones enter too (the key just below the value at the highest index).
        const float kth = __shfl_sync(0xffffffffu, warp_sort_f(tm), K - 1);
        if (kth > neg_inf()) {
          bound = (lp_key(kth, 0) & 0xffffffff00000000ull) - 1;
          fbound = kth;
        }
        first = false;
      }
      if (__any_sync(0xffffffffu, tm >= fbound && tm > neg_inf())) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float vm = f[i * VE];
#pragma unroll
          for (int j = 1; j < VE; ++j) vm = fmaxf(vm, f[i * VE + j]);
          if (!__any_sync(0xffffffffu, vm >= fbound && vm > neg_inf())) continue;
          const int e0 = int((vt + i * kLpThreads + tid) * VE - off);
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float v = f[i * VE + j];
            const uint64_t key = lp_key(v, e0 + j);
            const bool in = v > neg_inf() && key > bound;
            const uint32_t mask = __ballot_sync(0xffffffffu, in);
            if (mask) {
              if (in) cand[n_new + __popc(mask & ((1u << lane) - 1u))] = key;
              n_new += __popc(mask);
              if (n_new >= 32) {
                flush(32);
                n_new -= 32;
                if (lane < n_new) cand[lane] = cand[lane + 32];
                __syncwarp();
              }
            }
          }
        }
      }
    }
  }
  if (K > 0 && n_new > 0) flush(n_new);

  // ---- join the warps, then the cluster ------------------------------------------------------------
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpState b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.z, o),
                    __shfl_xor_sync(0xffffffffu, st.w, o)};
    // Both partners must compute the same sum: the lower lane's part first.
    st = (lane & o) ? lp_join(b, st) : lp_join(st, b);
  }
  if (lane == 0) s_state[warp] = st;
  s_top[warp][lane] = list;
  __syncthreads();
  if (K > 0) {
#pragma unroll
    for (int n = kLpWarps / 2; n > 0; n >>= 1) {
      if (warp < n) s_top[warp][lane] = warp_merge(s_top[warp][lane], s_top[warp + n][lane]);
      __syncthreads();
    }
  }
  if (warp == 0) {
    s_part.top[lane] = s_top[0][lane];
    if (lane == 0) {
      LpState a = s_state[0];
      for (int w = 1; w < kLpWarps; ++w) a = lp_join(a, s_state[w]);
      s_part.s = a;
    }
  }
  __syncthreads();
  if (ranks > 1) {
    cluster.sync();  // every rank's part is written
    if (rank == 0) {
      for (int r = warp; r < ranks; r += kLpWarps) {
        const LpPart *q = cluster.map_shared_rank(&s_part, r);
        s_parts[r].top[lane] = q->top[lane];
        if (lane == 0) s_parts[r].s = q->s;
      }
      __syncthreads();
      if (warp == 0) {
        uint64_t best = s_parts[0].top[lane];
        LpState a = s_parts[0].s;
        for (int r = 1; r < ranks; ++r) {
          if (K > 0) best = warp_merge(best, s_parts[r].top[lane]);
          a = lp_join(a, s_parts[r].s);
        }
        s_part.top[lane] = best;
        if (lane == 0) s_part.s = a;
      }
    }
    cluster.sync();  // no rank leaves while its shared memory is being read
  }
  if (rank != 0 || warp != 0) return;
  __syncwarp();
  const LpState a = s_part.s;
  // A NaN or +inf logit makes Z NaN and with it everything said of the row. A row without a
  // finite logit says that nothing can come: -inf for any token, no alternatives, entropy 0.
  const bool none = a.m == neg_inf() && a.z == 0.f;
  const float ln_z = none ? 0.f : logf(a.z);
  const float nan = __int_as_float(0x7fc00000);
  const bool bad = !(a.z == a.z) || a.m == -neg_inf();
  if (lane == 0) {
    if (p.token_ids) {
      const int32_t t = p.token_ids[row];
      float lp = 0.f;
      if (t < -1 || t >= V) {
        report(FA_DEVERR_TOKEN);
        lp = nan;
      } else if (t >= 0) {
        lp = bad ? nan : none ? neg_inf() : (Elem<T>::to_f(x[t]) - a.m) - ln_z;
      }
      p.logprobs[row] = lp;
    }
    if (p.entropy) p.entropy[row] = bad ? nan : none ? 0.f : fmaxf(ln_z - a.w / a.z, 0.f);
  }
  if (lane < K) {
    const uint64_t key = s_part.top[lane];
    const bool has = key != 0 && !bad;
    p.top_ids[row * K + lane] = has ? int32_t(0xffffffffu - uint32_t(key)) : -1;
    p.top_logprobs[row * K + lane] = bad ? nan : has ? (lp_value(key) - a.m) - ln_z : neg_inf();
  }
}

}  // namespace fa
