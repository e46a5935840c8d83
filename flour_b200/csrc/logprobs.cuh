// Log probabilities of given tokens, entropy and top alternatives of logits rows.
//
// With m near max x (the streaming form lets it lag by up to 8) and Z = sum e^(x - m) over a row's
// logits x:
//   log p(t) = x_t - m - ln Z,   H = -sum p ln p = ln Z - (1/Z) sum e^(x - m) (x - m),
// and the k tokens of highest logit, ties to the lower index. A logit of -inf is a token that a
// mask took out: it has probability 0, adds nothing, and is not listed.
//
// A row is read once, by one cluster of up to 16 CTAs; rank 0 joins the parts that the others
// write into its shared memory. No workspace, no atomics between CTAs, one launch, and one order of
// every sum. Two kernels:
//   part    each CTA's part of the row fits its registers (32 logits a thread): few rows, where
//           latency counts;
//   stream  each CTA walks its part in tiles, the next one's loads in flight: many rows.
//
// Top k without sorting the row. Among n groups that cover the logits, at least k maxima, hence at
// least k logits, are >= the k-th largest group maximum: a lower bound of the k-th largest logit.
// With 32 groups (lanes of a warp, or half warps of a CTA) one bitonic sort over the lanes of a
// warp gives it, and of the random logits about 32 ln(32 / (32 - k)) pass, 31 for k = 20. What
// passes is gathered and sorted as 64-bit keys: the float's bits in order, then the complement of
// the index.
#pragma once

#include <cooperative_groups.h>

#include "fa_common.cuh"

namespace fa {

constexpr int kLpMaxTop = 32;
constexpr int kLpMaxCluster = 16;    // 16 CTAs a cluster is opt-in; 8 without
constexpr int kLpPartLogits = 32;    // a thread's logits in the part kernel
constexpr int kLpPartThreads = 512;
constexpr int kLpSmallThreads = 128; // vocabularies that fit one CTA of this size

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

// Bitonic sort of one key per lane, largest first.
__device__ __forceinline__ uint64_t warp_sort(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint64_t w = __shfl_xor_sync(0xffffffffu, v, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);  // this lane keeps the larger
      v = (v > w) == larger ? v : w;
    }
  }
  return v;
}
__device__ __forceinline__ float warp_sort(float v) {
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

// The 32 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x & 31;
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  uint64_t v = a > r ? a : r;  // bitonic
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, j);
    v = (v > w) == ((lane & j) == 0) ? v : w;
  }
  return v;
}

// A part of a row: m a reference near its largest logit, z = sum e^(x - m), w = sum e^(x - m) (x - m).
// A part without a finite logit has m = -inf, z = 0. A NaN logit makes z NaN, for good.
struct LpState {
  float m, z, w;
};

// e^(x - m') = e^(x - m) e^(m - m'):  z' = c z,  w' = c (w + (m - m') z).
__device__ __forceinline__ void lp_shift(LpState &a, float m) {
  const float d = a.m - m;
  const float c = ex2(d * kLog2e);
  if (a.m != neg_inf()) {
    const float w = c * fmaf(d, a.z, a.w);
    a.z *= c;
    a.w = c > 0.f ? w : a.z;  // c = 0: nothing is left of the part, and d z may have overflowed
  }
  a.m = m;
}
__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  const float m = fmaxf(a.m, b.m);
  if (m != neg_inf()) {
    lp_shift(a, m);
    lp_shift(b, m);
  }
  return LpState{m, a.z + b.z, a.w + b.w};
}
// Join over the lanes of a warp; both partners of a step add the lower lane's part first, so that
// every lane ends with the same bits.
__device__ __forceinline__ LpState lp_warp_join(LpState st) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpState b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.z, o),
                    __shfl_xor_sync(0xffffffffu, st.w, o)};
    st = (lane & o) ? lp_join(b, st) : lp_join(st, b);
  }
  return st;
}

// Two floats of one instruction.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Logits e, e + 1 of the vectors `raw` (e even and constant once unrolled).
template <typename T, int NV>
__device__ __forceinline__ float2 lp_pair(const uint4 (&raw)[NV], int e) {
  constexpr int VE = 16 / sizeof(T);
  const uint4 &v = raw[e / VE];
  const int i = e % VE;
  if constexpr (sizeof(T) == 4)
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  else
    return unpack2<T>(i == 0 ? v.x : i == 2 ? v.y : i == 4 ? v.z : v.w);
}

// Sums of e^(x - m) and e^(x - m) (x - m) over N logits in vectors, against a reference m that no
// logit passes by much. Four operations a logit: with L = log2(e), M = m L rounded and r = m L - M
// (one fma, so exact), s = x L - M is one fma, e^(x - m) = 2^(s - r) and x - m = (s - r) / L; r
// leaves the sums. All but the exponential are done for two logits an instruction (2048 x 151643
// bf16 -4.9 us). The second sum is NaN for a NaN, no reference (m = -inf), logits whose product with
// log2(e) overflows, and without kMasked for masked logits (0 * -inf). It is made NaN where |r| > 1
// (|m| from 2^25 / log2(e) on): s near r is then rounded in steps that show in e^(x - m), and from
// |r| = 126 on 2^s is 0.
template <typename T, bool kMasked, int NV>
__device__ __forceinline__ float2 lp_sums_fast(const uint4 (&raw)[NV], float m) {
  constexpr int N = NV * 16 / sizeof(T);
  const float M = m * kLog2e, r = fmaf(m, kLog2e, -M);
  const uint64_t L2 = f32x2(kLog2e, kLog2e), M2 = f32x2(-M, -M);
  uint64_t z2 = 0, w2 = 0;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 x = lp_pair<T>(raw, j);
    uint64_t s2 = f32x2_fma(f32x2(x.x, x.y), L2, M2);
    const float2 s = f32x2_parts(s2);
    const uint64_t e2 = f32x2(ex2(s.x), ex2(s.y));
    if (kMasked) s2 = f32x2(fmaxf(s.x, -1e30f), fmaxf(s.y, -1e30f));
    z2 = f32x2_add(z2, e2);
    w2 = f32x2_fma(e2, s2, w2);
  }
  const float2 zz = f32x2_parts(z2), ww = f32x2_parts(w2);
  const float back = fabsf(r) <= 1.f ? ex2(-r) : __int_as_float(0x7fc00000), z = zz.x + zz.y;
  return make_float2(z * back, fmaf(-r, z, ww.x + ww.y) * (back * 0.693147180559945f));
}

// The same of one vector with care, where lp_sums_fast fails.
template <typename T> __device__ __forceinline__ float2 lp_sums_slow(uint4 v, float m) {
  const uint4 raw[1] = {v};
  float z = 0.f, w = 0.f;
#pragma unroll
  for (int j = 0; j < 16 / int(sizeof(T)); j += 2) {
    const float2 x = lp_pair<T>(raw, j);
    if (m == neg_inf()) {
      if (x.x != x.x || x.y != x.y) z = x.x + x.y;
    } else {
      const float d0 = x.x - m, d1 = x.y - m;
      const float e0 = ex2(d0 * kLog2e), e1 = ex2(d1 * kLog2e);
      z += e0 + e1;
      w = fmaf(e0, fmaxf(d0, -1e30f), w);
      w = fmaf(e1, fmaxf(d1, -1e30f), w);
    }
  }
  return make_float2(z, w);
}

// One vector that may hold masked logits.
template <typename T> __device__ __noinline__ float2 lp_sums_vec(uint4 v, float m) {
  const uint4 raw[1] = {v};
  const float2 f = lp_sums_fast<T, true>(raw, m);
  return f.y == f.y ? f : lp_sums_slow<T>(v, m);
}

// Logits e0 .. e0 + 15 bytes of x[0 .. end), -inf outside. Out of line: few vectors take it.
template <typename T> __device__ __noinline__ uint4 lp_edge(const T *x, int e0, int end) {
  constexpr int VE = 16 / sizeof(T);
  alignas(16) T e[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) e[j] = (e0 + j >= 0 && e0 + j < end) ? x[e0 + j] : Elem<T>::from_f(neg_inf());
  return *reinterpret_cast<const uint4 *>(e);
}

// A row as 16-byte vectors from the aligned address at or below its start: vector v holds logits
// v * VE - off and on.
template <typename T> struct LpRow {
  static constexpr int VE = 16 / sizeof(T);
  const T *x;
  const uint4 *xv;
  int off, vocab, nv;
  __device__ __forceinline__ LpRow(const LogprobParams &p, int64_t row) {
    x = static_cast<const T *>(p.logits) + row * p.row_stride;
    off = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    xv = reinterpret_cast<const uint4 *>(x - off);
    vocab = p.vocab;
    nv = (vocab + off + VE - 1) / VE;
  }
  // Vector v of a part that ends at v1; -inf past it. The row's first and last vectors may hold
  // its neighbours' logits too and are read element by element.
  __device__ __forceinline__ uint4 load(int v, int v1) const {
    const int e0 = v * VE - off;
    if (v < v1 && e0 >= 0 && e0 + VE <= vocab) return __ldcs(xv + v);
    return lp_edge<T>(x, e0, v < v1 ? vocab : 0);
  }
  // Vectors v, v + step, ... v + (NV - 1) step of this thread, where first .. last bound those of
  // all threads: one check for a tile inside the row.
  template <int NV>
  __device__ __forceinline__ void load_tile(uint4 (&raw)[NV], int first, int v, int step, int v1) const {
    if (first >= (off ? 1 : 0) && first + step * NV <= min(v1, (vocab + off) / VE)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i] = __ldcs(xv + v + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i] = load(v + i * step, v1);
    }
  }
  __device__ __forceinline__ int index(int v) const { return v * VE - off; }
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The largest logit of each vector, and of all; NaN if one is. 16-bit ones are compared two at a
// time.
template <typename T, int NV>
__device__ __forceinline__ float lp_maxima(const uint4 (&raw)[NV], float (&vm)[NV]) {
  float tm = neg_inf();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (sizeof(T) == 2) {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 *w = reinterpret_cast<const T2 *>(&raw[i]);
      const T2 m2 = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
      const float2 m = unpack2<T>(*reinterpret_cast<const uint32_t *>(&m2));
      vm[i] = max_nan(m.x, m.y);
    } else {
      const float2 a = lp_pair<T>(raw, i * 4), b = lp_pair<T>(raw, i * 4 + 2);
      vm[i] = max_nan(max_nan(a.x, a.y), max_nan(b.x, b.y));
    }
    tm = max_nan(tm, vm[i]);
  }
  return tm;
}

// This lane's logits that are >= bound, one at a time. Short loops over selected registers: updates
// unrolled over the tile miss the instruction cache, and few tiles take them.
template <typename T, int NV> struct LpHits {
  static constexpr int VE = 16 / sizeof(T);
  uint32_t vecs = 0, bits = 0;  // vectors not yet looked at, hits in the current one
  uint4 one[1];
  int vec = 0;
  __device__ __forceinline__ LpHits(const float (&vm)[NV], float bound) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (vm[i] >= bound) vecs |= 1u << i;
  }
  // The next hit: its value and number e (logit e % VE of vector e / VE); false when there is none.
  __device__ __forceinline__ bool next(const uint4 (&raw)[NV], float bound, float &x, int &e) {
    if (bits == 0) {
      if (vecs == 0) return false;
      vec = __ffs(vecs) - 1;
      vecs &= vecs - 1;
      one[0] = raw[0];
#pragma unroll
      for (int i = 1; i < NV; ++i)
        if (vec == i) one[0] = raw[i];
#pragma unroll
      for (int j = 0; j < VE; j += 2) {
        const float2 p = lp_pair<T>(one, j);
        if (p.x >= bound) bits |= 1u << j;
        if (p.y >= bound) bits |= 2u << j;
      }
    }
    const int j = __ffs(bits) - 1;  // a vector's maximum is a hit
    bits &= bits - 1;
    e = vec * VE + j;
    const int b = j * int(sizeof(T));
    const uint32_t w = b < 8 ? (b < 4 ? one[0].x : one[0].y) : (b < 12 ? one[0].z : one[0].w);
    if constexpr (sizeof(T) == 4) x = __uint_as_float(w);
    else x = (b & 2) ? unpack2<T>(w).y : unpack2<T>(w).x;
    return true;
  }
};

// The warp's list `mine` with its n <= 32 gathered candidates. Out of line: one copy of the sort.
__device__ __noinline__ uint64_t lp_take(uint64_t mine, const uint64_t *cand, int n) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  mine = warp_merge(mine, warp_sort(lane < n ? cand[lane] : 0));
  __syncwarp();
  return mine;
}

// A warp's best 32 logits so far, one key to a lane in order, and the candidates gathered since.
struct LpList {
  uint64_t mine = 0;                // this lane's key
  uint64_t bound = 0;               // only larger keys can be among the best k
  float fbound = -3.402823466e38f;  // its value; no -inf passes
  int n = 0;                        // gathered (warp-uniform)
  bool listed = false;              // the bound is a key of the list
  uint64_t *cand;                   // shared, 64 of this warp

  __device__ __forceinline__ void at_least(float v) {  // k logits are >= v
    if (v > fbound) {
      bound = (lp_key(v, 0) & 0xffffffff00000000ull) - 1;
      fbound = v;
    }
  }
  __device__ __forceinline__ void flush(int count, int k) {
    mine = lp_take(mine, cand, count);
    const uint64_t kth = __shfl_sync(0xffffffffu, mine, k - 1);
    if (kth > bound) {
      bound = kth;
      fbound = lp_value(kth);
      listed = true;
    }
  }
  // Gathers the logits of a tile that are >= pass. Logit e is e % VE of vector v0 + e / VE * step.
  template <typename T, int NV>
  __device__ __forceinline__ void gather(const uint4 (&raw)[NV], const float (&vm)[NV], float pass,
                                         const LpRow<T> &r, int v0, int step, int k) {
    const int lane = threadIdx.x & 31;
    LpHits<T, NV> hits(vm, pass);
    while (true) {
      float x;
      int e;
      uint64_t key = 0;
      const bool has = hits.next(raw, pass, x, e);
      if (has) key = lp_key(x, r.index(v0 + e / LpRow<T>::VE * step) + e % LpRow<T>::VE);
      if (!__any_sync(0xffffffffu, has)) break;
      const uint32_t mask = __ballot_sync(0xffffffffu, key > bound);
      if (key > bound) cand[n + __popc(mask & ((1u << lane) - 1u))] = key;
      n += __popc(mask);
      if (n >= 32) {
        flush(32, k);
        n -= 32;
        if (lane < n) cand[lane] = cand[lane + 32];
        __syncwarp();
      }
    }
  }
};

// The CTA's candidates: keys of the logits that passed the bound when their tile was read. One
// that comes when the pool is full is counted only, and the row's part is read again with lists.
constexpr int kLpPool = 2048;
struct LpPool {
  uint64_t key[kLpPool];
  int n;
};

template <typename T, int NV>
__device__ __forceinline__ void lp_pool_add(LpPool &pool, const uint4 (&raw)[NV], const float (&vm)[NV],
                                            float bound, const LpRow<T> &r, int v0, int step) {
  LpHits<T, NV> hits(vm, bound);
  float x;
  int e;
#pragma unroll 1
  while (hits.next(raw, bound, x, e)) {
    const int at = atomicAdd(&pool.n, 1);
    if (at < kLpPool)
      pool.key[at] = lp_key(x, r.index(v0 + e / LpRow<T>::VE * step) + e % LpRow<T>::VE);
  }
}

// The best 32 of n keys, one key to a lane of warp 0. Each warp sorts every WARPS-th run of 32.
template <int WARPS>
__device__ __forceinline__ uint64_t lp_pool_top(const uint64_t *keys, int n, uint64_t (&s_top)[WARPS][32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t top = 0;
  for (int i = 32 * warp; i < n; i += 32 * WARPS) {
    const uint64_t c = warp_sort(i + lane < n ? keys[i + lane] : 0);
    top = i == 32 * warp ? c : warp_merge(top, c);
  }
  const int lists = min(WARPS, (n + 31) / 32);
  if (lists <= 1) return top;
  s_top[warp][lane] = top;
  for (int h = WARPS / 2; h > 0; h >>= 1) {
    __syncthreads();
    if (warp < h && warp + h < lists) {
      top = warp_merge(top, s_top[warp + h][lane]);
      s_top[warp][lane] = top;
    }
  }
  return top;
}

// The next float above x (finite).
__device__ __forceinline__ float lp_above(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return __uint_as_float(b >> 31 ? b - 1 : b + 1);
}

struct LpPart {
  LpState s;
  uint64_t top[kLpMaxTop];
};

// Shared by both kernels once a CTA's part is known to its warp 0 (st in every lane, top one key a
// lane): ranks > 0 write theirs to rank 0 and leave; rank 0 joins all and writes the row's results.
template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobParams &p, const T *x, int64_t row, LpState st,
                                          uint64_t top, LpPart *s_parts) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int K = p.top_k;
  if (ranks > 1) {
    // The first barrier phase (arrived at on entry) says that rank 0 runs, so its memory may be
    // written; the second that every part is there.
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
      LpPart *q = cluster.map_shared_rank(s_parts, 0) + rank;
      q->top[lane] = top;
      if (lane == 0) q->s = st;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
    if (K > 0) {
      for (int n = kLpMaxCluster / 2; n > 0; n >>= 1) {
        for (int i = warp; i < n; i += warps)
          if (i + n < ranks)
            s_parts[i].top[lane] = warp_merge(s_parts[i].top[lane], s_parts[i + n].top[lane]);
        __syncthreads();
      }
    }
    if (warp != 0) return;
    top = s_parts[0].top[lane];
    st = lp_warp_join(lane < ranks ? s_parts[lane].s : LpState{neg_inf(), 0.f, 0.f});
  }
  if (warp != 0) return;
  // A NaN or +inf logit makes z NaN and with it everything said of the row. A row without a
  // finite logit says that nothing can come: -inf for any token, no alternatives, entropy 0. No
  // rounding makes a probability larger than 1.
  const bool bad = st.z != st.z || st.m == -neg_inf();
  const bool none = st.m == neg_inf();
  const float ln_z = none ? 0.f : logf(st.z);
  const float nan = __int_as_float(0x7fc00000);
  if (lane == 0) {
    if (p.token_ids) {
      const int32_t t = p.token_ids[row];
      float lp = 0.f;
      if (t < -1 || t >= p.vocab) {
        report(FA_DEVERR_TOKEN);
        lp = nan;
      } else if (t >= 0) {
        lp = bad ? nan : none ? neg_inf() : fminf((Elem<T>::to_f(x[t]) - st.m) - ln_z, 0.f);
      }
      p.logprobs[row] = lp;
    }
    if (p.entropy) p.entropy[row] = bad ? nan : none ? 0.f : fmaxf(ln_z - st.w / st.z, 0.f);
  }
  if (lane < K) {
    const bool has = top != 0 && !bad;
    p.top_ids[row * K + lane] = has ? int32_t(0xffffffffu - uint32_t(top)) : -1;
    p.top_logprobs[row * K + lane] = bad ? nan : has ? fminf((lp_value(top) - st.m) - ln_z, 0.f) : neg_inf();
  }
}

__device__ __forceinline__ void lp_cluster_arrive() {
  if (cooperative_groups::this_cluster().num_blocks() > 1)
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}

// ---- part kernel --------------------------------------------------------------------------------
// Every thread keeps its logits (vector i * THREADS + tid of the CTA's part) in registers.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_part_kernel(const LogprobParams p) {
  using Row = LpRow<T>;
  constexpr int VE = Row::VE, NV = kLpPartLogits / VE, WARPS = THREADS / 32;
  constexpr int PER_GROUP = THREADS / 32;  // threads of one of the 32 groups
  __shared__ float s_max[32];
  __shared__ float2 s_sum[WARPS];
  __shared__ LpPool s_pool;
  __shared__ uint64_t s_top[WARPS][32];
  __shared__ LpPart s_parts[kLpMaxCluster];
  const int ranks = int(cooperative_groups::this_cluster().num_blocks());
  const int rank = int(cooperative_groups::this_cluster().block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.top_k;
  lp_cluster_arrive();
  if (tid == 0) {
    pdl_trigger();
    s_pool.n = 0;
  }
  pdl_wait();
  const int64_t row = blockIdx.x / ranks;
  const Row r(p, row);
  const int per = (r.nv + ranks - 1) / ranks, v0 = rank * per, v1 = min(r.nv, v0 + per);
  uint4 raw[NV];
  r.load_tile(raw, v0, v0 + tid, THREADS, v1);
  float vm[NV];
  const float tm = lp_maxima<T>(raw, vm);
  float m = tm;
#pragma unroll
  for (int o = 1; o < PER_GROUP; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane % PER_GROUP == 0) s_max[tid / PER_GROUP] = m;
  __syncthreads();

  // Each warp by itself: the part's maximum and the bound of its k-th largest.
  m = s_max[lane];
  if (K > 0) {
    const float sorted = warp_sort(m);
    m = __shfl_sync(0xffffffffu, sorted, 0);
    const float bound = fmaxf(__shfl_sync(0xffffffffu, sorted, K - 1), -3.402823466e38f);
    lp_pool_add(s_pool, raw, vm, bound, r, v0 + tid, THREADS);
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  float z = 0.f, w = 0.f;
  const float2 f = lp_sums_fast<T, false>(raw, m);
  if (f.y == f.y) {
    z = f.x;
    w = f.y;
  } else {  // in place: every row's last threads come here (-0.5 us against a call)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 v = lp_sums_slow<T>(raw[i], m);
      z += v.x;
      w += v.y;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  if (lane == 0) s_sum[warp] = make_float2(z, w);
  __syncthreads();

  const int n = s_pool.n;
  uint64_t top = 0;
  if (n > kLpPool) {  // many equal logits: the warps' own lists, which drop ties past the k-th
    static_assert(WARPS * 64 <= kLpPool, "the lists' candidates reuse the pool");
    LpList list;
    list.cand = s_pool.key + warp * 64;
    list.at_least(__shfl_sync(0xffffffffu, warp_sort(tm), K - 1));
    list.gather(raw, vm, list.fbound, r, v0 + tid, THREADS, K);
    if (list.n > 0) list.flush(list.n, K);
    s_top[warp][lane] = list.mine;
    __syncthreads();
    if (warp == 0)
      for (int i = 0; i < WARPS; ++i) top = warp_merge(top, s_top[i][lane]);
  } else {
    top = lp_pool_top<WARPS>(s_pool.key, n, s_top);
  }
  LpState st{m, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    st.z += s_sum[i].x;
    st.w += s_sum[i].y;
  }
  lp_finish<T>(p, r.x, row, st, top, s_parts);
}

// A part once more, with a list a warp (the pool was too small). Out of line: its registers are not
// the streaming loop's.
template <typename T, int THREADS>
__device__ __noinline__ uint64_t lp_reread(const LpRow<T> r, int v0, int v1, float bound, uint64_t *cand,
                                           int K) {
  constexpr int NV = 4;
  const int tid = threadIdx.x;
  LpList list;
  list.cand = cand;
  list.at_least(bound);
  for (int vt = v0; vt < v1; vt += THREADS * NV) {
    uint4 raw[NV];
    r.load_tile(raw, vt, vt + tid, THREADS, v1);
    float vm[NV];
    lp_maxima<T>(raw, vm);
    // A key already in the list has a lower index than any of this tile: equal logits are out.
    list.gather(raw, vm, list.listed ? lp_above(list.fbound) : list.fbound, r, vt + tid, THREADS, K);
  }
  if (list.n > 0) list.flush(list.n, K);
  return list.mine;
}

// ---- stream kernel ------------------------------------------------------------------------------
// Tiles of 64 bytes a thread, the next one in flight. The 32 groups of the CTA (THREADS / 32 lanes
// each) keep their running maxima in shared memory, and the warps take a new bound from them after tiles
// 1, 2, 4, 8, ...: without a barrier but the first, for maxima that a warp sees too early are still
// a lower bound. About 32 ln(32 / (32 - k)) logits pass in each doubling. The vectors that hold them
// are kept whole, and their logits looked at once behind the loop, a thread each, against the last
// bound (2048 x 151643, 20 alternatives, f16: 133 us, 151 with the logits picked out in the loop, and
// 120 without alternatives). Where more pass than the lists hold (ascending rows, many equal logits)
// the part is read a second time, with a list a warp.
constexpr int kLpVecs = 512, kLpKeys = 512;
template <int WARPS> struct LpStreamPool {
  union {
    uint4 vec[kLpVecs];
    uint64_t cand[WARPS * 64];  // of the second reading
  };
  int at[kLpVecs];              // a vector's number in the row
  uint64_t key[kLpKeys];
  int vecs, keys;
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_stream_kernel(const LogprobParams p) {
  using Row = LpRow<T>;
  constexpr int NV = 4, WARPS = THREADS / 32, GROUP = THREADS / 32, TILE = THREADS * NV;  // 32 groups
  __shared__ LpState s_state[WARPS];
  __shared__ volatile float s_max[32];
  __shared__ LpStreamPool<WARPS> s_pool;
  __shared__ uint64_t s_top[WARPS][32];
  __shared__ LpPart s_parts[kLpMaxCluster];
  const int ranks = int(cooperative_groups::this_cluster().num_blocks());
  const int rank = int(cooperative_groups::this_cluster().block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.top_k;
  lp_cluster_arrive();
  if (tid == 0) {
    pdl_trigger();
    s_pool.vecs = s_pool.keys = 0;
  }
  pdl_wait();
  const int64_t row = blockIdx.x / ranks;
  const Row r(p, row);
  const int per = (r.nv + ranks - 1) / ranks, v0 = rank * per, v1 = min(r.nv, v0 + per);
  LpState st{neg_inf(), 0.f, 0.f};
  float largest = neg_inf(), bound = -3.402823466e38f;  // no -inf passes
  auto put_max = [&] {
    float m = largest;
#pragma unroll
    for (int o = 1; o < GROUP; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane % GROUP == 0) s_max[tid / GROUP] = m;
  };
  auto raise_bound = [&] { bound = fmaxf(bound, __shfl_sync(0xffffffffu, warp_sort(float(s_max[lane])), K - 1)); };
  uint4 next[NV];
  r.load_tile(next, v0, v0 + tid, THREADS, v1);
  int tile = 0;
  bool masked = false;  // a tile held masked logits: the others are taken to do so too
  for (int vt = v0; vt < v1; vt += TILE, ++tile) {
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = next[i];
    if (vt + TILE < v1) r.load_tile(next, vt + TILE, vt + TILE + tid, THREADS, v1);
    float vm[NV];
    const float tm = lp_maxima<T>(raw, vm);
    largest = fmaxf(largest, tm);
    // The reference moves only where e^(x - m) would leave e^8 behind: hardly ever after the first
    // tile, where some lane of a warp finds a new maximum in most tiles (-1.9 us). x - m and ln z
    // near 8 round in steps of 2^-21, and 2^s with s to 11.5 in such of 2^-20: what a near-certain
    // token's log probability may be off by, about 2^-23 with m at its logit.
    if (tm > st.m + 8.f) lp_shift(st, tm);
    if (K > 0) {
      if ((tile & (tile + 1)) == 0) {
        put_max();
        if (tile == 0) __syncthreads();
        __syncwarp();
        raise_bound();
      }
      if (tm >= bound) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (vm[i] >= bound) {
            const int at = atomicAdd(&s_pool.vecs, 1);
            if (at < kLpVecs) {
              s_pool.vec[at] = raw[i];
              s_pool.at[at] = vt + tid + i * THREADS;
            }
          }
      }
    }
    if (!(tm > neg_inf())) {  // masked logits only, or a NaN
      if (tm != tm) st.z = tm;
      continue;
    }
    // The sums; vector by vector, and by a call (the loop's code has to stay in the instruction
    // cache), in the last tile, whose vectors behind the row are left out, and where logits are masked.
    if (!masked && vt + TILE <= v1) {
      const float2 f = lp_sums_fast<T, false>(raw, st.m);
      if (f.y == f.y) {
        st.z += f.x;
        st.w += f.y;
        continue;
      }
      masked = tile > 0;  // the first may fail for what lies before the row
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (vm[i] > neg_inf()) {
        const float2 f = lp_sums_vec<T>(raw[i], st.m);
        st.z += f.x;
        st.w += f.y;
      }
  }
  if (K > 0) put_max();
  st = lp_warp_join(st);
  if (lane == 0) s_state[warp] = st;
  __syncthreads();
  uint64_t top = 0;
  if (K > 0) {
    const int n = s_pool.vecs;
    raise_bound();
    for (int i = tid; i < n && n <= kLpVecs; i += THREADS) {
      const uint4 one[1] = {s_pool.vec[i]};
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < Row::VE; j += 2) {
        const float2 x = lp_pair<T>(one, j);
        if (x.x >= bound) bits |= 1u << j;
        if (x.y >= bound) bits |= 2u << j;
      }
      const T *x = reinterpret_cast<const T *>(&s_pool.vec[i]);
      for (; bits; bits &= bits - 1) {
        const int j = __ffs(bits) - 1, at = atomicAdd(&s_pool.keys, 1);
        if (at < kLpKeys) s_pool.key[at] = lp_key(Elem<T>::to_f(x[j]), r.index(s_pool.at[i]) + j);
      }
    }
    __syncthreads();
    if (n <= kLpVecs && s_pool.keys <= kLpKeys) {
      top = lp_pool_top<WARPS>(s_pool.key, s_pool.keys, s_top);
    } else {
      s_top[warp][lane] = lp_reread<T, THREADS>(r, v0, v1, bound, s_pool.cand + warp * 64, K);
      __syncthreads();
      if (warp == 0)
        for (int i = 0; i < WARPS; ++i) top = warp_merge(top, s_top[i][lane]);
    }
  }
  st = lp_warp_join(lane < WARPS ? s_state[lane] : LpState{neg_inf(), 0.f, 0.f});
  lp_finish<T>(p, r.x, row, st, top, s_parts);
}

}  // namespace fa
