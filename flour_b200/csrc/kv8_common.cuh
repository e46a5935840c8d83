// 8-bit KV cache: element formats and the append that fills it.
//
// A cache value is byte * scale[block, kv head], K and V apart. The append writes scales that are
// powers of two, which makes every quotient x / scale exact (one rounding, to the 8-bit grid) and
// every dequantised value exact in bf16 (e4m3 has 4 significant bits, an int8 magnitude 7). A
// part-filled block of a cache quantised elsewhere may keep another scale: its quotients are formed
// in 64 bits (to_odd), so that they too are rounded once.
#pragma once

#include "fa_common.cuh"

namespace fa {

// Formats of the 8-bit pools (fa_kv8_dtype).
struct E4m3 {
  static constexpr float kMax = 448.f;
  // 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6: significand bits of the largest value and its exponent.
  static constexpr uint32_t kMaxMant = 0x600000u;
  static constexpr int kMaxExp = 8;
};
struct I8 {
  static constexpr float kMax = 127.f;
  static constexpr uint32_t kMaxMant = 0x7e0000u;
  static constexpr int kMaxExp = 6;
};

// Two e4m3 bytes as f16x2 (exact: e4m3 is a subset of f16; NaN stays NaN).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(d)
      : "r"(v));
  return d;
}

// Four cache bytes b0..b3 of one register as f16 pairs, without their scale: unpack4 gives
// (b0, b1), (b2, b3); unpack4_t gives (b0, b2), (b1, b3).
// int8: the byte plus 128 becomes the low mantissa bits of 1024.0h (f16 steps of 1 there), and
// subtracting 1152 leaves the signed value, exactly.
template <class F> __device__ __forceinline__ void unpack4(uint32_t r, uint32_t &a, uint32_t &b);
template <class F> __device__ __forceinline__ void unpack4_t(uint32_t r, uint32_t &a, uint32_t &b);
template <> __device__ __forceinline__ void unpack4<E4m3>(uint32_t r, uint32_t &a, uint32_t &b) {
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=&r"(a), "=r"(b)
      : "r"(r));
}
template <> __device__ __forceinline__ void unpack4_t<E4m3>(uint32_t r, uint32_t &a, uint32_t &b) {
  unpack4<E4m3>(__byte_perm(r, 0u, 0x3120), a, b);
}
__device__ __forceinline__ uint32_t i8_bias(uint32_t v) {
  const __half2 k = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), k);
  return *reinterpret_cast<uint32_t *>(&h);
}
template <> __device__ __forceinline__ void unpack4<I8>(uint32_t r, uint32_t &a, uint32_t &b) {
  r ^= 0x80808080u;
  a = i8_bias(__byte_perm(r, 0x64646464u, 0x4140));
  b = i8_bias(__byte_perm(r, 0x64646464u, 0x4342));
}
template <> __device__ __forceinline__ void unpack4_t<I8>(uint32_t r, uint32_t &a, uint32_t &b) {
  r ^= 0x80808080u;
  a = i8_bias(__byte_perm(r, 0x64646464u, 0x4240));
  b = i8_bias(__byte_perm(r, 0x64646464u, 0x4341));
}

__device__ __forceinline__ float2 f16x2_to_f2(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

template <class F> __device__ __forceinline__ float byte_to_f(uint8_t b);
template <> __device__ __forceinline__ float byte_to_f<E4m3>(uint8_t b) {
  return f16x2_to_f2(e4m3x2_to_f16x2(b)).x;
}
template <> __device__ __forceinline__ float byte_to_f<I8>(uint8_t b) { return float(int8_t(b)); }

// Two values already divided by their scale -> two bytes (lo = a), nearest, ties to even.
// Magnitudes past the largest value saturate; NaN is e4m3's NaN and int8's 0.
template <class F> __device__ __forceinline__ uint32_t to_bytes2(float a, float b);
template <> __device__ __forceinline__ uint32_t to_bytes2<E4m3>(float a, float b) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
  return d;
}
template <> __device__ __forceinline__ uint32_t to_bytes2<I8>(float a, float b) {
  const int x = min(max(__float2int_rn(a), -127), 127), y = min(max(__float2int_rn(b), -127), 127);
  return (uint32_t(x) & 0xffu) | ((uint32_t(y) & 0xffu) << 8);
}

// The smallest power of two s >= 2^-126 with a <= kMax * s (a finite, >= 0), from a's exponent.
template <class F> __device__ __forceinline__ float pow2_scale(float a) {
  const uint32_t bits = __float_as_uint(a);
  int e = int(bits >> 23) - 127 - F::kMaxExp;  // subnormal a: far below the floor of -126
  if ((bits & 0x7fffffu) > F::kMaxMant) ++e;
  return __uint_as_float(uint32_t(max(e, -126) + 127) << 23);
}

struct Kv8AppendParams {
  const void *x[2];              // key, value: x[t*stride_t + h*stride_h + i]
  int64_t stride_t[2], stride_h[2];
  uint8_t *cache[2];             // [num_blocks, num_kv_heads, block_size, head_dim]
  float *scale[2];               // [num_blocks, num_kv_heads]
  const int32_t *cu_seqlens_q;   // [num_seqs + 1]; nullptr: one new token per sequence
  const int32_t *context_lens;
  const int32_t *block_tables;
  int32_t max_blocks_per_seq;
  int32_t num_seqs;
  int32_t total_q;
  int32_t num_kv_heads;
  int32_t num_blocks;
  int32_t block_size;
  int32_t head_dim;
};

// The new rows of one block: rows [row0, row0 + n) of physical block `id` from tokens tok0...
struct Kv8Run {
  int32_t id, row0, n, tok0;
};

constexpr int kAppendThreads = 128;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendChunk = 16;     // tokens per CTA of the varlen form
constexpr int kAppendCuSmem = 1024;  // cu_seqlens entries searched in shared memory

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The scale of a block after an append whose new rows reach `amax`, and the factor that moves the
// rows it held before (1: they stay as they are). A block whose first row is new starts afresh:
// the scale that an earlier owner left does not count.
template <class F>
__device__ __forceinline__ float append_scale(float amax, float before, bool held, float &move) {
  const float need = pow2_scale<F>(amax);
  const float after = held ? fmaxf(before, need) : need;
  move = held ? before / after : 1.f;
  return after;
}

__device__ __forceinline__ bool is_pow2(float s) { return (__float_as_uint(s) & 0x7fffffu) == 0; }

// x in f32 with what was cut off kept in the last bit, so that rounding the result to 8 significant
// bits or fewer gives what rounding x would: no border between two codes has that bit.
__device__ __forceinline__ float to_odd(double x) {
  const float f = __double2float_rz(x);
  return double(f) == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// One warp appends one run to one head of K or V: any head_dim, block_size, alignment and scale.
template <typename T, class F>
__device__ __forceinline__ bool append_run(const Kv8AppendParams &p, const Kv8Run &r, int h, int kv) {
  const int lane = threadIdx.x & 31, D = p.head_dim;
  const T *x = static_cast<const T *>(p.x[kv]) + int64_t(r.tok0) * p.stride_t[kv] +
               int64_t(h) * p.stride_h[kv];
  uint8_t *page = p.cache[kv] + (size_t(r.id) * p.num_kv_heads + h) * p.block_size * size_t(D);
  float *sc = p.scale[kv] + size_t(r.id) * p.num_kv_heads + h;
  const float before = *sc;
  bool bad = false;
  float amax = 0.f;
  for (int i = lane; i < r.n * D; i += 32) {
    const float a = fabsf(Elem<T>::to_f(x[int64_t(i / D) * p.stride_t[kv] + i % D]));
    const bool fin = a <= 3.402823466e38f;
    bad |= !fin;
    if (fin) amax = fmaxf(amax, a);
  }
  float move;
  const float after = append_scale<F>(warp_max(amax), before, r.row0 > 0, move), inv = 1.f / after;
  const bool exact = is_pow2(after) && is_pow2(move);
  if (move != 1.f)
    for (int i = lane; i < r.row0 * D; i += 32) {
      const float b = byte_to_f<F>(page[i]);
      page[i] = uint8_t(to_bytes2<F>(exact ? b * move : to_odd(double(b) * double(move)), 0.f));
    }
  for (int i = lane; i < r.n * D; i += 32) {
    const float f = Elem<T>::to_f(x[int64_t(i / D) * p.stride_t[kv] + i % D]);
    page[size_t(r.row0) * D + i] =
        uint8_t(to_bytes2<F>(exact ? f * inv : to_odd(double(f) / double(after)), 0.f));
  }
  if (lane == 0) *sc = after;
  return bad;
}

// The same for block_size 16, head_dim D of 64 or 128 and 16-byte aligned rows: the run's rows are
// loaded at once, 8 values a lane and row (4 KB of bf16 a warp in flight at D = 128), and stay in
// registers between the maximum and the rounding. Magnitudes are compared as integers, two 16-bit
// ones an instruction; a run with an infinity or NaN (the largest patterns), and a block whose scale
// is or was not a power of two, takes append_run.
template <typename T, class F, int D>
__device__ __forceinline__ bool append_run_vec(const Kv8AppendParams &p, const Kv8Run &r, int h, int kv) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES, PASSES = 16 / ROWS, W = sizeof(T) * 2;
  const int lane = threadIdx.x & 31, row = lane / LANES, col = lane % LANES * 8;
  const T *x = static_cast<const T *>(p.x[kv]) + int64_t(r.tok0) * p.stride_t[kv] +
               int64_t(h) * p.stride_h[kv] + col;
  uint8_t *page = p.cache[kv] + (size_t(r.id) * p.num_kv_heads + h) * (16 * D) + col;
  float *sc = p.scale[kv] + size_t(r.id) * p.num_kv_heads + h;
  const float before = *sc;
  uint32_t v[PASSES][W];  // 8 values of a row
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
#pragma unroll
    for (int q = 0; q < W / 4; ++q) {
      uint4 t = make_uint4(0u, 0u, 0u, 0u);
      if (i * ROWS + row < r.n)
        t = __ldcs(reinterpret_cast<const uint4 *>(x + int64_t(i * ROWS + row) * p.stride_t[kv]) + q);
      v[i][4 * q] = t.x;
      v[i][4 * q + 1] = t.y;
      v[i][4 * q + 2] = t.z;
      v[i][4 * q + 3] = t.w;
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int q = 0; q < W; ++q) {
      if constexpr (sizeof(T) == 4) mx = max(mx, v[i][q] & 0x7fffffffu);
      else mx = __vmaxu2(mx, v[i][q] & 0x7fff7fffu);
    }
  if constexpr (sizeof(T) == 2) mx = max(mx & 0xffffu, mx >> 16);
  mx = __reduce_max_sync(0xffffffffu, mx);
  float amax;
  bool fin;
  if constexpr (sizeof(T) == 4) {
    amax = __uint_as_float(mx);
    fin = mx < 0x7f800000u;
  } else {
    amax = unpack2<T>(mx).x;
    fin = mx < (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
  }
  float move;
  const float after = append_scale<F>(amax, before, r.row0 > 0, move), inv = 1.f / after;
  if (!fin || !is_pow2(after) || !is_pow2(move)) return append_run<T, F>(p, r, h, kv);
  if (move != 1.f) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int o = i * ROWS + row;
      if (o < r.row0) {
        uint2 *at = reinterpret_cast<uint2 *>(page + o * D);
        uint2 b = *at;
        uint32_t lo, hi;
        unpack4<F>(b.x, lo, hi);
        float2 f0 = f16x2_to_f2(lo), f1 = f16x2_to_f2(hi);
        b.x = to_bytes2<F>(f0.x * move, f0.y * move) | to_bytes2<F>(f1.x * move, f1.y * move) << 16;
        unpack4<F>(b.y, lo, hi);
        f0 = f16x2_to_f2(lo);
        f1 = f16x2_to_f2(hi);
        b.y = to_bytes2<F>(f0.x * move, f0.y * move) | to_bytes2<F>(f1.x * move, f1.y * move) << 16;
        *at = b;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float2 f;
      if constexpr (sizeof(T) == 4) f = make_float2(__uint_as_float(v[i][2 * q]), __uint_as_float(v[i][2 * q + 1]));
      else f = unpack2<T>(v[i][q]);
      b[q] = to_bytes2<F>(f.x * inv, f.y * inv);
    }
    if (i * ROWS + row < r.n)
      *reinterpret_cast<uint2 *>(page + (r.row0 + i * ROWS + row) * D) =
          make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
  }
  if (lane == 0) *sc = after;
  return false;
}

// Tokens [16 c, 16 c + 16) of the packed batch: the runs that begin there, in `runs` (each token
// that is its sequence's first or its block's first begins one). Called by the first 16 threads
// of a warp with `cu` in shared or global memory.
__device__ __forceinline__ int append_runs(const Kv8AppendParams &p, const int32_t *cu, int chunk,
                                           Kv8Run *runs) {
  const int lane = threadIdx.x & 31;
  const int t = chunk * kAppendChunk + lane;
  bool begins = false;
  Kv8Run r{};
  if (lane < kAppendChunk && t < p.total_q && t < cu[p.num_seqs]) {
    int lo = 0, hi = p.num_seqs;  // last s with cu[s] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    const int q0 = cu[lo], q1 = cu[lo + 1];
    if (q0 < 0 || q0 > t || q1 <= t || q1 > p.total_q) {
      report(FA_DEVERR_SEQLEN);
    } else {
      const int n = q1 - q0, L = p.context_lens[lo];
      if (L < n || int64_t(L) > int64_t(p.max_blocks_per_seq) * p.block_size) {
        report(FA_DEVERR_CONTEXT);
      } else {
        const int pos = L - n + (t - q0);
        r.row0 = pos % p.block_size;
        if (t == q0 || r.row0 == 0) {
          r.id = p.block_tables[size_t(lo) * p.max_blocks_per_seq + pos / p.block_size];
          r.n = min(p.block_size - r.row0, q1 - t);
          r.tok0 = t;
          begins = uint32_t(r.id) < uint32_t(p.num_blocks);
          if (!begins) report(FA_DEVERR_BLOCK_ID);
        }
      }
    }
  }
  const uint32_t mask = __ballot_sync(0xffffffffu, begins);
  if (begins) runs[__popc(mask & ((1u << lane) - 1u))] = r;
  return __popc(mask);
}

// Varlen form (cu_seqlens_q given): CTA (c, y) finds the runs that begin in its 16 tokens, and
// its warps take (run, head, K | V) units. A run belongs to one warp, so the scale of a block is
// read, grown and written by one owner, and no order of the warps changes a result.
// One-token form: a unit is (sequence, head, K | V), with nothing to search.
// D: 64 or 128 for the vector form, 0 for any shape. 32 warps per SM, each with 4 KB of bf16 in flight
// (64 registers; f32 rows need twice as many): 57k tokens x 8 heads x 128 from bf16 49.0 us, 5.67
// TB/s of the 6.56 that a copy reaches; 24 warps in CTAs of 256 took 54.9.
template <typename T, class F, int D>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 4 ? 4 : 8) kv8_append_kernel(const Kv8AppendParams p) {
  auto append = [&](const Kv8Run &r, int h, int kv) {
    if constexpr (D > 0) return append_run_vec<T, F, D>(p, r, h, kv);
    else return append_run<T, F>(p, r, h, kv);
  };
  __shared__ Kv8Run runs[kAppendChunk];
  __shared__ int s_n;
  __shared__ int32_t s_cu[kAppendCuSmem];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  const int per_run = 2 * p.num_kv_heads;
  bool bad = false;
  if (p.cu_seqlens_q == nullptr) {
    const int64_t u = int64_t(blockIdx.x) * kAppendWarps + warp;
    if (u >= int64_t(p.num_seqs) * per_run) return;
    const int s = int(u / per_run), hk = int(u % per_run);
    const int L = p.context_lens[s];
    if (L < 1 || int64_t(L) > int64_t(p.max_blocks_per_seq) * p.block_size) {
      report(FA_DEVERR_CONTEXT);
      return;
    }
    const int id = p.block_tables[size_t(s) * p.max_blocks_per_seq + (L - 1) / p.block_size];
    if (uint32_t(id) >= uint32_t(p.num_blocks)) {
      report(FA_DEVERR_BLOCK_ID);
      return;
    }
    const Kv8Run r{id, (L - 1) % p.block_size, 1, s};
    bad = append(r, hk >> 1, hk & 1);
  } else {
    const int32_t *cu = p.cu_seqlens_q;
    if (p.num_seqs < kAppendCuSmem) {
      for (int i = threadIdx.x; i <= p.num_seqs; i += kAppendThreads) s_cu[i] = cu[i];
      cu = s_cu;
    }
    __syncthreads();
    if (warp == 0) {
      const int n = append_runs(p, cu, blockIdx.x, runs);
      if (threadIdx.x == 0) s_n = n;
    }
    __syncthreads();
    const int units = s_n * per_run;
    for (int u = blockIdx.y * kAppendWarps + warp; u < units; u += gridDim.y * kAppendWarps) {
      const int hk = u % per_run;
      bad |= append(runs[u / per_run], hk >> 1, hk & 1);
    }
  }
  if (bad) report(FA_DEVERR_VALUE);
}

}  // namespace fa
