// The 16/32-bit copy of an 8-bit cache that a prefill reads.
//
// A prompt's attention is tensor-bound: every cache byte meets up to 64 n_rep query rows per work
// item, so the bytes are turned into the query type once (1 byte read, 2 written, 2 read again
// through L2: 20 of the 188 us of 16 prompts with 18k cached and new tokens), and the tcgen05
// kernel (prefill_sm100.cuh) then runs as it is, fed by TMA. Converting inside it would need
// converter warps, for which its register budget (96 a thread at 18 warps) has no room.
//
// byte * scale is exact in bf16 for the append's power-of-two scales; in f16 it is exact above
// f16's subnormals, and saturates (pack2_sat). Rows behind the last token are written as zeros:
// NaN bytes that an earlier owner left there would survive a probability of 0.
#pragma once

#include "kv8_common.cuh"

namespace fa {

struct Kv8ExpandParams {
  const uint8_t *cache[2];       // [num_blocks, num_kv_heads, block_size, head_dim]
  const float *scale[2];
  void *out[2];                  // [total_blocks, num_kv_heads, block_size, head_dim]
  const int32_t *context_lens;
  const int32_t *block_tables;
  int32_t *out_ctx;              // [num_seqs]: the context length, or 0 for a refused sequence
  int32_t *out_tables;           // [num_seqs, out_width]: blocks of `out`
  const void *q;                 // q_out given: q_elems 16-bit values, then zeros up to q_out_elems
  void *q_out;
  int64_t q_elems, q_out_elems;
  int32_t max_blocks_per_seq;
  int32_t out_width;
  int32_t num_seqs;
  int32_t total_blocks;
  int32_t num_kv_heads;
  int32_t num_blocks;
  int32_t block_size;
  int32_t head_dim;
  int32_t max_context_len;
};

constexpr int kExpandThreads = 256;
constexpr int kExpandMaxSeqs = 2048;  // sequences per call (page prefix sums in shared memory)

// CTA x takes blocks x, x + gridDim.x, ... of the copy; which sequence's page a block is follows
// from prefix sums of the page counts, which every CTA computes for itself (a few KB from L2).
// Sequences are packed in order; one whose pages do not fit total_blocks is refused as a whole.
template <typename T, class F>
__global__ void __launch_bounds__(kExpandThreads) kv8_expand_kernel(const Kv8ExpandParams p) {
  static_assert(sizeof(T) == 2, "a copy in the type of the tensor-core prefill");
  __shared__ int32_t offs[kExpandMaxSeqs + 1];
  __shared__ int32_t warp_sum[kExpandThreads / 32];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.q_out) {
    for (int64_t i = int64_t(blockIdx.x) * kExpandThreads + tid; i < p.q_out_elems;
         i += int64_t(gridDim.x) * kExpandThreads)
      static_cast<uint16_t *>(p.q_out)[i] = i < p.q_elems ? static_cast<const uint16_t *>(p.q)[i] : uint16_t(0);
  }
  // Exclusive prefix sums, 256 sequences a turn. Counts saturate past total_blocks, so that sums
  // of many long (refused) sequences stay within 32 bits.
  int carry = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += kExpandThreads) {
    const int s = s0 + tid;
    int n = 0;
    if (s < p.num_seqs) {
      const int L = p.context_lens[s];
      const bool ok = L >= 0 && L <= p.max_context_len &&
                      int64_t(L) <= int64_t(p.max_blocks_per_seq) * p.block_size;
      n = ok ? (L + p.block_size - 1) / p.block_size : 0;
      n = min(n, p.total_blocks + 1);
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = min(incl + v, p.total_blocks + 1);
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < warp; ++w) base = min(base + warp_sum[w], p.total_blocks + 1);
    if (s < p.num_seqs) offs[s + 1] = min(base + incl, p.total_blocks + 1);
    for (int w = warp; w < kExpandThreads / 32; ++w) base = min(base + warp_sum[w], p.total_blocks + 1);
    carry = base;
    __syncthreads();
  }
  if (tid == 0) offs[0] = 0;
  __syncthreads();
  for (int s = blockIdx.x * kExpandThreads + tid; s < p.num_seqs; s += gridDim.x * kExpandThreads) {
    const int L = p.context_lens[s];
    const bool fits = offs[s + 1] <= p.total_blocks && L >= 0 && L <= p.max_context_len &&
                      int64_t(L) <= int64_t(p.max_blocks_per_seq) * p.block_size;
    if (!fits) report(FA_DEVERR_CONTEXT);
    p.out_ctx[s] = fits ? L : 0;
  }
  const int used = min(offs[p.num_seqs], p.total_blocks);
  const int D = p.head_dim, page = p.block_size * D;
  bool bad = false;
  for (int w = blockIdx.x; w < used; w += gridDim.x) {
    int lo = 0, hi = p.num_seqs;  // last s with offs[s] <= w
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offs[mid] <= w) lo = mid; else hi = mid;
    }
    if (offs[lo + 1] > p.total_blocks) continue;  // refused
    const int j = w - offs[lo];
    int id = p.block_tables[size_t(lo) * p.max_blocks_per_seq + j];
    if (uint32_t(id) >= uint32_t(p.num_blocks)) { bad = true; id = 0; }
    if (tid == 0) p.out_tables[size_t(lo) * p.out_width + j] = w;
    const int live = min(p.block_size, p.context_lens[lo] - j * p.block_size) * D;  // elements of a page
    for (int u = warp; u < 2 * p.num_kv_heads; u += kExpandThreads / 32) {
      const int kv = u & 1, h = u >> 1;
      const size_t src = size_t(id) * p.num_kv_heads + h, dst = size_t(w) * p.num_kv_heads + h;
      const float sc = p.scale[kv][src];
      const uint8_t *in = p.cache[kv] + src * page;
      T *out = static_cast<T *>(p.out[kv]) + dst * page;
      for (int i = lane * 8; i < page; i += 256) {  // 8 bytes in, 8 elements out; a row is a multiple of 8
        uint2 r = make_uint2(0u, 0u);
        if (i < live) r = *reinterpret_cast<const uint2 *>(in + i);
        float2 f[4];
        uint32_t a, b;
        unpack4<F>(r.x, a, b);
        f[0] = f16x2_to_f2(a);
        f[1] = f16x2_to_f2(b);
        unpack4<F>(r.y, a, b);
        f[2] = f16x2_to_f2(a);
        f[3] = f16x2_to_f2(b);
        if (i >= live) f[0] = f[1] = f[2] = f[3] = make_float2(0.f, 0.f);
        uint4 v;
        v.x = pack2_sat<T>(f[0].x * sc, f[0].y * sc);
        v.y = pack2_sat<T>(f[1].x * sc, f[1].y * sc);
        v.z = pack2_sat<T>(f[2].x * sc, f[2].y * sc);
        v.w = pack2_sat<T>(f[3].x * sc, f[3].y * sc);
        *reinterpret_cast<uint4 *>(out + i) = v;
      }
    }
  }
  if (bad && lane == 0) report(FA_DEVERR_BLOCK_ID);
}

}  // namespace fa
