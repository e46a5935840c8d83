// Paged GQA decode over an 8-bit KV cache: block_size 16, head_dim 64 or 128, n_rep <= 8, 16-bit
// queries.
//
//   o = sum_j p_j vs(j) v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = scale log2(e) ks(j) q.k_j
//
// with k_j, v_j the bytes and ks(j), vs(j) the scales of position j's block and KV head.
//
// Work. A step is a pair of pages (32 tokens) of one (sequence, KV head): one maximum, one exchange
// over the lanes for both. All pairs of the batch, in order of (sequence, KV head, page), are cut
// into equal contiguous ranges, one per warp, three CTAs of four warps per SM; a warp streams its
// range through a ring of its own, across the ends of sequences, with no barrier to wait at. So
// every SM has the same bytes to read whatever the lengths, and the latencies of a start (lengths,
// block table, first bytes) are paid once a launch and not once a split: half the bytes of a
// 16-bit cache leave half the time to hide them in. Measured: 64 contexts of U[512, 4096], 8 KV
// heads of 128, 60.4 us (4.95 TB/s; 63.3 with the 16-bit decode's grid of splits and this inner
// loop); 59 of U[1, 6438], 4 KV heads, 7 query heads each, int8, 52.0 us (61.1); 16 of U[16384,
// 32768] 148 us (5.77 TB/s of the 6.56 that a copy reaches). Loud pages' probabilities at 2^12 (below)
// cost these nothing that shows: 61.4, 52.9 and 149.6, in turn with 61.7, 52.6 and 149.9 without.
// A (sequence, KV head) that ends inside one range is written by its warp; the others leave pieces
// (O / l, log2-sum-exp) in the workspace, which the CTA joins when its warps are done, and the last
// CTA of a (sequence, KV head) to finish (a ticket, no waiting) joins the CTAs' pieces. The ranges
// follow from the lengths alone, so results do not depend on timing.
//
// Bytes become f16 in registers, exactly (e4m3 and int8 are subsets of f16), and feed
// mma.sync m16n8k16 with f32 accumulation:
//   K: ldmatrix gives lane (g, t) bytes 4t..4t+3 of token g's 16-byte chunk. The dot product does
//      not care about the order of head_dim, so the four bytes are taken as k = 2t, 2t+1, 2t+8,
//      2t+9 of the fragment, and Q's fragments are loaded in the same order: no shuffles.
//   V: ldmatrix.trans on byte pairs gives tokens 2t, 2t+1 of dims 2g, 2g+1; one byte permutation
//      makes them the token pairs of two accumulator rows: row g is dim 2g, row g + 8 dim 2g + 1.
// q is divided by a power of two that brings each head's largest |q| into [1, 2), so that bf16
// queries fit f16 (a value 2^-24 below its head's largest is lost, as it is in an f32 sum of this
// length), and the factor returns with the score's scale. P is rounded to f16, which loses 8 times
// less than the bf16 of the 16-bit decode. The scale of K multiplies a score in f32; the larger of
// the pair's two scales of V multiplies its product in f32, and the other page's probabilities take
// the ratio (a power of two for scales of the append, and then exact). Probabilities are rounded at
// 2^12 times their size, so that neither the ratio nor a loud page (whose scale multiplies the
// rounding of its small probabilities) meets f16's subnormals above 2^-26.
#pragma once

#include "decode_sm100.cuh"
#include "kv8_common.cuh"

namespace fa {

constexpr int kKv8MaxSeqs = 384;   // sequences per launch (prefix sums and lengths in shared memory)
// A warp's range is at least this long (1 / 2 / 4 / 8 pairs: one sequence of 4000 tokens, 8 KV heads,
// 16.9 / 15.3 / 15.8 / 19.7 us; 4 of 300 tokens 11.3 / 11.3 / 14.6 / 19.0).
constexpr int kKv8MinPairs = 2;
constexpr int kKv8ItemPairs = 16;  // up to this length a CTA may take one (sequence, KV head)
// CTAs that may share an item before each joins its own pieces (one sequence of 2000 tokens, 2 KV
// heads: 15.1 us at 8, 14.0 at 2; 64 contexts of U[512, 4096] the same).
constexpr int kKv8Direct = 2;
constexpr int kKv8Pieces = 10;     // of a CTA in the workspace: 4 warps x (first, last), then its own two

struct Kv8DecodeParams {
  const void *q;                 // [num_seqs, num_heads, HD]
  void *out;
  const int32_t *cu_seqlens_q;   // given: sequence s's token is row cu[s] of total_q, if it has one
  int32_t total_q;
  const int32_t *context_lens;
  const int32_t *block_tables;
  const float *k_scale;          // [num_blocks, num_kv_heads]
  const float *v_scale;
  int32_t *tickets;              // [num_seqs * num_kv_heads], zero between launches
  float *pieces;                 // [gridDim.x][kKv8Pieces][n_rep][HD]
  float *piece_lse;              // [gridDim.x][kKv8Pieces][n_rep]
  int32_t max_blocks_per_seq;
  int32_t num_seqs;
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t n_rep;
  int32_t num_blocks;
  int32_t max_context_len;
  float scale_log2;              // scale * log2(e)
};

// What a warp needs of 32 pairs of its range, filled ahead by one lane each.
struct Kv8Window {
  int32_t row[2][32];  // of the slab viewed as [rows, HD]; second page: -1 if the context ends before
  float ks[2][32], vs[2][32];
};

template <int HD, int NSTAGE>
struct Kv8DecodeSmem {
  static constexpr int kPageBytes = kPage * HD;               // K (or V) of one page
  static constexpr int kStageBytes = 4 * kPageBytes;          // K, K, V, V of a pair
  static constexpr int kRingBytes = kDecodeWarps * NSTAGE * kStageBytes;
  static constexpr int kWinOff = kRingBytes;
  static constexpr int kOffsOff = kWinOff + kDecodeWarps * 2 * int(sizeof(Kv8Window));
  static constexpr int kCtxOff = kOffsOff + (kKv8MaxSeqs + 4) * 4;
  static constexpr int kBarOff = kCtxOff + kKv8MaxSeqs * 4;
  static constexpr int kMiscOff = kBarOff + kDecodeWarps * NSTAGE * 8;
  static constexpr int kAlloc = kMiscOff + 128 + 1024;  // slack to align the base to 1024 B
  static_assert(3 * (kAlloc + 1024) <= 228 * 1024, "three CTAs per SM");
};

// c = a b (no accumulator to clear first).
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

template <typename T, class F, int HD, int NSTAGE>
__global__ void __launch_bounds__(kDecodeThreads, 3)
    kv8_decode_kernel(const __grid_constant__ Kv8DecodeParams p, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v) {
  using S = Kv8DecodeSmem<HD, NSTAGE>;
  constexpr int CH = HD / 16;  // 16-byte chunks of a row = k16 steps of S = m16 tiles of O
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  Kv8Window *s_win = reinterpret_cast<Kv8Window *>(smem + S::kWinOff);
  int32_t *offs = reinterpret_cast<int32_t *>(smem + S::kOffsOff);  // pairs of sequences < s
  int32_t *s_ctx = reinterpret_cast<int32_t *>(smem + S::kCtxOff);
  uint64_t *s_bar = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  int32_t *s_misc = reinterpret_cast<int32_t *>(smem + S::kMiscOff);  // scan sums, piece items, flag

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_rep = p.n_rep, H = p.num_kv_heads;
  if (tid == 0) {
    pdl_trigger();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
#pragma unroll
    for (int i = 0; i < kDecodeWarps * NSTAGE; ++i) mbar_init(smem_u32(&s_bar[i]), 1);
    fence_mbar_init();
  }
  pdl_wait();

  auto has_token = [&](int s) {
    if (!p.cu_seqlens_q) return true;
    const int row = p.cu_seqlens_q[s];
    return row >= 0 && row < p.total_q && p.cu_seqlens_q[s + 1] == row + 1;
  };
  auto token_of = [&](int s) { return p.cu_seqlens_q ? p.cu_seqlens_q[s] : s; };

  // ---- prefix sums of the sequences' pairs; 128 sequences a turn ------------------------------
  int longest = 0;
  for (int s0 = 0, carry = 0; s0 < p.num_seqs; s0 += kDecodeThreads) {
    const int s = s0 + tid;
    int n = 0;
    if (s < p.num_seqs) {
      const int ctx = p.context_lens[s];
      const bool ok = ctx >= 1 && ctx <= p.max_context_len &&
                      int64_t(ctx) <= int64_t(p.max_blocks_per_seq) * kPage && has_token(s);
      n = ok ? (ctx + 2 * kPage - 1) / (2 * kPage) : 0;
      s_ctx[s] = ctx;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    n = __reduce_max_sync(0xffffffffu, n);
    if (lane == 31) {
      s_misc[warp] = incl;
      s_misc[8 + warp] = n;
    }
    __syncthreads();
    int base = carry, sum = carry;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      if (w < warp) base += s_misc[w];
      sum += s_misc[w];
      longest = max(longest, s_misc[8 + w]);
    }
    if (s < p.num_seqs) offs[s + 1] = base + incl;
    carry = sum;
    __syncthreads();
  }
  if (tid == 0) offs[0] = 0;
  __syncthreads();
  auto pairs_of = [&](int s) { return offs[s + 1] - offs[s]; };
  for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x) {
    if (pairs_of(s) > 0) continue;
    if (!has_token(s)) {  // no row of its own: fine when it has no token, an error otherwise
      if (tid == 0 && p.cu_seqlens_q[s + 1] != p.cu_seqlens_q[s]) report(FA_DEVERR_SEQLEN);
      continue;
    }
    // Nothing valid to attend to: one CTA zeroes the sequence's heads and reports.
    if (tid == 0) report(FA_DEVERR_CONTEXT);
    uint2 *o = reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + size_t(token_of(s)) * p.num_heads * HD);
    for (int x = tid; x < p.num_heads * (HD / 4); x += kDecodeThreads) o[x] = make_uint2(0u, 0u);
  }
  // Short contexts of few (sequence, KV head) items: a CTA takes one item each, a warp a quarter of
  // its pairs, and joins it without a ticket (16 contexts of 300, 8 KV heads: 9.5 us, 13.4 in
  // ranges). The items are then laid out at a stride of four quarters of the longest, which is all
  // that differs: pair f of the batch is pair f % stride of item f / stride.
  const int workers = int(gridDim.x) * kDecodeWarps;
  const bool by_item = p.num_seqs * H <= int(gridDim.x) && longest <= kKv8ItemPairs;
  const int stride = (longest + kDecodeWarps - 1) / kDecodeWarps * kDecodeWarps;
  const int total = by_item ? p.num_seqs * H * stride : offs[p.num_seqs] * H;
  const int ppw = by_item ? stride / kDecodeWarps  // pairs per warp
                          : max(kKv8MinPairs, (total + workers - 1) / workers);
  const int c0 = int(blockIdx.x) * (kDecodeWarps * ppw);
  if (c0 >= total) return;
  const int c1 = min(total, c0 + kDecodeWarps * ppw);
  const int w0 = min(total, c0 + warp * ppw);
  const int end = by_item ? c0 + pairs_of(int(blockIdx.x) / H) : total;  // of this CTA's pairs
  const int n_my = max(0, min(end, w0 + ppw) - w0);

  // Pair f of the flattened batch: its sequence, KV head, number in the (sequence, KV head) item.
  struct Pair {
    int s, kvh, j, of;
  };
  auto find = [&](int f) {
    if (by_item) {
      const int item = f / stride;
      return Pair{item / H, item % H, f % stride, pairs_of(item / H)};
    }
    int lo = 0, hi = p.num_seqs;  // last s with H * offs[s] <= f (of those with pairs)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offs[mid] * H <= f) lo = mid; else hi = mid;
    }
    const int np = pairs_of(lo), rem = f - offs[lo] * H;
    return Pair{lo, rem / np, rem % np, np};
  };

  // ---- this warp's stream -----------------------------------------------------------------------
  const uint32_t ring = smem_u32(smem) + warp * NSTAGE * S::kStageBytes;
  const uint32_t bar0 = smem_u32(&s_bar[warp * NSTAGE]);
  const uint64_t policy = policy_evict_first();
  Kv8Window *win = s_win + warp * 2;

  // Rows of window w go to shared memory at once; scales follow (fill_scales), behind the first loads.
  int fill_at0 = 0, fill_at1 = 0;
  auto fill_rows = [&](int w) {
    const int i = 32 * w + lane;
    if (i < n_my) {
      const Pair pr = find(w0 + i);
      const int32_t *table = p.block_tables + size_t(pr.s) * p.max_blocks_per_seq + 2 * pr.j;
      const bool two = (2 * pr.j + 1) * kPage < s_ctx[pr.s];
      int id0 = table[0], id1 = two ? table[1] : 0;
      if (uint32_t(id0) >= uint32_t(p.num_blocks) || uint32_t(id1) >= uint32_t(p.num_blocks)) {
        report(FA_DEVERR_BLOCK_ID);  // such a block is read as block 0
        if (uint32_t(id0) >= uint32_t(p.num_blocks)) id0 = 0;
        if (uint32_t(id1) >= uint32_t(p.num_blocks)) id1 = 0;
      }
      fill_at0 = id0 * H + pr.kvh;
      fill_at1 = two ? id1 * H + pr.kvh : fill_at0;
      win[w & 1].row[0][lane] = fill_at0 * kPage;
      win[w & 1].row[1][lane] = two ? fill_at1 * kPage : -1;
    }
    __syncwarp();
  };
  auto fill_scales = [&](int w) {
    if (32 * w + lane < n_my) {
      win[w & 1].ks[0][lane] = p.k_scale[fill_at0];
      win[w & 1].ks[1][lane] = p.k_scale[fill_at1];
      win[w & 1].vs[0][lane] = p.v_scale[fill_at0];
      win[w & 1].vs[1][lane] = p.v_scale[fill_at1];
    }
    __syncwarp();
  };
  auto issue = [&](int i) {
    const Kv8Window &w = win[(i >> 5) & 1];
    const int st = i % NSTAGE, r0 = w.row[0][i & 31], r1 = w.row[1][i & 31];
    const uint32_t dst = ring + st * S::kStageBytes, bar = bar0 + st * 8;
    mbar_arrive_expect_tx(bar, (r1 >= 0 ? 4 : 2) * S::kPageBytes);
    tma_load_2d_hint(dst, &tm_k, bar, 0, r0, policy);
    if (r1 >= 0) tma_load_2d_hint(dst + S::kPageBytes, &tm_k, bar, 0, r1, policy);
    tma_load_2d_hint(dst + 2 * S::kPageBytes, &tm_v, bar, 0, r0, policy);
    if (r1 >= 0) tma_load_2d_hint(dst + 3 * S::kPageBytes, &tm_v, bar, 0, r1, policy);
  };
  if (n_my > 0) {
    fill_rows(0);
    if (lane == 0)
      for (int i = 0; i < NSTAGE && i < n_my; ++i) issue(i);
    fill_scales(0);
  }

  // This lane's ldmatrix row (token) and its swizzled chunk: 128-byte rows xor the chunk with
  // row & 7, 64-byte rows with (row >> 1) & 3.
  const int l_tok = lane & 15, l_hi = lane >> 4;
  const int l_xor = HD == 128 ? (l_tok & 7) : ((l_tok >> 1) & 3);
  auto at = [&](int c) { return uint32_t(l_tok * HD + (((c + l_hi) ^ l_xor) << 4)); };

  int pieces[2] = {-1, -1};  // items of this warp's first and last piece
  bool dead = false;         // a wait gave up: nothing more is loaded or computed
  Pair pr = n_my > 0 ? find(w0) : Pair{};
  for (int i = 0; i < n_my;) {
    // ---- a segment: this warp's part of one (sequence, KV head) ------------------------------
    const int seg = min(pr.of - pr.j, n_my - i);
    const int ctx = s_ctx[pr.s];
    const int hq0 = pr.kvh * n_rep;

    // Q^T fragments (n = head g): k = 2t, 2t+1 <-> dims 4t, 4t+1 of the chunk, k + 8 <-> dims + 2.
    uint32_t qb[CH][2];
    float f0, f1;  // score factors of heads 2t, 2t+1
    {
      const T *qrow = static_cast<const T *>(p.q) + (size_t(token_of(pr.s)) * p.num_heads + hq0 + g) * HD;
      uint2 raw[CH];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        raw[c] = g < n_rep ? *reinterpret_cast<const uint2 *>(qrow + c * 16 + 4 * t) : make_uint2(0u, 0u);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float2 a = unpack2<T>(raw[c].x), b = unpack2<T>(raw[c].y);
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^floor(log2 amax), kept where its reciprocal is a normal number too.
      const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 3u), 251u);
      const float up = __uint_as_float(ex << 23), down = __uint_as_float((254u - ex) << 23);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float2 a = unpack2<T>(raw[c].x), b = unpack2<T>(raw[c].y);
        qb[c][0] = pack2<__half>(a.x * down, a.y * down);
        qb[c][1] = pack2<__half>(b.x * down, b.y * down);
      }
      // Lane 4 h holds head h's factor.
      f0 = __shfl_sync(0xffffffffu, up, 8 * t) * p.scale_log2;
      f1 = __shfl_sync(0xffffffffu, up, 8 * t + 4) * p.scale_log2;
    }
    Pair next{};
    if (i + seg < n_my) {  // the next segment's queries, on their way while this one is worked on
      next = find(w0 + i + seg);
      const char *at = reinterpret_cast<const char *>(
          static_cast<const T *>(p.q) + (size_t(token_of(next.s)) * p.num_heads + next.kvh * n_rep) * HD);
      if (lane * 128 < n_rep * HD * 2) asm volatile("prefetch.global.L1 [%0];" ::"l"(at + lane * 128));
    }
    float m0 = neg_inf(), m1 = neg_inf(), l0 = 0.f, l1 = 0.f;  // heads 2t, 2t+1
    float o[CH][4];
#pragma unroll
    for (int c = 0; c < CH; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;

    // Two accumulators, so that a page's products are two chains of CH / 2.
    auto scores = [&](uint32_t kb, float (&c)[4]) {
      float d[4];
#pragma unroll
      for (int ch = 0; ch < CH; ch += 2) {
        uint32_t r[4], a[4];
        ldsm_x4(kb + at(ch), r);
        unpack4<F>(r[0], a[0], a[2]);
        unpack4<F>(r[1], a[1], a[3]);
        if (ch == 0) mma_f16_zero(c, a, qb[ch][0], qb[ch][1]);
        else mma16816<__half>(c, a, qb[ch][0], qb[ch][1]);
        unpack4<F>(r[2], a[0], a[2]);
        unpack4<F>(r[3], a[1], a[3]);
        if (ch == 0) mma_f16_zero(d, a, qb[ch + 1][0], qb[ch + 1][1]);
        else mma16816<__half>(d, a, qb[ch + 1][0], qb[ch + 1][1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += d[e];
    };
    // Scaled scores of a page whose first token is tok0; tokens past the context are -inf.
    auto finish = [&](float (&c)[4], float ks, int tok0) {
      const float a0 = f0 * ks, a1 = f1 * ks;
      const bool v0 = tok0 + g < ctx, v1 = tok0 + g + 8 < ctx;
      c[0] = v0 ? c[0] * a0 : neg_inf();
      c[1] = v0 ? c[1] * a1 : neg_inf();
      c[2] = v1 ? c[2] * a0 : neg_inf();
      c[3] = v1 ? c[3] * a1 : neg_inf();
    };

    for (const int end = i + seg; i < end; ++i) {
      if ((i & 31) == 0 && i + 32 < n_my) {  // the next window, while this one is worked on
        fill_rows((i >> 5) + 1);
        fill_scales((i >> 5) + 1);
      }
      const int st = i % NSTAGE;
      // Warp-uniform outcome: every lane polls (bounded), and the warp goes on together.
      if (!dead && !__all_sync(0xffffffffu, mbar_wait(bar0 + st * 8, (i / NSTAGE) & 1))) {
        if (lane == 0) report(FA_DEVERR_TIMEOUT);
        for (int j = i + 1; j < n_my && j < i + NSTAGE; ++j)  // drain the loads in flight
          mbar_wait(bar0 + (j % NSTAGE) * 8, (j / NSTAGE) & 1);
        dead = true;
      }
      if (dead) continue;
      const Kv8Window &w = win[(i >> 5) & 1];
      const int e32 = i & 31;
      const int tok0 = (pr.j + seg - (end - i)) * (2 * kPage);
      const uint32_t kb = ring + st * S::kStageBytes, vb = kb + 2 * S::kPageBytes;
      if (ctx - tok0 < 2 * kPage) {
        // The context ends in this pair. What lies behind its last token (another owner's bytes, or
        // a page that was not loaded) may be e4m3's NaN, which a probability of 0 would not mask:
        // clear those rows of V, and order the stores before the ring's next load into them.
        for (int x = (ctx - tok0) * (HD / 16) + lane; x < 2 * kPage * (HD / 16); x += 32)
          *reinterpret_cast<uint4 *>(smem + (vb - smem_u32(smem)) + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }

      float ca[4], cb[4];
      scores(kb, ca);
      scores(kb + S::kPageBytes, cb);
      finish(ca, w.ks[0][e32], tok0);
      finish(cb, w.ks[1][e32], tok0 + kPage);
      float bm0 = fmaxf(fmaxf(ca[0], ca[2]), fmaxf(cb[0], cb[2]));
      float bm1 = fmaxf(fmaxf(ca[1], ca[3]), fmaxf(cb[1], cb[3]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        bm0 = fmaxf(bm0, __shfl_xor_sync(0xffffffffu, bm0, x));
        bm1 = fmaxf(bm1, __shfl_xor_sync(0xffffffffu, bm1, x));
      }
      if (__any_sync(0xffffffffu, bm0 > m0 || bm1 > m1)) {  // few steps raise a maximum late in a context
        const float mn0 = fmaxf(m0, bm0), mn1 = fmaxf(m1, bm1);
        const float r0 = ex2(m0 - mn0), r1 = ex2(m1 - mn1);
        l0 *= r0;
        l1 *= r1;
        m0 = mn0;
        m1 = mn1;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          o[c][0] *= r0;
          o[c][1] *= r1;
          o[c][2] *= r0;
          o[c][3] *= r1;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ca[e] = ex2(ca[e] - (e & 1 ? m1 : m0));
        cb[e] = ex2(cb[e] - (e & 1 ? m1 : m0));
      }
      l0 += (ca[0] + ca[2]) + (cb[0] + cb[2]);
      l1 += (ca[1] + ca[3]) + (cb[1] + cb[3]);
      const float vs0 = w.vs[0][e32], vs1 = w.vs[1][e32];
      const float vs = fmaxf(vs0, vs1);
      const bool apart = fminf(vs0, vs1) < vs * 0.015625f || vs < 1.e-34f;
      const float inv = vs > 0.f ? 4096.f / vs : 0.f;  // both scales 0: nothing to add
      const float ra = apart ? 4096.f : vs0 * inv, rb = apart ? 4096.f : vs1 * inv;
      const uint32_t pa0 = movmatrix_t(pack2<__half>(ca[0] * ra, ca[1] * ra));
      const uint32_t pa1 = movmatrix_t(pack2<__half>(ca[2] * ra, ca[3] * ra));
      const uint32_t pb0 = movmatrix_t(pack2<__half>(cb[0] * rb, cb[1] * rb));
      const uint32_t pb1 = movmatrix_t(pack2<__half>(cb[2] * rb, cb[3] * rb));
      // o += (P_a V_a + P_b V_b) down factor
      auto values = [&](uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, float down, float factor) {
#pragma unroll
        for (int ch = 0; ch < CH; ch += 2) {
          float ta[2][4];
          uint32_t ra4[4], rb4[4], a[4];
          ldsm_x4_t(vb + at(ch), ra4);
          ldsm_x4_t(vb + S::kPageBytes + at(ch), rb4);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            unpack4_t<F>(ra4[2 * e], a[0], a[1]);
            unpack4_t<F>(ra4[2 * e + 1], a[2], a[3]);
            mma_f16_zero(ta[e], a, a0, a1);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            unpack4_t<F>(rb4[2 * e], a[0], a[1]);
            unpack4_t<F>(rb4[2 * e + 1], a[2], a[3]);
            mma16816<__half>(ta[e], a, b0, b1);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int q = 0; q < 4; ++q) o[ch + e][q] = fmaf(ta[e][q] * down, factor, o[ch + e][q]);
        }
      };
      if (!apart) {
        values(pa0, pa1, pb0, pb1, 1.f, vs * (1.f / 4096.f));
      } else {  // more than a factor 64 between the pages, or tiny scales: one after the other
#pragma unroll 1
        for (int x = 0; x < 2; ++x)
          values(x ? 0u : pa0, x ? 0u : pa1, x ? pb0 : 0u, x ? pb1 : 0u, 1.f / 4096.f, x ? vs1 : vs0);
      }
      __syncwarp();
      if (lane == 0 && i + NSTAGE < n_my) issue(i + NSTAGE);
    }

    // ---- the segment's end: the output, or a piece ---------------------------------------------
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    const float i0 = 1.f / l0, i1 = 1.f / l1;
    if (seg == pr.of) {
      T *out = static_cast<T *>(p.out) + (size_t(token_of(pr.s)) * p.num_heads + hq0) * HD + 2 * g;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (2 * t < n_rep)
          *reinterpret_cast<uint32_t *>(out + (2 * t) * HD + c * 16) = pack2_sat<T>(o[c][0] * i0, o[c][2] * i0);
        if (2 * t + 1 < n_rep)
          *reinterpret_cast<uint32_t *>(out + (2 * t + 1) * HD + c * 16) = pack2_sat<T>(o[c][1] * i1, o[c][3] * i1);
      }
    } else {
      const int which = i == seg ? 0 : 1;  // the range's first segment, or its last
      pieces[which] = pr.s * H + pr.kvh;
      const size_t slot = size_t(blockIdx.x) * kKv8Pieces + warp * 2 + which;
      float *po = p.pieces + slot * n_rep * HD + 2 * g;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (2 * t < n_rep)
          *reinterpret_cast<float2 *>(po + (2 * t) * HD + c * 16) = make_float2(o[c][0] * i0, o[c][2] * i0);
        if (2 * t + 1 < n_rep)
          *reinterpret_cast<float2 *>(po + (2 * t + 1) * HD + c * 16) = make_float2(o[c][1] * i1, o[c][3] * i1);
      }
      if (g == 0) {
        float *pl = p.piece_lse + slot * n_rep;
        if (2 * t < n_rep) pl[2 * t] = m0 + __log2f(l0);
        if (2 * t + 1 < n_rep) pl[2 * t + 1] = m1 + __log2f(l1);
      }
    }
    pr = next;
  }
  if (lane == 0) {
    s_misc[2 * warp] = pieces[0];
    s_misc[2 * warp + 1] = pieces[1];
  }
  __syncthreads();  // the warps' pieces are written, and every ring is drained

  // ---- join the pieces ------------------------------------------------------------------------
  // The pieces of an item are those of the workers (warps) that its pairs fall to, the first
  // segment of a worker's range in its slot 0, a later one in slot 1. An item inside this CTA is
  // joined here; one that others have a part of by the last CTA to take its ticket. Where more than
  // kKv8Direct CTAs share an item, each joins its own pieces first.
  const int cpp = kDecodeWarps * ppw;  // pairs per CTA
  // Piece k of n at row(k) of the pieces -> dst (f32, with its lse), or the output. Four values of
  // head_dim a thread; eight pieces and their sums in flight, folded into a running maximum.
  auto join = [&](int item, int n, auto row, float *dst, float *dst_lse) {
    for (int x = tid; x < n_rep * (HD / 4); x += kDecodeThreads) {
      const int h = x / (HD / 4), d = x % (HD / 4) * 4;
      float M = neg_inf(), W = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k0 = 0; k0 < n; k0 += 8) {
        float4 v[8];
        float e[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          e[u] = neg_inf();
          v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k0 + u < n) {
            const size_t r = row(k0 + u) * n_rep + h;
            e[u] = __ldcg(p.piece_lse + r);
            v[u] = __ldcg(reinterpret_cast<const float4 *>(p.pieces + r * HD + d));
          }
        }
        float m = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) m = fmaxf(m, e[u]);
        const float c = ex2(M - m);
        O = make_float4(O.x * c, O.y * c, O.z * c, O.w * c);
        W *= c;
        M = m;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float w = ex2(e[u] - m);
          O.x += w * v[u].x;
          O.y += w * v[u].y;
          O.z += w * v[u].z;
          O.w += w * v[u].w;
          W += w;
        }
      }
      const float i = 1.f / W;
      if (dst) {
        *reinterpret_cast<float4 *>(dst + h * HD + d) = make_float4(O.x * i, O.y * i, O.z * i, O.w * i);
        if (d == 0) dst_lse[h] = M + __log2f(W);
      } else {
        T *out = static_cast<T *>(p.out) +
                 (size_t(token_of(item / H)) * p.num_heads + (item % H) * n_rep + h) * HD + d;
        *reinterpret_cast<uint2 *>(out) = make_uint2(pack2_sat<T>(O.x * i, O.y * i), pack2_sat<T>(O.z * i, O.w * i));
      }
    }
  };
  struct Span {
    int a0, a1;  // the item's pairs
  };
  auto span = [&](int item) {
    const int s = item / H, np = pairs_of(s), a0 = by_item ? item * stride : offs[s] * H + (item % H) * np;
    return Span{a0, a0 + np};
  };
  // Workers first .. first + n - 1 of item; the row of a worker's piece.
  auto pieces_of = [&](const Span &sp, int from, int to, int &first) {
    first = max(sp.a0, from) / ppw;
    return (min(sp.a1, to) - 1) / ppw - first + 1;
  };
  auto row_of = [&](const Span &sp, int worker) {
    return size_t(worker / kDecodeWarps) * kKv8Pieces + worker % kDecodeWarps * 2 +
           (worker * ppw < sp.a0 ? 1 : 0);
  };
  auto own_row = [&](const Span &sp, int c) {
    return size_t(c) * kKv8Pieces + 2 * kDecodeWarps + (sp.a0 < c * cpp ? 0 : 1);
  };
  // The (at most two) items that other CTAs share: the first with a piece here, and the last.
  int shared[2] = {-1, -1};
  for (int k = 0, seen = -1; k < 2 * kDecodeWarps; ++k) {
    const int item = s_misc[k];
    if (item < 0 || item == seen) continue;  // an item's pieces follow one another
    seen = item;
    const Span sp = span(item);
    int first;
    const int n = pieces_of(sp, c0, c1, first);
    if (sp.a0 >= c0 && sp.a1 <= c1) {
      join(item, n, [&](int q) { return row_of(sp, first + q); }, nullptr, nullptr);
      continue;
    }
    if ((sp.a1 - 1) / cpp - sp.a0 / cpp >= kKv8Direct) {
      const size_t own = own_row(sp, blockIdx.x);
      join(item, n, [&](int q) { return row_of(sp, first + q); }, p.pieces + own * n_rep * HD,
           p.piece_lse + own * n_rep);
    }
    shared[sp.a0 < c0 ? 0 : 1] = item;
  }
  if (shared[0] < 0 && shared[1] < 0) return;
  // The barrier orders the CTA's pieces before the release of its tickets.
  __syncthreads();
  if (tid < 2) {
    const int item = shared[tid];
    int last = 0;
    if (item >= 0) {
      const Span sp = span(item);
      __threadfence();
      last = atomicAdd(&p.tickets[item], 1) == (sp.a1 - 1) / cpp - sp.a0 / cpp;
      __threadfence();
    }
    s_misc[16 + tid] = last;
  }
  __syncthreads();
  if (!s_misc[16] && !s_misc[17]) return;
#pragma unroll 1
  for (int x = 0; x < 2; ++x) {
    if (!s_misc[16 + x]) continue;
    const int item = shared[x];
    const Span sp = span(item);
    const int ctas = (sp.a1 - 1) / cpp - sp.a0 / cpp + 1;
    int first;
    if (ctas > kKv8Direct) {
      join(item, ctas, [&](int q) { return own_row(sp, sp.a0 / cpp + q); }, nullptr, nullptr);
    } else {
      const int n = pieces_of(sp, 0, total, first);
      join(item, n, [&](int q) { return row_of(sp, first + q); }, nullptr, nullptr);
    }
    if (tid == 0) p.tickets[item] = 0;  // ready for the next launch
  }
}

}  // namespace fa
