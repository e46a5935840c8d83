// Paged GQA decode over an 8-bit KV cache: block_size 16, head_dim 64 or 128, n_rep <= 8, 16-bit
// queries.
//
//   o = sum_j p_j vs(j) v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = scale log2(e) ks(j) q.k_j
//
// with k_j, v_j the bytes and ks(j), vs(j) the scales of position j's block and KV head.
//
// The split into (split, kv head, sequence) CTAs, the per-warp TMA rings, the online softmax and
// the ticketed merge are those of the 16-bit decode (decode_sm100.cuh); half the bytes per token
// leave half the time per token, so a ring step is two pages (32 tokens: one max, one exchange
// over the lanes and one rescale of the accumulators for both).
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
// less than the bf16 of the 16-bit decode. The scale of K multiplies a score in f32; the scale
// of V multiplies the page's product in f32, two pages of one scale (powers of two: the usual
// case) share an accumulator.
#pragma once

#include "decode_sm100.cuh"
#include "kv8_common.cuh"

namespace fa {

struct Kv8Cache {
  const float *k_scale;  // [num_blocks, num_kv_heads]
  const float *v_scale;
};

template <int HD, int NSTAGE>
struct Kv8DecodeSmem {
  static constexpr int kPageBytes = kPage * HD;               // K (or V) of one page
  static constexpr int kStageBytes = 4 * kPageBytes;          // K, K, V, V of a step's two pages
  static constexpr int kRingBytes = kDecodeWarps * NSTAGE * kStageBytes;
  static constexpr int kIdsOff = kRingBytes;
  static constexpr int kKsOff = kIdsOff + kDecodeMaxPagesPerSplit * 4;
  static constexpr int kVsOff = kKsOff + kDecodeMaxPagesPerSplit * 4;
  static constexpr int kBarOff = kVsOff + kDecodeMaxPagesPerSplit * 4;
  static constexpr int kFlagOff = kBarOff + kDecodeWarps * NSTAGE * 8;
  static constexpr int kAlloc = kFlagOff + 16 + 1024;  // slack to align the base to 1024 B
  static constexpr int kRedStride = HD + 4;            // reduction scratch over the drained ring
  static_assert(kDecodeWarps * 8 * (kRedStride + 2) * 4 + 8 * kDecodeMaxSplits * 4 <= kRingBytes,
                "reduction scratch must fit in the ring");
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
    kv8_decode_kernel(const __grid_constant__ DecodeParams p, const Kv8Cache sc,
                      const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v) {
  using S = Kv8DecodeSmem<HD, NSTAGE>;
  constexpr int CH = HD / 16;  // 16-byte chunks of a row = k16 steps of S = m16 tiles of O
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  int32_t *s_ids = reinterpret_cast<int32_t *>(smem + S::kIdsOff);
  float *s_ks = reinterpret_cast<float *>(smem + S::kKsOff);
  float *s_vs = reinterpret_cast<float *>(smem + S::kVsOff);
  uint64_t *s_bar = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  int32_t *s_flag = reinterpret_cast<int32_t *>(smem + S::kFlagOff);

  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_rep = p.n_rep;
  if (tid == 0) pdl_trigger();
  pdl_wait();

  const int ctx = p.context_lens[b];
  if (ctx < 1 || ctx > p.max_context_len || int64_t(ctx) > int64_t(p.max_blocks_per_seq) * kPage) {
    if (split == 0) {
      if (tid == 0) report(FA_DEVERR_CONTEXT);
      for (int x = tid; x < n_rep * HD; x += kDecodeThreads)
        store_out<T>(p, b, kvh * n_rep + x / HD, HD, x % HD, 0.f);
    }
    return;
  }
  const int n_pages = (ctx + kPage - 1) / kPage;
  const int n_splits = (n_pages + p.pages_per_split - 1) / p.pages_per_split;
  if (split >= n_splits) return;
  const int pg0 = split * p.pages_per_split;
  const int npg = min(n_pages, pg0 + p.pages_per_split) - pg0;

  if (tid == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
#pragma unroll
    for (int i = 0; i < kDecodeWarps * NSTAGE; ++i) mbar_init(smem_u32(&s_bar[i]), 1);
    fence_mbar_init();
  }
  const int32_t *table = p.block_tables + size_t(b) * p.max_blocks_per_seq + pg0;
  bool bad = false;
  for (int i = tid; i < npg; i += kDecodeThreads) {
    int id = table[i];
    if (uint32_t(id) >= uint32_t(p.num_blocks)) { bad = true; id = 0; }
    s_ids[i] = id;
  }
  if (bad) report(FA_DEVERR_BLOCK_ID);
  __syncthreads();

  // ---- per-warp stream of page pairs --------------------------------------------------------
  const int n_pairs = (npg + 1) / 2;
  const int n_my = n_pairs > warp ? (n_pairs - warp + kDecodeWarps - 1) / kDecodeWarps : 0;
  const uint32_t ring = smem_u32(smem) + warp * NSTAGE * S::kStageBytes;
  const uint32_t bar0 = smem_u32(&s_bar[warp * NSTAGE]);
  const uint64_t policy = policy_evict_first();

  auto issue = [&](int i) {
    const int st = i % NSTAGE, j = 2 * (warp + i * kDecodeWarps);
    const uint32_t dst = ring + st * S::kStageBytes, bar = bar0 + st * 8;
    const int n = min(2, npg - j);
    mbar_arrive_expect_tx(bar, n * 2 * S::kPageBytes);
    for (int x = 0; x < n; ++x) {
      const int row = (s_ids[j + x] * p.num_kv_heads + kvh) * kPage;
      tma_load_2d_hint(dst + x * S::kPageBytes, &tm_k, bar, 0, row, policy);
      tma_load_2d_hint(dst + (2 + x) * S::kPageBytes, &tm_v, bar, 0, row, policy);
    }
  };
  if (lane == 0)
    for (int i = 0; i < NSTAGE && i < n_my; ++i) issue(i);
  // Scales arrive while the first pages do.
  for (int i = tid; i < npg; i += kDecodeThreads) {
    const size_t at = size_t(s_ids[i]) * p.num_kv_heads + kvh;
    s_ks[i] = sc.k_scale[at];
    s_vs[i] = sc.v_scale[at];
  }

  // Q^T fragments (n = head g): k = 2t, 2t+1 <-> dims 4t, 4t+1 of the chunk, k + 8 <-> dims + 2.
  uint32_t qb[CH][2];
  float f0, f1;  // score factors of heads 2t, 2t+1
  {
    const T *qrow = static_cast<const T *>(p.q) + (size_t(b) * p.num_heads + kvh * n_rep + g) * HD;
    float2 v[CH][2];
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint2 raw = make_uint2(0u, 0u);
      if (g < n_rep) raw = *reinterpret_cast<const uint2 *>(qrow + c * 16 + 4 * t);
      v[c][0] = unpack2<T>(raw.x);
      v[c][1] = unpack2<T>(raw.y);
#pragma unroll
      for (int e = 0; e < 2; ++e) amax = fmaxf(amax, fmaxf(fabsf(v[c][e].x), fabsf(v[c][e].y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^floor(log2 amax), kept where its reciprocal is a normal number too.
    const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 3u), 251u);
    const float up = __uint_as_float(ex << 23), down = __uint_as_float((254u - ex) << 23);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) qb[c][e] = pack2<__half>(v[c][e].x * down, v[c][e].y * down);
    // Lane 4 h holds head h's factor.
    f0 = __shfl_sync(0xffffffffu, up, 8 * t) * p.scale_log2;
    f1 = __shfl_sync(0xffffffffu, up, 8 * t + 4) * p.scale_log2;
  }
  __syncthreads();  // scales are in shared memory

  float m0 = neg_inf(), m1 = neg_inf(), l0 = 0.f, l1 = 0.f;  // heads 2t, 2t+1
  float o[CH][4];
#pragma unroll
  for (int c = 0; c < CH; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;

  // This lane's ldmatrix row (token) and its swizzled chunk: 128-byte rows xor the chunk with
  // row & 7, 64-byte rows with (row >> 1) & 3.
  const int l_tok = lane & 15, l_hi = lane >> 4;
  const int l_xor = HD == 128 ? (l_tok & 7) : ((l_tok >> 1) & 3);
  auto at = [&](int c) { return uint32_t(l_tok * HD + (((c + l_hi) ^ l_xor) << 4)); };

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

  int timed_out_at = -1;
  for (int i = 0; i < n_my; ++i) {
    const int st = i % NSTAGE;
    if (!__all_sync(0xffffffffu, mbar_wait(bar0 + st * 8, (i / NSTAGE) & 1))) {
      timed_out_at = i;
      break;
    }
    const int j = 2 * (warp + i * kDecodeWarps);
    const int tok0 = (pg0 + j) * kPage;
    const uint32_t kb = ring + st * S::kStageBytes, vb = kb + 2 * S::kPageBytes;
    const bool two = j + 1 < npg;
    if (ctx - tok0 < 2 * kPage) {
      // The context ends in this step, the warp's last. What lies behind its last token (another
      // owner's bytes, or a page that was not loaded) may be e4m3's NaN, which a probability of 0
      // would not mask: clear those rows of V.
      for (int x = (ctx - tok0) * (HD / 16) + lane; x < 2 * kPage * (HD / 16); x += 32)
        *reinterpret_cast<uint4 *>(smem + (vb - smem_u32(smem)) + x * 16) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }

    float ca[4], cb[4];
    scores(kb, ca);
    scores(kb + S::kPageBytes, cb);
    finish(ca, s_ks[j], tok0);
    finish(cb, s_ks[j + 1], tok0 + kPage);
    float bm0 = fmaxf(fmaxf(ca[0], ca[2]), fmaxf(cb[0], cb[2]));
    float bm1 = fmaxf(fmaxf(ca[1], ca[3]), fmaxf(cb[1], cb[3]));
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      bm0 = fmaxf(bm0, __shfl_xor_sync(0xffffffffu, bm0, x));
      bm1 = fmaxf(bm1, __shfl_xor_sync(0xffffffffu, bm1, x));
    }
    if (__any_sync(0xffffffffu, bm0 > m0 || bm1 > m1)) {  // few steps raise a maximum late in a context
      const float mn0 = fmaxf(m0, bm0), mn1 = fmaxf(m1, bm1);
      const float c0 = ex2(m0 - mn0), c1 = ex2(m1 - mn1);
      l0 *= c0;
      l1 *= c1;
      m0 = mn0;
      m1 = mn1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        o[c][0] *= c0;
        o[c][1] *= c1;
        o[c][2] *= c0;
        o[c][3] *= c1;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ca[e] = ex2(ca[e] - (e & 1 ? m1 : m0));
      cb[e] = ex2(cb[e] - (e & 1 ? m1 : m0));
    }
    l0 += (ca[0] + ca[2]) + (cb[0] + cb[2]);
    l1 += (ca[1] + ca[3]) + (cb[1] + cb[3]);
    // V's scales: the larger multiplies the step's product, the other page's probabilities take the
    // ratio (a power of two for scales of one append history, and then exact).
    const float vs0 = s_vs[j], vs1 = two ? s_vs[j + 1] : vs0;
    const float vs = fmaxf(vs0, vs1);
    const bool apart = fminf(vs0, vs1) < vs * 0.015625f || vs < 1.2e-38f;
    const float inv = vs > 0.f ? 1.f / vs : 0.f;  // both scales 0: nothing to add
    const float ra = apart ? 1.f : vs0 * inv, rb = apart ? 0.f : vs1 * inv;
    const uint32_t pa0 = movmatrix_t(pack2<__half>(ca[0] * ra, ca[1] * ra));
    const uint32_t pa1 = movmatrix_t(pack2<__half>(ca[2] * ra, ca[3] * ra));
    const uint32_t pb0 = movmatrix_t(pack2<__half>(cb[0] * rb, cb[1] * rb));
    const uint32_t pb1 = movmatrix_t(pack2<__half>(cb[2] * rb, cb[3] * rb));
    // o += (P_a V_a + P_b V_b) factor
    auto values = [&](uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, float factor) {
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
          for (int q = 0; q < 4; ++q) o[ch + e][q] = fmaf(ta[e][q], factor, o[ch + e][q]);
      }
    };
    if (!apart) {
      values(pa0, pa1, pb0, pb1, vs);
    } else {  // more than a factor 64 between the pages: one after the other
#pragma unroll 1
      for (int x = 0; x < 2; ++x) {
        const uint32_t q0 = movmatrix_t(pack2<__half>(cb[0], cb[1])), q1 = movmatrix_t(pack2<__half>(cb[2], cb[3]));
        values(x ? 0u : pa0, x ? 0u : pa1, x ? q0 : 0u, x ? q1 : 0u, x ? vs1 : vs0);
      }
    }
    __syncwarp();
    if (lane == 0 && i + NSTAGE < n_my) issue(i + NSTAGE);
  }
  if (timed_out_at >= 0) {
    // Drain this warp's loads still in flight (each wait bounded again) before leaving.
    if (lane == 0) report(FA_DEVERR_TIMEOUT);
    for (int j = timed_out_at + 1; j < n_my && j < timed_out_at + NSTAGE; ++j)
      mbar_wait(bar0 + (j % NSTAGE) * 8, (j / NSTAGE) & 1);
  }
#pragma unroll
  for (int x = 4; x < 32; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  __syncthreads();  // every warp is done with its ring: reuse it as reduction scratch

  // ---- combine the 4 warps ------------------------------------------------------------------
  float *red_o = reinterpret_cast<float *>(smem);                           // [W][8][HD+4]
  float *red_m = red_o + kDecodeWarps * 8 * S::kRedStride;                  // [W][8]
  float *red_l = red_m + kDecodeWarps * 8;                                  // [W][8]
  float *s_lse = red_l + kDecodeWarps * 8;                                  // [8][max_splits]
  {
    float *ro = red_o + warp * 8 * S::kRedStride;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      *reinterpret_cast<float2 *>(ro + (2 * t) * S::kRedStride + c * 16 + 2 * g) =
          make_float2(o[c][0], o[c][2]);
      *reinterpret_cast<float2 *>(ro + (2 * t + 1) * S::kRedStride + c * 16 + 2 * g) =
          make_float2(o[c][1], o[c][3]);
    }
    if (g == 0) {
      red_m[warp * 8 + 2 * t] = m0;
      red_m[warp * 8 + 2 * t + 1] = m1;
      red_l[warp * 8 + 2 * t] = l0;
      red_l[warp * 8 + 2 * t + 1] = l1;
    }
  }
  __syncthreads();

  const int hq0 = kvh * n_rep;
  const bool single = n_splits == 1;
  for (int idx = tid; idx < n_rep * HD; idx += kDecodeThreads) {
    const int h = idx / HD, x = idx % HD;
    float M = neg_inf();
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) M = fmaxf(M, red_m[w * 8 + h]);
    float O = 0.f, Lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float e = ex2(red_m[w * 8 + h] - M);  // warps without pages: m = -inf -> 0
      O += e * red_o[(w * 8 + h) * S::kRedStride + x];
      Lsum += e * red_l[w * 8 + h];
    }
    const size_t ob = size_t(b) * p.num_heads + hq0 + h;
    if (single) {
      store_out<T>(p, b, hq0 + h, HD, x, O / Lsum);
    } else {
      const size_t pi = ob * p.max_splits + split;
      p.part_o[pi * HD + x] = O / Lsum;
      if (x == 0) p.part_lse[pi] = M + __log2f(Lsum);
    }
  }
  if (single) return;

  // ---- last split of this (sequence, kv_head) merges the partials ------------------------
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    const int prev = atomicAdd(&p.counters[b * p.num_kv_heads + kvh], 1);
    s_flag[0] = (prev == n_splits - 1);
  }
  __syncthreads();
  if (!s_flag[0]) return;
  __threadfence();
  for (int idx = tid; idx < n_rep * n_splits; idx += kDecodeThreads) {
    const int h = idx / n_splits, sp = idx % n_splits;
    s_lse[h * kDecodeMaxSplits + sp] =
        __ldcg(&p.part_lse[(size_t(b) * p.num_heads + hq0 + h) * p.max_splits + sp]);
  }
  __syncthreads();
  for (int idx = tid; idx < n_rep * HD; idx += kDecodeThreads) {
    const int h = idx / HD, x = idx % HD;
    const float *lse = s_lse + h * kDecodeMaxSplits;
    float M = neg_inf();
    for (int sp = 0; sp < n_splits; ++sp) M = fmaxf(M, lse[sp]);
    const size_t ob = size_t(b) * p.num_heads + hq0 + h;
    const float *po = p.part_o + ob * p.max_splits * HD + x;
    float O = 0.f, W = 0.f;
    for (int sp = 0; sp < n_splits; ++sp) {
      const float w = ex2(lse[sp] - M);
      O += w * __ldcg(po + size_t(sp) * HD);
      W += w;
    }
    store_out<T>(p, b, hq0 + h, HD, x, O / W);
  }
  if (tid == 0) p.counters[b * p.num_kv_heads + kvh] = 0;  // ready for the next launch
}

}  // namespace fa
