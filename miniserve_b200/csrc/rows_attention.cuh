// Kernel F: paged attention of up to 32 query tokens per work item, through an 8-bit pool (decode
// rows, verify rows, chunks of up to 64 tokens) or over a tree of drafted tokens (bf16 or 8-bit pool).
//
// One CTA owns (item, KV head): query rows r = token * 2 + head-in-pair, up to 64 of them, against
// a contiguous range of the sequence's pages.  A producer warp streams whole pages (K and V of
// this head) into a ring; four consumer warps form R row groups of 16 rows (R = 1, 2 or 4, the
// smallest that holds the rows) times 4 / R page phases, so a short tile still uses every warp: warp
// w takes row group w % R and the pages j with j % (4 / R) == w / R.  The phases merge through the
// idle ring at the end.
//
// The mathematics per page (16 keys), in the exp2 domain with an online softmax:
//   S = Q K^T, p = 2^(S c - m) with c = scale log2(e), l += p, O += p V, out = O / l.
// A tree token sees the cached context and the drafts its mask names (ancestors and itself); a row
// that sees nothing writes zeros.
//
// bf16 pool: mma.sync m16n8k16 with bf16 operands, as in kernel B.
//
// 8-bit pool.  K needs no conversion: mma.sync m16n8k32 multiplies e4m3 codes directly, so a
// query row (bf16, 8 significant bits) is written as two e4m3 rows, q 2^-e = hi + lo / 16, each of 4
// significant bits.  hi is the nearest e4m3 to q 2^-e, the remainder is exact, and lo holds it to
// 2^-14 against a row maximum of up to 448: S is as exact as fp32 accumulation (2^-23 of the row's
// largest |q|).  The two products run at four times the rate per multiply of the bf16 form (1.07
// against 2.0 cycles per SM and warp instruction, twice the depth, measured), and K's page is read
// once for both query heads as it lies in memory.
// V's codes become f16 pairs (exact) on the way to the P V product: ldmatrix.trans moves 16-bit
// units, so a register holds two neighbouring columns of two neighbouring tokens; one byte permute and
// two conversions give the B operands of two column tiles (even and odd columns).
// The row exponents of K multiply S's columns in fp32; those of V multiply p before it is rounded
// to f16: p 2^(b - E), with E the largest exponent byte this warp has met (raised only when a page
// exceeds it by more than 7, as the running maximum is raised only beyond 2^8, so a product stays
// below 2^15).  f16 keeps 11 bits of p, three more than the bf16 form; what it drops lies 2^-40
// below the largest p 2^b.
#pragma once

#include "kv8.cuh"
#include "paged_attention.cuh"

namespace ms {

constexpr int kRowsWarps = 4;                        // consumer warps
constexpr int kRowsThreads = (kRowsWarps + 1) * 32;  // and one producer warp
constexpr int kRowsTokens = 32;                      // query tokens of a work item (64 rows)

struct RowsArgs {
  AttnArgs a;           // queries, output, plan sections, partials
  const uint8_t* pool;  // 8-bit layer (null for a bf16 pool, which the tensor map describes)
  const int* plan;      // start of the packed plan: tree masks are at sequence record field 6
  int n_single;         // items of one tile; the items after them are two tiles of 32 tokens
};

template <bool kKv8>
struct RowsCfg {
  static constexpr int kPage = kKv8 ? kPage8Bytes : kPageKVBytes;
  // A multiple of 4: a slot's previous fill is then a page of the same phase (the parity waits
  // are exact only then).
  static constexpr int kStages = kKv8 ? 16 : 8;
  static constexpr int kStageBytes = kStages * kPage;
  // Merge scratch in the ring: per warp 16 column tiles and (m, l), a float4 per lane each.
  static_assert(kRowsWarps * 17 * 32 * 16 <= kStageBytes, "merge scratch reuses the ring");
  static constexpr int kBarOffset = kStageBytes;
  static constexpr int kSmemBytes = 1024 + kBarOffset + 2 * kStages * 8 + 16;
};

// ---- small pieces -----------------------------------------------------------------------------

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Which of a page's 16 keys (bit k: key0 + k) the query at position qpos sees: keys 0..qpos.
__device__ __forceinline__ uint32_t causal_bits(int qpos, int key0) {
  const int d = qpos - key0;
  return d < 0 ? 0u : (d >= 15 ? 0xffffu : (2u << d) - 1u);
}

// The same for a tree token: `row` is its mask (bit j: it sees draft j), `words` its length, and
// `first` the page's first key relative to the first draft (negative: cached keys before it).
__device__ __forceinline__ uint32_t tree_bits(const int* row, int words, int first) {
  const int at = max(first, 0);
  const int w = at >> 5, sh = at & 31;
  const uint32_t lo = w < words ? static_cast<uint32_t>(__ldg(row + w)) : 0u;
  const uint32_t hi = w + 1 < words ? static_cast<uint32_t>(__ldg(row + w + 1)) : 0u;
  uint32_t bits = __funnelshift_r(lo, hi, sh);
  if (first < 0) bits = (bits << -first) | ((1u << -first) - 1u);
  return bits & 0xffffu;
}

// Per-thread state of one row group: rows r0 = lane / 4 and r1 = r0 + 8 of the group.
struct RowsState {
  float o[16][4];
  float m[2], l[2];
  int eb;      // 8-bit pool: the exponent byte E that O is held against
  float inv_e; // 2^(127 - E)
};

// Raises the running maxima to the page's (mx, in exp2 units) where they exceed them by 2^8, and,
// for an 8-bit pool, E to the page's largest exponent byte (vb: this thread's four, invisible keys as
// 0) where that exceeds it by 7; O and l follow.
template <bool kKv8>
__device__ __forceinline__ void raise(RowsState& st, float mx0, float mx1, const int (&vb)[4]) {
  const bool up0 = mx0 > st.m[0] + 8.f, up1 = mx1 > st.m[1] + 8.f;
  bool hot = false;
  if constexpr (kKv8) hot = max(max(vb[0], vb[1]), max(vb[2], vb[3])) > st.eb + 7;
  if (!__any_sync(0xffffffffu, up0 || up1 || hot)) return;
  float al0 = 1.f, al1 = 1.f;
  if (up0) {
    al0 = fast_exp2(st.m[0] - mx0);
    st.m[0] = mx0;
  }
  if (up1) {
    al1 = fast_exp2(st.m[1] - mx1);
    st.m[1] = mx1;
  }
  st.l[0] *= al0;
  st.l[1] *= al1;
  if constexpr (kKv8) {
    // The largest exponent of a finite row (a NaN row's 255 does not move E: it acts through its
    // infinite factor, and only on the rows that see it).
    int top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, vb[i] == static_cast<int>(kExpNan) ? 0 : vb[i]);
    top = __reduce_max_sync(0xffffffffu, top);
    if (top > st.eb + 7 || st.eb < 0) {
      const int d = st.eb - top + kExpBias;  // 2^(E_old - E_new); O is still zero when E was unset
      const float f = d <= 0 ? 0.f : __int_as_float(d << 23);
      al0 *= f;
      al1 *= f;
      st.eb = top;
      st.inv_e = __int_as_float((2 * kExpBias - top) << 23);
    }
  }
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    st.o[n][0] *= al0;
    st.o[n][1] *= al0;
    st.o[n][2] *= al1;
    st.o[n][3] *= al1;
  }
}

// Masked scores of a thread's 8 (row, key) pairs: keys 2q, 2q + 1 (s0) and 2q + 8, 2q + 9 (s1).
__device__ __forceinline__ void mask_scores(float (&s0)[4], float (&s1)[4], uint32_t vis0,
                                            uint32_t vis1, int q2) {
  const float ninf = -INFINITY;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!(vis0 >> (q2 + i) & 1u)) s0[i] = ninf;
    if (!(vis1 >> (q2 + i) & 1u)) s0[2 + i] = ninf;
    if (!(vis0 >> (q2 + 8 + i) & 1u)) s1[i] = ninf;
    if (!(vis1 >> (q2 + 8 + i) & 1u)) s1[2 + i] = ninf;
  }
}

// Row maxima of the page over the quad that holds a row.
__device__ __forceinline__ void page_max(const float (&s0)[4], const float (&s1)[4], float& mx0,
                                         float& mx1) {
  mx0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1]));
  mx1 = fmaxf(fmaxf(s0[2], s0[3]), fmaxf(s1[2], s1[3]));
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
}

// p = 2^(s c - m) for the page, and its sums into l.
__device__ __forceinline__ void page_exp(const float (&s0)[4], const float (&s1)[4], float c0,
                                         float c1, RowsState& st, float (&p0)[4], float (&p1)[4]) {
  const float mu0 = st.m[0] == -INFINITY ? 0.f : st.m[0];
  const float mu1 = st.m[1] == -INFINITY ? 0.f : st.m[1];
  p0[0] = fast_exp2(__fmaf_rn(s0[0], c0, -mu0));
  p0[1] = fast_exp2(__fmaf_rn(s0[1], c0, -mu0));
  p0[2] = fast_exp2(__fmaf_rn(s0[2], c1, -mu1));
  p0[3] = fast_exp2(__fmaf_rn(s0[3], c1, -mu1));
  p1[0] = fast_exp2(__fmaf_rn(s1[0], c0, -mu0));
  p1[1] = fast_exp2(__fmaf_rn(s1[1], c0, -mu0));
  p1[2] = fast_exp2(__fmaf_rn(s1[2], c1, -mu1));
  p1[3] = fast_exp2(__fmaf_rn(s1[3], c1, -mu1));
  st.l[0] += (p0[0] + p0[1]) + (p1[0] + p1[1]);
  st.l[1] += (p0[2] + p0[3]) + (p1[2] + p1[3]);
}

// ---- one page, 8-bit pool -----------------------------------------------------------------------

// qh/ql: the query rows' high and low e4m3 parts, [chunk of 16 dims][row r0, r1].  c0, c1: scale
// log2(e) times the rows' query scale.  Accumulator tile 2u + p holds columns 16u + 2j + p, so a
// thread's o[2u][0], o[2u + 1][0], o[2u][1], o[2u + 1][1] are four neighbouring columns.
template <bool kMask>
__device__ __forceinline__ void rows_page8(uint32_t page, const uint32_t (&qh)[8][2],
                                           const uint32_t (&ql)[8][2], RowsState& st, float c0,
                                           float c1, uint32_t vis0, uint32_t vis1, int lane) {
  const int mi = lane >> 3, t8 = lane & 7, q2 = 2 * (lane & 3);
  float s[2][4], e[2][4];  // hi and lo products of the two key tiles
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = e[t][i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t b0, b1, b2, b3;
      ldsm_x4(page + (t * 8 + t8) * kRow8Bytes + (((4 * u + mi) ^ t8) << 4), b0, b1, b2, b3);
      mma_e4m3(s[t], qh[4 * u][0], qh[4 * u][1], qh[4 * u + 1][0], qh[4 * u + 1][1], b0, b1);
      mma_e4m3(e[t], ql[4 * u][0], ql[4 * u][1], ql[4 * u + 1][0], ql[4 * u + 1][1], b0, b1);
      mma_e4m3(s[t], qh[4 * u + 2][0], qh[4 * u + 2][1], qh[4 * u + 3][0], qh[4 * u + 3][1], b2, b3);
      mma_e4m3(e[t], ql[4 * u + 2][0], ql[4 * u + 2][1], ql[4 * u + 3][0], ql[4 * u + 3][1], b2, b3);
    }
  }
  // Exponent bytes of this thread's four keys (K, then V).
  uint32_t kb[2], vb16[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    asm volatile("ld.shared.u16 %0, [%1];" : "=r"(kb[t]) : "r"(page + kExp8Off + t * 8 + q2));
    asm volatile("ld.shared.u16 %0, [%1];"
                 : "=r"(vb16[t])
                 : "r"(page + kExp8Off + kBlockTokens + t * 8 + q2));
  }
  int vb[4] = {static_cast<int>(vb16[0] & 255u), static_cast<int>(vb16[0] >> 8),
               static_cast<int>(vb16[1] & 255u), static_cast<int>(vb16[1] >> 8)};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float fa = scale8(kb[t] & 255u), fb = scale8(kb[t] >> 8);
    s[t][0] = __fmaf_rn(e[t][0], 0.0625f, s[t][0]) * fa;
    s[t][1] = __fmaf_rn(e[t][1], 0.0625f, s[t][1]) * fb;
    s[t][2] = __fmaf_rn(e[t][2], 0.0625f, s[t][2]) * fa;
    s[t][3] = __fmaf_rn(e[t][3], 0.0625f, s[t][3]) * fb;
  }
  uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // V words of tokens some row sees
  if constexpr (kMask) {
    mask_scores(s[0], s[1], vis0, vis1, q2);
    // Rows of keys no row here sees may hold anything (pages of a finished sequence, unused drafts).
    const uint32_t any = __reduce_or_sync(0xffffffffu, vis0 | vis1);
    keep0 = (any >> q2 & 1u ? 0xffffu : 0u) | (any >> (q2 + 1) & 1u ? 0xffff0000u : 0u);
    keep1 = (any >> (q2 + 8) & 1u ? 0xffffu : 0u) | (any >> (q2 + 9) & 1u ? 0xffff0000u : 0u);
    if (!(keep0 & 0xffffu)) vb[0] = 0;
    if (!(keep0 >> 16)) vb[1] = 0;
    if (!(keep1 & 0xffffu)) vb[2] = 0;
    if (!(keep1 >> 16)) vb[3] = 0;
  }
  float mx0, mx1;
  page_max(s[0], s[1], mx0, mx1);
  raise<true>(st, mx0 * c0, mx1 * c1, vb);
  float p0[4], p1[4];
  page_exp(s[0], s[1], c0, c1, st, p0, p1);
  const float f[4] = {scale8(vb[0]) * st.inv_e, scale8(vb[1]) * st.inv_e, scale8(vb[2]) * st.inv_e,
                      scale8(vb[3]) * st.inv_e};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // A key this row does not see contributes nothing, whatever its exponent byte.
    p0[i] = kMask && s[0][i] == -INFINITY ? 0.f : p0[i] * f[i & 1];
    p1[i] = kMask && s[1][i] == -INFINITY ? 0.f : p1[i] * f[2 + (i & 1)];
  }
  const uint32_t pa[4] = {pack_f16(p0[0], p0[1]), pack_f16(p0[2], p0[3]), pack_f16(p1[0], p1[1]),
                          pack_f16(p1[2], p1[3])};
  const uint32_t vrow = page + kCodes8Bytes + (t8 + (mi & 1) * 8) * kRow8Bytes;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t w[4];
    ldsm_x4_t(vrow + (((2 * u + (mi >> 1)) ^ t8) << 4), w[0], w[1], w[2], w[3]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t a = w[2 * h], b = w[2 * h + 1];
      if constexpr (kMask) {
        a &= keep0;
        b &= keep1;
      }
      // Bytes (token t: columns 2j, 2j + 1; token t + 1: the same) -> column 2j of both tokens in
      // the low half, column 2j + 1 in the high half.
      a = __byte_perm(a, 0, 0x3120);
      b = __byte_perm(b, 0, 0x3120);
      mma_f16(st.o[4 * u + 2 * h], pa, e4m3x2_to_f16x2<0>(a), e4m3x2_to_f16x2<0>(b));
      mma_f16(st.o[4 * u + 2 * h + 1], pa, e4m3x2_to_f16x2<1>(a), e4m3x2_to_f16x2<1>(b));
    }
  }
}

// ---- one page, bf16 pool ------------------------------------------------------------------------

__device__ __forceinline__ bool bf16_pair_bad(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// qf: query fragments as in kernel B.  Accumulator tile n holds columns 8n + 2q, 8n + 2q + 1.
template <bool kMask>
__device__ __forceinline__ void rows_page16(uint32_t page, const uint32_t (&qf)[8][4],
                                            RowsState& st, float c, uint32_t vis0, uint32_t vis1,
                                            int lane) {
  const int mi = lane >> 3, q2 = 2 * (lane & 3);
  float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
  {
    const int key = (lane & 7) + (mi >> 1) * 8;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t b0, b1, b2, b3;
      ldsm_x4(page + swz_off(key, ks * 16 + (mi & 1) * 8, 16), b0, b1, b2, b3);
      mma_bf16(s0, qf[ks], b0, b1);
      mma_bf16(s1, qf[ks], b2, b3);
    }
  }
  uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
  if constexpr (kMask) {
    mask_scores(s0, s1, vis0, vis1, q2);
    const uint32_t any = __reduce_or_sync(0xffffffffu, vis0 | vis1);
    keep0 = (any >> q2 & 1u ? 0xffffu : 0u) | (any >> (q2 + 1) & 1u ? 0xffff0000u : 0u);
    keep1 = (any >> (q2 + 8) & 1u ? 0xffffu : 0u) | (any >> (q2 + 9) & 1u ? 0xffff0000u : 0u);
  }
  float mx0, mx1;
  page_max(s0, s1, mx0, mx1);
  const int none[4] = {0, 0, 0, 0};
  raise<false>(st, mx0 * c, mx1 * c, none);
  float p0[4], p1[4];
  page_exp(s0, s1, c, c, st, p0, p1);
  // p is rounded to bf16 for the product (half a step of 2^-8), as in kernels B and D.
  const uint32_t pa[4] = {pack_bf16(p0[0], p0[1]), pack_bf16(p0[2], p0[3]),
                          pack_bf16(p1[0], p1[1]), pack_bf16(p1[2], p1[3])};
  const int key = (lane & 7) + (mi & 1) * 8;
  const uint32_t vbase = page + kPageBytes;
  bool bad = false;
#pragma unroll
  for (int np = 0; np < 8; ++np) {
    uint32_t b[4];
    ldsm_x4_t(vbase + swz_off(key, np * 16 + (mi >> 1) * 8, 16), b[0], b[1], b[2], b[3]);
    if constexpr (kMask) {
      // Values of keys no row here sees are dropped; infinities and NaN of the others too, and
      // added below for the rows that do see them (0 times them would reach every row).
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[i] &= (i & 1) ? keep1 : keep0;
        if (bf16_pair_bad(b[i])) {
          bad = true;
          if ((b[i] & 0x7f80u) == 0x7f80u) b[i] &= 0xffff0000u;
          if ((b[i] & 0x7f800000u) == 0x7f800000u) b[i] &= 0xffffu;
        }
      }
    }
    mma_bf16(st.o[2 * np], pa, b[0], b[1]);
    mma_bf16(st.o[2 * np + 1], pa, b[2], b[3]);
  }
  if constexpr (kMask) {
    if (__any_sync(0xffffffffu, bad)) {
      for (int k = 0; k < 16; ++k) {
        const int src = (lane & ~3) | ((k & 7) >> 1);
        const float a0 = (k & 8) ? ((k & 1) ? p1[1] : p1[0]) : ((k & 1) ? p0[1] : p0[0]);
        const float a1 = (k & 8) ? ((k & 1) ? p1[3] : p1[2]) : ((k & 1) ? p0[3] : p0[2]);
        const float w0 = __shfl_sync(0xffffffffu, a0, src);
        const float w1 = __shfl_sync(0xffffffffu, a1, src);
        const bool see0 = vis0 >> k & 1u, see1 = vis1 >> k & 1u;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vbase + swz_off(k, n * 8 + q2, 16)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t bits = i == 0 ? w << 16 : w & 0xffff0000u;
            if ((bits & 0x7f800000u) != 0x7f800000u) continue;
            const float v = __uint_as_float(bits);
            if (see0) st.o[n][i] += w0 * v;
            if (see1) st.o[n][2 + i] += w1 * v;
          }
        }
      }
    }
  }
}

// ---- the kernel ---------------------------------------------------------------------------------

// Where one row's result goes: bf16 output, or a partial row (normalised O and log2-sum-exp), with
// the shared-prefix partial of a cascade row merged in.
struct RowOut {
  __nv_bfloat16* dst;   // output row (null: partial row)
  float* part;          // partial row
  const float* prefix;  // shared-prefix partial row to merge (null: none)
  float w, wp;          // weights of this item's O and of the prefix partial
};

__device__ __forceinline__ RowOut row_out(const AttnArgs& a, int r, int tok, bool live, float m,
                                          float L, int kvh, int part_row, int merge_row,
                                          int flat_tok, bool first_col) {
  RowOut o;
  const float inv = live && L != 0.f ? 1.f / L : 0.f;  // a NaN sum stays NaN
  o.dst = nullptr;
  o.part = nullptr;
  o.prefix = nullptr;
  o.w = inv;
  o.wp = 0.f;
  if (part_row >= 0) {
    const long long prow = static_cast<long long>(part_row + r) * a.num_kv + kvh;
    o.part = a.ws_o + prow * kHeadDim;
    if (first_col) a.ws_lse[prow] = live && L != 0.f ? m + __log2f(L) : -INFINITY;
    return o;
  }
  o.dst = a.out + static_cast<long long>(flat_tok + tok) * a.out_row_stride +
          (kvh * kGroup + (r & 1)) * kHeadDim;
  if (merge_row >= 0) {
    const long long prow = static_cast<long long>(merge_row + r) * a.num_kv + kvh;
    const float lse_p = a.ws_lse[prow];
    const float lse_u = L != 0.f ? m + __log2f(L) : -INFINITY;
    const float M = fmaxf(lse_u, lse_p);
    const float wu = lse_u == -INFINITY ? 0.f : fast_exp2(lse_u - M);
    const float wp = lse_p == -INFINITY ? 0.f : fast_exp2(lse_p - M);
    const float den = wu + wp;
    const float n = den != 0.f ? 1.f / den : 0.f;
    o.w = inv * wu * n;
    o.wp = wp * n;
    o.prefix = a.ws_o + prow * kHeadDim;
  }
  return o;
}

template <int kN>  // kN neighbouring columns from column d
__device__ __forceinline__ void put_cols(const RowOut& o, int d, const float (&x)[kN], bool live) {
  float y[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    y[i] = live ? x[i] * o.w : 0.f;
    if (o.prefix != nullptr) y[i] += o.prefix[d + i] * o.wp;
  }
  if (o.part != nullptr) {
    if constexpr (kN == 4)
      *reinterpret_cast<float4*>(o.part + d) = make_float4(y[0], y[1], y[2], y[3]);
    else
      *reinterpret_cast<float2*>(o.part + d) = make_float2(y[0], y[1]);
  } else {
    if constexpr (kN == 4)
      *reinterpret_cast<uint2*>(o.dst + d) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    else
      *reinterpret_cast<uint32_t*>(o.dst + d) = pack_bf16(y[0], y[1]);
  }
}

template <bool kKv8, bool kTree>
__global__ void __launch_bounds__(kRowsThreads, 3)
    rows_attn_kernel(const __grid_constant__ CUtensorMap kv_map, const RowsArgs ra) {
  using Cfg = RowsCfg<kKv8>;
  constexpr int kStages = Cfg::kStages;
  const AttnArgs& a = ra.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kStages);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // Work item: the first n_single items are one tile, the rest two tiles of 32 tokens.
  const int slot = blockIdx.x / a.num_kv;
  const int kvh = blockIdx.x - slot * a.num_kv;
  const int item_idx = slot < ra.n_single ? slot : ra.n_single + ((slot - ra.n_single) >> 1);
  const int sub = slot < ra.n_single ? 0 : (slot - ra.n_single) & 1;
  // The plan was copied in before the previous kernel started, so it is read before the wait.
  const int* it = a.items + static_cast<long long>(item_idx) * kRec;
  const int seq = it[0], tok0 = it[1] + sub * kRowsTokens, page_begin = it[3];
  const int n_q = min(it[2] - sub * kRowsTokens, kRowsTokens);
  const int part_row = it[5] < 0 ? -1 : it[5] + sub * kRowsTokens * kGroup;
  const int merge_row = it[7] == 1 ? it[6] : -1;
  const int* sr = a.seqs + static_cast<long long>(seq) * kRec;
  const int flat_start = sr[0], num_cached = sr[2], table_off = sr[4];
  // Keys after the tile's last token are visible to none of its rows.
  const int npages = min(it[4], (num_cached + tok0 + n_q + kBlockTokens - 1) / kBlockTokens) - page_begin;
  if (n_q <= 0) return;  // the second half of a chunk of up to 32 tokens

  const int groups = n_q * kGroup <= 16 ? 1 : (n_q * kGroup <= 32 ? 2 : 4);
  const int phases = kRowsWarps / groups;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], groups);  // one warp of each row group reads a page
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  if (warp == kRowsWarps) {
    // ---------------- producer warp ----------------
    const uint64_t policy = l2_policy_evict_first();
    const int* table = a.tables + table_off + page_begin;
    int issued = 0;
    bool stop = false;
    for (int j0 = 0; j0 < npages && !stop; j0 += 32) {
      int mine = 0;
      if (j0 + lane < npages) mine = table[j0 + lane];
      const int cnt = min(32, npages - j0);
      for (int jj = 0; jj < cnt; ++jj) {
        const int blk = __shfl_sync(0xffffffffu, mine, jj);
        const bool inside = static_cast<unsigned>(blk) < static_cast<unsigned>(a.num_blocks);
        const int s = (j0 + jj) % kStages;
        int ok = 1;
        if (lane == 0) {
          const int j = j0 + jj;
          if (*abort_flag) ok = 0;
          if (ok && j >= kStages && !mbar_wait(&empty[s], ((j / kStages) - 1) & 1)) {
            atomicOr(&g_status_word, kErrTimeout);
            *abort_flag = 1;
            ok = 0;
          }
          if (ok) {
            // Block ids outside the pool are flagged and read as zeros (the TMA unit's fill, or
            // written below).
            if (!inside) atomicOr(&g_status_word, kErrBlock);
            if constexpr (kKv8) {
              if (inside) {
                mbar_arrive_expect_tx(&full[s], Cfg::kPage);
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::"
                    "cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(ring + s * Cfg::kPage)),
                    "l"(ra.pool + (static_cast<long long>(blk) * a.num_kv + kvh) * Cfg::kPage),
                    "r"(Cfg::kPage), "r"(smem_u32(&full[s])), "l"(policy)
                    : "memory");
              }
            } else {
              mbar_arrive_expect_tx(&full[s], Cfg::kPage);
              tma_load_5d(ring + s * Cfg::kPage, &kv_map, &full[s], 0, 0, 0, kvh, blk, policy);
            }
            ++issued;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          stop = true;
          break;
        }
        if constexpr (kKv8) {
          if (!inside) {
            for (int i = lane; i < Cfg::kPage / 16; i += 32)
              reinterpret_cast<uint4*>(ring + s * Cfg::kPage)[i] = make_uint4(0u, 0u, 0u, 0u);
            // Later copies into the slot go through the async proxy.
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[s]);
          }
        }
      }
    }
    // Drain: never leave the CTA with a copy in flight.
    if (lane == 0) {
      for (int j = issued > kStages ? issued - kStages : 0; j < issued; ++j) {
        if (!mbar_wait(&full[j % kStages], (j / kStages) & 1)) {
          atomicOr(&g_status_word, kErrTimeout);
          break;
        }
      }
    }
    return;
  }

  // ---------------- consumer warps ----------------
  const int group = warp % groups, phase = warp / groups;
  const int row_base = group * 16;
  const int ra0 = row_base + (lane >> 2), ra1 = ra0 + 8;  // this thread's two rows
  const int tk0 = ra0 >> 1, tk1 = ra1 >> 1;               // and their tokens
  const bool warp_active = (row_base >> 1) < n_q;
  const int q2 = 2 * (lane & 3);

  // Query fragments, straight from memory.
  const __nv_bfloat16* qrow0 = a.q + static_cast<long long>(flat_start + tok0 + tk0) * a.q_row_stride +
                               (kvh * kGroup + (ra0 & 1)) * kHeadDim;
  const __nv_bfloat16* qrow1 = a.q + static_cast<long long>(flat_start + tok0 + tk1) * a.q_row_stride +
                               (kvh * kGroup + (ra1 & 1)) * kHeadDim;
  uint32_t qh[8][2], ql[8][2];  // 8-bit pool
  uint32_t qf[8][4];            // bf16 pool
  float c0 = a.scale_log2, c1 = a.scale_log2;
  if constexpr (kKv8) {
    uint2 x[2][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[0][i] = x[1][i] = make_uint2(0u, 0u);
      if (tk0 < n_q) x[0][i] = __ldg(reinterpret_cast<const uint2*>(qrow0 + 16 * i + 2 * q2));
      if (tk1 < n_q) x[1][i] = __ldg(reinterpret_cast<const uint2*>(qrow1 + 16 * i + 2 * q2));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        top = __vmaxu2(top, __vmaxu2(x[r][i].x & 0x7fff7fffu, x[r][i].y & 0x7fff7fffu));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int b = exp_byte8(max(top & 0xffffu, top >> 16));
      const float inv = inv_scale8(b);
      // The row's query scale; a row with a NaN or an infinity scores NaN.
      (r == 0 ? c0 : c1) *= row_scale8(b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y[4] = {bf16_lo(x[r][i].x) * inv, bf16_hi(x[r][i].x) * inv,
                            bf16_lo(x[r][i].y) * inv, bf16_hi(x[r][i].y) * inv};
        const uint32_t hi = cvt_e4m3x4(y[0], y[1], y[2], y[3]);
        const uint32_t h0 = e4m3x2_to_f16x2<0>(hi), h1 = e4m3x2_to_f16x2<1>(hi);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        qh[i][r] = hi;
        ql[i][r] = cvt_e4m3x4((y[0] - f0.x) * 16.f, (y[1] - f0.y) * 16.f, (y[2] - f1.x) * 16.f,
                              (y[3] - f1.y) * 16.f);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qf[i][0] = qf[i][1] = qf[i][2] = qf[i][3] = 0u;
      if (tk0 < n_q) {
        qf[i][0] = __ldg(reinterpret_cast<const uint32_t*>(qrow0 + 16 * i + q2));
        qf[i][2] = __ldg(reinterpret_cast<const uint32_t*>(qrow0 + 16 * i + 8 + q2));
      }
      if (tk1 < n_q) {
        qf[i][1] = __ldg(reinterpret_cast<const uint32_t*>(qrow1 + 16 * i + q2));
        qf[i][3] = __ldg(reinterpret_cast<const uint32_t*>(qrow1 + 16 * i + 8 + q2));
      }
    }
  }

  // Tree masks of the two rows' tokens; a token whose mask misses itself sees nothing.
  const int* mask0 = nullptr;
  const int* mask1 = nullptr;
  int words = 0;
  bool live0 = tk0 < n_q, live1 = tk1 < n_q;
  if constexpr (kTree) {
    words = sr[7];
    const int g0 = tok0 + min(tk0, n_q - 1), g1 = tok0 + min(tk1, n_q - 1);
    mask0 = ra.plan + sr[6] + static_cast<long long>(g0) * words;
    mask1 = ra.plan + sr[6] + static_cast<long long>(g1) * words;
    live0 = live0 && (mask0[g0 >> 5] >> (g0 & 31) & 1);
    live1 = live1 && (mask1[g1 >> 5] >> (g1 & 31) & 1);
  }

  RowsState st;
#pragma unroll
  for (int n = 0; n < 16; ++n) st.o[n][0] = st.o[n][1] = st.o[n][2] = st.o[n][3] = 0.f;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
  st.eb = -1000;
  st.inv_e = 0.f;
  const int qpos0 = num_cached + tok0 + tk0, qpos1 = num_cached + tok0 + tk1;
  // First key position that some row of the tile may not see.
  const int first_masked = kTree ? num_cached : num_cached + tok0 + (row_base >> 1) + 1;
  const uint32_t ring_u32 = smem_u32(ring);
  for (int j = phase; j < npages; j += phases) {
    const int s = j % kStages;
    // Leave the loop only as a whole warp: the tensor-core operations are warp-collective.
    const bool ok = __all_sync(0xffffffffu, mbar_wait_fast(&full[s], (j / kStages) & 1, abort_flag));
    if (!ok) {
      if (lane == 0) {
        atomicOr(&g_status_word, kErrTimeout);
        *abort_flag = 1;
      }
      break;
    }
    const int key0 = (page_begin + j) * kBlockTokens;
    const uint32_t page = ring_u32 + s * Cfg::kPage;
    if (warp_active) {
      if (key0 + kBlockTokens > first_masked) {
        uint32_t vis0, vis1;
        if constexpr (kTree) {
          vis0 = live0 ? tree_bits(mask0, words, key0 - num_cached) : 0u;
          vis1 = live1 ? tree_bits(mask1, words, key0 - num_cached) : 0u;
        } else {
          vis0 = live0 ? causal_bits(qpos0, key0) : 0u;
          vis1 = live1 ? causal_bits(qpos1, key0) : 0u;
        }
        if constexpr (kKv8)
          rows_page8<true>(page, qh, ql, st, c0, c1, vis0, vis1, lane);
        else
          rows_page16<true>(page, qf, st, c0, vis0, vis1, lane);
      } else {
        if constexpr (kKv8)
          rows_page8<false>(page, qh, ql, st, c0, c1, 0xffffu, 0xffffu, lane);
        else
          rows_page16<false>(page, qf, st, c0, 0xffffu, 0xffffu, lane);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }

#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
  }
  if constexpr (kKv8) {  // O back to the values the codes stand for
    const float f = st.eb < 0 ? 0.f : scale8(st.eb);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[n][i] *= f;
    }
  }

  if (phases == 1) {
    if (!warp_active) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = h == 0 ? ra0 : ra1;
      const int tok = r >> 1;
      if (tok >= n_q) continue;
      const bool live = h == 0 ? live0 : live1;
      const RowOut out = row_out(a, r, tok, live, st.m[h], st.l[h], kvh, part_row, merge_row,
                                 flat_start + tok0, q2 == 0);
      if constexpr (kKv8) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float x[4] = {st.o[2 * u][2 * h], st.o[2 * u + 1][2 * h], st.o[2 * u][2 * h + 1],
                              st.o[2 * u + 1][2 * h + 1]};
          put_cols<4>(out, 16 * u + 2 * q2, x, live);
        }
      } else {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const float x[2] = {st.o[n][2 * h], st.o[n][2 * h + 1]};
          put_cols<2>(out, 8 * n + q2, x, live);
        }
      }
    }
    return;
  }

  // Merge of the page phases: every warp leaves its (O, m, l) in the idle ring (each page has been
  // read once all consumer warps reach the barrier; a copy that was abandoned on a timeout is
  // drained by the producer before the CTA ends), and each warp merges and writes 16 / phases of
  // its row group's column tiles.
  float4* scratch = reinterpret_cast<float4*>(ring);
  asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
#pragma unroll
  for (int n = 0; n < 16; ++n)
    scratch[(warp * 17 + n) * 32 + lane] =
        make_float4(st.o[n][0], st.o[n][1], st.o[n][2], st.o[n][3]);
  scratch[(warp * 17 + 16) * 32 + lane] = make_float4(st.m[0], st.m[1], st.l[0], st.l[1]);
  asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
  if (!warp_active) return;
  float mx[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f}, wt[kRowsWarps][2];
#pragma unroll
  for (int p = 0; p < kRowsWarps; ++p) {
    if (p < phases) {
      const float4 ml = scratch[((p * groups + group) * 17 + 16) * 32 + lane];
      mx[0] = fmaxf(mx[0], ml.x);
      mx[1] = fmaxf(mx[1], ml.y);
    }
  }
#pragma unroll
  for (int p = 0; p < kRowsWarps; ++p) {
    wt[p][0] = wt[p][1] = 0.f;
    if (p < phases) {
      const float4 ml = scratch[((p * groups + group) * 17 + 16) * 32 + lane];
      wt[p][0] = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mx[0]);
      wt[p][1] = ml.y == -INFINITY ? 0.f : fast_exp2(ml.y - mx[1]);
      // A phase whose scores were all NaN never raised its maximum: its sum is kept as it is.
      if (ml.z != ml.z) wt[p][0] = 1.f;
      if (ml.w != ml.w) wt[p][1] = 1.f;
      L[0] += ml.z * wt[p][0];
      L[1] += ml.w * wt[p][1];
    }
  }
  const int per = 16 / phases;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = h == 0 ? ra0 : ra1;
    const int tok = r >> 1;
    if (tok >= n_q) continue;
    const bool live = h == 0 ? live0 : live1;
    const RowOut out = row_out(a, r, tok, live, mx[h], L[h], kvh, part_row, merge_row,
                               flat_start + tok0, phase == 0 && q2 == 0);
    for (int n = phase * per; n < (phase + 1) * per; n += 2) {
      float x0[2] = {0.f, 0.f}, x1[2] = {0.f, 0.f};  // tiles n and n + 1
#pragma unroll
      for (int p = 0; p < kRowsWarps; ++p) {
        if (p < phases) {
          const float2* base = reinterpret_cast<const float2*>(
              scratch + ((p * groups + group) * 17 + n) * 32 + lane);
          const float2 y0 = base[h], y1 = base[64 + h];
          x0[0] += y0.x * wt[p][h];
          x0[1] += y0.y * wt[p][h];
          x1[0] += y1.x * wt[p][h];
          x1[1] += y1.y * wt[p][h];
        }
      }
      if constexpr (kKv8) {
        const float x[4] = {x0[0], x1[0], x0[1], x1[1]};
        put_cols<4>(out, 8 * n + 2 * q2, x, live);
      } else {
        put_cols<2>(out, 8 * n + q2, x0, live);
        put_cols<2>(out, 8 * n + 8 + q2, x1, live);
      }
    }
  }
}

}  // namespace ms
