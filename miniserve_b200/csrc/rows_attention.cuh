// Kernel F: paged attention of up to 32 query tokens per work item, through an 8-bit pool (decode
// rows, verify rows, chunks of up to 64 tokens) or over a tree of drafted tokens (bf16 or 8-bit pool).
//
// One CTA owns (item, KV head): query rows r = token * 2 + head-in-pair, up to 64 of them, against
// a contiguous range of the sequence's pages.  A producer warp streams whole pages (K and V of
// this head) into a ring; four consumer warps form R row groups of 16 rows (R = 1, 2 or 4, the
// smallest that holds the rows) times 4 / R page phases, so a short tile still uses every warp: warp
// w takes row group w % R and the page pairs i with i % (4 / R) == w / R.  The phases merge through the
// idle ring at the end.
//
// The mathematics per page (16 keys), in the exp2 domain with an online softmax:
//   S = Q K^T, p = 2^(S c - m) with c = scale log2(e), l += p, O += p V, out = O / l.
// A tree token sees the cached context and the drafts its mask names (ancestors and itself); a row
// that sees nothing writes zeros.
//
// bf16 pool: mma.sync m16n8k16 with bf16 operands, as in kernel B.
//
// 8-bit pool: mma.sync m16n8k16 with f16 operands.  e4m3 codes are f16 values, so they are converted
// exactly, two codes per instruction, after ldmatrix has brought them (16-bit units of two codes)
// to the lanes.  K: a lane's word is four neighbouring dims of one key; the query fragments are
// loaded in that order of dims, so two conversions give a B operand.  V: ldmatrix.trans
// leaves two neighbouring columns of two neighbouring tokens in a word; one byte permute and two
// conversions give the operands of two column tiles (even and odd columns).  The query row (bf16, 8
// significant bits) is scaled by a power of two into f16's range: exact down to 2^-33 of its
// largest value.  (mma.sync on e4m3 operands would need no conversion, but it runs at less than
// half the rate per product here: 256 decode rows took 431 us with K multiplied that way.)
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
  // A multiple of 8: a slot's previous fill is then a page of the same phase (the parity waits
  // are exact only then).
  static constexpr int kStages = kKv8 ? 16 : 8;
  static constexpr int kBatch = 4;  // pages the producer's lanes issue side by side
  static_assert(kStages % kBatch == 0 && kBatch <= 32, "a lane's pages reuse the same slots");
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
  float inv_e;   // 2^(127 - E)
  uint32_t hot;  // E + 7 in every byte (0 while E is unset)
};

// A warp takes two pages (32 keys) at a time: the products of one page hide the latencies of the
// other, and one maximum, one vote and one rescale serve both (256 decode rows over an 8-bit pool:
// 219 us page by page).
constexpr int kBlockPages = 2;

// Raises the running maxima to the block's (mx, in exp2 units) where they exceed them by 2^8, and,
// for an 8-bit pool, E to the block's largest exponent byte (vw: this thread's exponent words,
// invisible keys as 0) where that exceeds it by 7; O and l follow.
template <bool kKv8>
__device__ __forceinline__ void raise(RowsState& st, float mx0, float mx1,
                                      const uint32_t (&vw)[kBlockPages]) {
  const bool up0 = mx0 > st.m[0] + 8.f, up1 = mx1 > st.m[1] + 8.f;
  bool hot = false;
  uint32_t top4 = 0;
  if constexpr (kKv8) {
    top4 = __vmaxu4(vw[0], vw[1]);
    // Any byte above E + 7 (E >= 0 once set; an unset E lets everything through).
    hot = __vcmpgtu4(top4, st.hot) != 0;
  }
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
    for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = static_cast<int>(vw[t] >> (8 * i) & 255u);
        top = max(top, e == static_cast<int>(kExpNan) ? 0 : e);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (top > st.eb + 7 || st.eb < 0) {
      const int d = st.eb - top + kExpBias;  // 2^(E_old - E_new); O is still zero when E was unset
      const float f = d <= 0 ? 0.f : __int_as_float(d << 23);
      al0 *= f;
      al1 *= f;
      st.eb = top;
      st.inv_e = __int_as_float((2 * kExpBias - top) << 23);
      st.hot = static_cast<uint32_t>(min(top + 7, 255)) * 0x01010101u;
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

// Row maxima of the block over the quad that holds a row.
__device__ __forceinline__ void block_max(const float (&s)[2 * kBlockPages][4], float& mx0,
                                          float& mx1) {
  mx0 = fmaxf(s[0][0], s[0][1]);
  mx1 = fmaxf(s[0][2], s[0][3]);
#pragma unroll
  for (int t = 1; t < 2 * kBlockPages; ++t) {
    mx0 = fmaxf(mx0, fmaxf(s[t][0], s[t][1]));
    mx1 = fmaxf(mx1, fmaxf(s[t][2], s[t][3]));
  }
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
}

// p = 2^(s c - m) in place, and its sums into l.
__device__ __forceinline__ void block_exp(float (&s)[2 * kBlockPages][4], float c0, float c1,
                                          RowsState& st) {
  const float mu0 = st.m[0] == -INFINITY ? 0.f : st.m[0];
  const float mu1 = st.m[1] == -INFINITY ? 0.f : st.m[1];
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int t = 0; t < 2 * kBlockPages; ++t) {
    s[t][0] = fast_exp2(__fmaf_rn(s[t][0], c0, -mu0));
    s[t][1] = fast_exp2(__fmaf_rn(s[t][1], c0, -mu0));
    s[t][2] = fast_exp2(__fmaf_rn(s[t][2], c1, -mu1));
    s[t][3] = fast_exp2(__fmaf_rn(s[t][3], c1, -mu1));
    l0 += s[t][0] + s[t][1];
    l1 += s[t][2] + s[t][3];
  }
  st.l[0] += l0;
  st.l[1] += l1;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t w;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(addr));
  return w;
}

// 2^(b - 127) of byte i of a word of exponent bytes (infinity for 255, 0 for 0).
template <int i>
__device__ __forceinline__ float scale_of_byte(uint32_t w) {
  const uint32_t m = i == 3 ? w >> 1 : w << (23 - 8 * i);
  return __uint_as_float(m & 0x7f800000u);
}

// ---- two pages, 8-bit pool ----------------------------------------------------------------------

// qf: the query rows' fragments, f16, dims 16 ks + 4 (lane % 4) .. + 3 of rows r0, r1.  c0, c1: scale
// log2(e) times the rows' query scale.  Key column j of tile t (of two per page) is token
// 4 (j / 2) + j % 2 + 2 t, so a thread's four keys of a page are neighbours (4 (lane % 4) .. + 3) and
// their exponent bytes one word.  Accumulator tile 2u + p holds columns 16u + 2j + p, so a thread's
// o[2u][0], o[2u + 1][0], o[2u][1], o[2u + 1][1] are four neighbouring columns.  vis: bit k of page t
// in vis[t] (kMask only).
template <bool kMask>
__device__ __forceinline__ void rows_block8(const uint32_t (&page)[kBlockPages],
                                            const uint32_t (&qf)[8][4], RowsState& st, float c0,
                                            float c1, const uint32_t (&vis0)[kBlockPages],
                                            const uint32_t (&vis1)[kBlockPages], int lane) {
  const int mi = lane >> 3, t8 = lane & 7, q4 = 4 * (lane & 3);
  const int tok = 4 * (t8 >> 1) + (t8 & 1);  // this lane's ldmatrix row in tile 0
  const int sw = code_swizzle8(tok);         // the same for tok + 2
  float s[2 * kBlockPages][4];
#pragma unroll
  for (int t = 0; t < 2 * kBlockPages; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int t = 0; t < 2 * kBlockPages; ++t) {
      uint32_t b[4];
      ldsm_x4(page[t >> 1] + (tok + 2 * (t & 1)) * kRow8Bytes + (((4 * u + mi) ^ sw) << 4), b[0],
              b[1], b[2], b[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mma_f16(s[t], qf[4 * u + i], e4m3x2_to_f16x2<0>(b[i]), e4m3x2_to_f16x2<1>(b[i]));
    }
  }
  uint32_t vw[kBlockPages], keep[kBlockPages][2];
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    const uint32_t kw = lds32(page[t] + kExp8Off + q4);
    vw[t] = lds32(page[t] + kExp8Off + kBlockTokens + q4);
    const float f[4] = {scale_of_byte<0>(kw), scale_of_byte<1>(kw), scale_of_byte<2>(kw),
                        scale_of_byte<3>(kw)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[2 * t][i] *= f[i & 1];
      s[2 * t + 1][i] *= f[2 + (i & 1)];
    }
    if constexpr (kMask) {
      // Rows of keys no row here sees may hold anything (pages of a finished sequence, unused
      // drafts, a second page that is not there): their values and exponents become zero.
      const uint32_t v0 = vis0[t] >> q4, v1 = vis1[t] >> q4;
      const uint32_t any = __reduce_or_sync(0xffffffffu, vis0[t] | vis1[t]) >> q4;
      keep[t][0] = (any & 1u ? 0xffffu : 0u) | (any & 2u ? 0xffff0000u : 0u);
      keep[t][1] = (any & 4u ? 0xffffu : 0u) | (any & 8u ? 0xffff0000u : 0u);
      vw[t] &= (any & 1u ? 0xffu : 0u) | (any & 2u ? 0xff00u : 0u) | (any & 4u ? 0xff0000u : 0u) |
               (any & 8u ? 0xff000000u : 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = (i & 2) ? v1 : v0;
        if (!(v >> (i & 1) & 1u)) s[2 * t][i] = -INFINITY;
        if (!(v >> (2 + (i & 1)) & 1u)) s[2 * t + 1][i] = -INFINITY;
      }
    }
  }
  float mx0, mx1;
  block_max(s, mx0, mx1);
  raise<true>(st, mx0 * c0, mx1 * c1, vw);
  block_exp(s, c0, c1, st);
  const int vtok = tok + 2 * (mi & 1);
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    const float f[4] = {scale_of_byte<0>(vw[t]) * st.inv_e, scale_of_byte<1>(vw[t]) * st.inv_e,
                        scale_of_byte<2>(vw[t]) * st.inv_e, scale_of_byte<3>(vw[t]) * st.inv_e};
    float p[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[0][i] = s[2 * t][i] * f[i & 1];
      p[1][i] = s[2 * t + 1][i] * f[2 + (i & 1)];
      if constexpr (kMask) {
        // A key this row does not see contributes nothing, whatever its exponent byte.
        const uint32_t v = ((i & 2) ? vis1[t] : vis0[t]) >> q4;
        if (!(v >> (i & 1) & 1u)) p[0][i] = 0.f;
        if (!(v >> (2 + (i & 1)) & 1u)) p[1][i] = 0.f;
      }
    }
    const uint32_t pa[4] = {pack_f16(p[0][0], p[0][1]), pack_f16(p[0][2], p[0][3]),
                            pack_f16(p[1][0], p[1][1]), pack_f16(p[1][2], p[1][3])};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t w[4];
      ldsm_x4_t(page[t] + kCodes8Bytes + vtok * kRow8Bytes + (((2 * u + (mi >> 1)) ^ sw) << 4), w[0],
                w[1], w[2], w[3]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t a = w[2 * h], b = w[2 * h + 1];
        if constexpr (kMask) {
          a &= keep[t][0];
          b &= keep[t][1];
        }
        // Bytes (token t: columns 2j, 2j + 1; token t + 1: the same) -> column 2j of both tokens
        // in the low half, column 2j + 1 in the high half.
        a = __byte_perm(a, 0, 0x3120);
        b = __byte_perm(b, 0, 0x3120);
        mma_f16(st.o[4 * u + 2 * h], pa, e4m3x2_to_f16x2<0>(a), e4m3x2_to_f16x2<0>(b));
        mma_f16(st.o[4 * u + 2 * h + 1], pa, e4m3x2_to_f16x2<1>(a), e4m3x2_to_f16x2<1>(b));
      }
    }
  }
}

// ---- two pages, bf16 pool -----------------------------------------------------------------------

__device__ __forceinline__ bool bf16_pair_bad(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// qf: query fragments as in kernel B; a thread's keys of a page are 2q, 2q + 1, 2q + 8, 2q + 9
// (q = lane % 4).  Accumulator tile n holds columns 8n + 2q, 8n + 2q + 1.
template <bool kMask>
__device__ __forceinline__ void rows_block16(const uint32_t (&page)[kBlockPages],
                                             const uint32_t (&qf)[8][4], RowsState& st, float c,
                                             const uint32_t (&vis0)[kBlockPages],
                                             const uint32_t (&vis1)[kBlockPages], int lane) {
  const int mi = lane >> 3, q2 = 2 * (lane & 3);
  float s[2 * kBlockPages][4];
#pragma unroll
  for (int t = 0; t < 2 * kBlockPages; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      uint32_t b0, b1, b2, b3;
      ldsm_x4(page[t] + swz_off((lane & 7) + (mi >> 1) * 8, ks * 16 + (mi & 1) * 8, 16), b0, b1, b2,
              b3);
      mma_bf16(s[2 * t], qf[ks], b0, b1);
      mma_bf16(s[2 * t + 1], qf[ks], b2, b3);
    }
  }
  uint32_t keep[kBlockPages][2];
  if constexpr (kMask) {
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      const uint32_t any = __reduce_or_sync(0xffffffffu, vis0[t] | vis1[t]) >> q2;
      keep[t][0] = (any & 1u ? 0xffffu : 0u) | (any & 2u ? 0xffff0000u : 0u);
      keep[t][1] = (any & 0x100u ? 0xffffu : 0u) | (any & 0x200u ? 0xffff0000u : 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = ((i & 2) ? vis1[t] : vis0[t]) >> q2;
        if (!(v >> (i & 1) & 1u)) s[2 * t][i] = -INFINITY;
        if (!(v >> (8 + (i & 1)) & 1u)) s[2 * t + 1][i] = -INFINITY;
      }
    }
  }
  float mx0, mx1;
  block_max(s, mx0, mx1);
  const uint32_t none[kBlockPages] = {};
  raise<false>(st, mx0 * c, mx1 * c, none);
  block_exp(s, c, c, st);
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    // p is rounded to bf16 for the product (half a step of 2^-8), as in kernels B and D.
    const float(&p0)[4] = s[2 * t];
    const float(&p1)[4] = s[2 * t + 1];
    const uint32_t pa[4] = {pack_bf16(p0[0], p0[1]), pack_bf16(p0[2], p0[3]),
                            pack_bf16(p1[0], p1[1]), pack_bf16(p1[2], p1[3])};
    const int key = (lane & 7) + (mi & 1) * 8;
    const uint32_t vbase = page[t] + kPageBytes;
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
          b[i] &= keep[t][i & 1];
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
          const bool see0 = vis0[t] >> k & 1u, see1 = vis1[t] >> k & 1u;
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const uint32_t w = lds32(vbase + swz_off(k, n * 8 + q2, 16));
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
__global__ void __launch_bounds__(kRowsThreads, 2)
    rows_attn_kernel(const __grid_constant__ CUtensorMap kv_map, const RowsArgs ra) {
  using Cfg = RowsCfg<kKv8>;
  constexpr int kStages = Cfg::kStages, kBatch = Cfg::kBatch;
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
    // Lane i of the first kBatch takes the pages j with j % kBatch == i: the lanes wait for their
    // slots and issue their copies side by side.  (One lane issuing every page takes a chain of
    // several hundred cycles per page, which three CTAs of 4 KiB pages per SM cannot afford.)
    const uint64_t policy = l2_policy_evict_first();
    const int* table = a.tables + table_off + page_begin;
    int issued = 0;  // by this lane
    bool stop = false;
    for (int j0 = 0; j0 < npages && !stop; j0 += 32) {
      const int mine = j0 + lane < npages ? table[j0 + lane] : 0;
      for (int b = 0; b < 32 && j0 + b < npages; b += kBatch) {
        const int blk = __shfl_sync(0xffffffffu, mine, b + (lane & (kBatch - 1)));
        const int j = j0 + b + lane;
        bool ok = *abort_flag == 0;
        if (ok && lane < kBatch && j < npages) {
          const int s = j % kStages;
          if (j >= kStages && !mbar_wait(&empty[s], ((j / kStages) - 1) & 1)) {
            atomicOr(&g_status_word, kErrTimeout);
            *abort_flag = 1;
            ok = false;
          } else {
            const bool inside = static_cast<unsigned>(blk) < static_cast<unsigned>(a.num_blocks);
            uint8_t* dst = ring + s * Cfg::kPage;
            // Block ids outside the pool are flagged and read as zeros (the TMA unit's fill, or
            // written here).
            if (!inside) atomicOr(&g_status_word, kErrBlock);
            if constexpr (kKv8) {
              if (inside) {
                mbar_arrive_expect_tx(&full[s], Cfg::kPage);
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::"
                    "cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
                    "l"(ra.pool + (static_cast<long long>(blk) * a.num_kv + kvh) * Cfg::kPage),
                    "r"(Cfg::kPage), "r"(smem_u32(&full[s])), "l"(policy)
                    : "memory");
              } else {
                for (int i = 0; i < Cfg::kPage / 16; ++i)
                  reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
                // Later copies into the slot go through the async proxy.
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&full[s]);
              }
            } else {
              mbar_arrive_expect_tx(&full[s], Cfg::kPage);
              tma_load_5d(dst, &kv_map, &full[s], 0, 0, 0, kvh, blk, policy);
            }
            ++issued;
          }
        }
        if (!__all_sync(0xffffffffu, ok)) {
          stop = true;
          break;
        }
      }
    }
    // Drain: never leave the CTA with a copy in flight.
    constexpr int kPerLane = kStages / kBatch;
    for (int i = issued > kPerLane ? issued - kPerLane : 0; i < issued; ++i) {
      const int j = i * kBatch + lane;
      if (!mbar_wait(&full[j % kStages], (j / kStages) & 1)) {
        atomicOr(&g_status_word, kErrTimeout);
        break;
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
  uint32_t qf[8][4];
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
        qf[i][r] = pack_f16(bf16_lo(x[r][i].x) * inv, bf16_hi(x[r][i].x) * inv);
        qf[i][2 + r] = pack_f16(bf16_lo(x[r][i].y) * inv, bf16_hi(x[r][i].y) * inv);
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
  st.hot = 0;
  const int qpos0 = num_cached + tok0 + tk0, qpos1 = num_cached + tok0 + tk1;
  // First key position that some row of the tile may not see.
  const int first_masked = kTree ? num_cached : num_cached + tok0 + (row_base >> 1) + 1;
  const uint32_t ring_u32 = smem_u32(ring);
  for (int j = phase * kBlockPages; j < npages; j += phases * kBlockPages) {
    const int cnt = min(kBlockPages, npages - j);
    uint32_t page[kBlockPages];
    bool ok = true;
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      // A second page that is not there is masked out; its slot's leftovers are read.
      const int s = (j + t) % kStages;
      page[t] = ring_u32 + s * Cfg::kPage;
      if (t < cnt) ok = ok && mbar_wait_fast(&full[s], ((j + t) / kStages) & 1, abort_flag);
    }
    // Leave the loop only as a whole warp: the tensor-core operations are warp-collective.
    if (!__all_sync(0xffffffffu, ok)) {
      if (lane == 0) {
        atomicOr(&g_status_word, kErrTimeout);
        *abort_flag = 1;
      }
      break;
    }
    const int key0 = (page_begin + j) * kBlockTokens;
    if (warp_active) {
      uint32_t vis0[kBlockPages], vis1[kBlockPages];
      if (cnt < kBlockPages || key0 + kBlockPages * kBlockTokens > first_masked) {
#pragma unroll
        for (int t = 0; t < kBlockPages; ++t) {
          const int k0 = key0 + t * kBlockTokens;
          if (k0 + kBlockTokens <= first_masked) {
            vis0[t] = live0 ? 0xffffu : 0u;
            vis1[t] = live1 ? 0xffffu : 0u;
          } else if constexpr (kTree) {
            vis0[t] = live0 ? tree_bits(mask0, words, k0 - num_cached) : 0u;
            vis1[t] = live1 ? tree_bits(mask1, words, k0 - num_cached) : 0u;
          } else {
            vis0[t] = live0 ? causal_bits(qpos0, k0) : 0u;
            vis1[t] = live1 ? causal_bits(qpos1, k0) : 0u;
          }
          if (t >= cnt) vis0[t] = vis1[t] = 0u;
        }
        if constexpr (kKv8)
          rows_block8<true>(page, qf, st, c0, c1, vis0, vis1, lane);
        else
          rows_block16<true>(page, qf, st, c0, vis0, vis1, lane);
      } else {
#pragma unroll
        for (int t = 0; t < kBlockPages; ++t) vis0[t] = vis1[t] = 0xffffu;
        if constexpr (kKv8)
          rows_block8<false>(page, qf, st, c0, c1, vis0, vis1, lane);
        else
          rows_block16<false>(page, qf, st, c0, vis0, vis1, lane);
      }
    }
    __syncwarp();
    if (lane < cnt) mbar_arrive(&empty[(j + lane) % kStages]);
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
