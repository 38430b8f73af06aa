// Kernel F: paged attention of up to 32 query tokens per work item, through an 8-bit pool (decode
// rows, verify rows, chunks of up to 64 tokens) or over a tree of drafted tokens (bf16 or 8-bit pool).
//
// One CTA owns (item, KV head): query rows r = token * 2 + head-in-pair against a contiguous range of
// the sequence's pages.  A producer warp streams whole pages (K and V of this head) into a ring; four
// consumer warps, kRG row groups of 16 rows each, form S = 1 or 2 row sets times 4 / S page phases,
// so a short tile still uses every warp: warp w takes row set w % S and the page pairs i with
// i % (4 / S) == w / S.  The phases merge through the idle ring at the end; the CTA that finishes last of
// a tile whose pages are split over several merges their partials (in the order of the splits).
//
// The mathematics per pair of pages (32 keys), in the exp2 domain with an online softmax:
//   S = Q K^T, p = 2^(S c - m) with c = scale log2(e), l += p, O += p V, out = O / l.
// A tree token sees the cached context and the drafts its mask names (ancestors and itself); a row
// that sees nothing writes zeros.
//
// bf16 pool: mma.sync m16n8k16 with bf16 operands, as in kernel B.
//
// 8-bit pool: mma.sync m16n8k16 with f16 operands.  e4m3 codes are f16 values, so they are converted
// exactly, two codes per instruction, after ldmatrix has brought them (16-bit units of two codes)
// to the lanes.  K: a lane's word is four neighbouring dims of one key; the query rows lie in shared
// memory in that order of dims, so two conversions give a B operand.  V: ldmatrix.trans
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
//
// Why this shape.  A decode row needs its bytes and little else: up to 32 rows per CTA, three CTAs per SM
// at 128 registers (the query rows stay in shared memory and are read again for every pair of pages).
// Tiles of more than 16 tokens are bound by the conversions and the products, so a warp holds two row
// groups (kRG = 2) and uses each converted operand twice; that takes more than 168 registers, which
// two CTAs of two warpgroups have once the producer's warpgroup hands its share to the consumers.
#pragma once

#include "kv8.cuh"
#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace ms {

constexpr int kRowsWarps = 4;        // consumer warps
constexpr int kRowsTokens = 32;      // query tokens of a wide work item (64 rows)
constexpr int kRowsNarrowTokens = 16;  // of a narrow one (32 rows)

struct RowsArgs {
  AttnArgs a;           // queries, output, plan sections, partials
  const uint8_t* pool;  // 8-bit layer (null for a bf16 pool, which the tensor map describes)
  const int* plan;      // start of the packed plan: tree masks are at sequence record field 6
  const int* combines;  // combine records of split tiles (an item names its record in field 6)
  int* arrived;         // [record][KVH] splits that have finished: zero between calls
};

template <bool kKv8, int kRG>
struct RowsCfg {
  static constexpr int kPage = kKv8 ? kPage8Bytes : kPageKVBytes;
  // A multiple of 8: a slot's previous fill is then a page of the same phase (the parity waits
  // are exact only then).
  static constexpr int kStages = kKv8 ? 16 : 8;
  static constexpr int kBatch = 4;  // pages the producer's lanes issue side by side
  static_assert(kStages % 8 == 0 && kStages % kBatch == 0, "slots are reused by the same lane, warp");
  static constexpr int kStageBytes = kStages * kPage;
  // Merge scratch in the ring: per warp 16 column tiles and (m, l) of one row group, a float4 per
  // lane each.
  static_assert(kRowsWarps * 17 * 32 * 16 <= kStageBytes, "merge scratch reuses the ring");
  static constexpr int kRows = kRG == 1 ? 32 : 64;
  static constexpr int kQOffset = (kStageBytes + 127) / 128 * 128;
  static constexpr int kScaleOffset = kQOffset + kRows * kHeadDim * 2;  // the rows' query scales
  static constexpr int kBarOffset = kScaleOffset + kRows * 4;
  static constexpr int kSmemBytes = 1024 + kBarOffset + 2 * kStages * 8 + 16;
  // kRG == 1: four consumer warps and a producer warp, three CTAs per SM.  kRG == 2: a consumer
  // warpgroup and a producer warpgroup (one warp of it works), two CTAs per SM launched with 128
  // registers per thread: 128 x 232 + 128 x 24 = 256 x 128.
  static constexpr int kThreads = kRG == 1 ? (kRowsWarps + 1) * 32 : 256;
  static constexpr int kCtasPerSm = kRG == 1 ? 3 : 2;
  static constexpr int kLaunchRegs = 128, kConsumerRegs = 232, kProducerRegs = 24;
  static_assert(128 * (kConsumerRegs + kProducerRegs) <= 256 * kLaunchRegs, "register split");
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

// A warp takes two pages (32 keys) at a time: the products of one page hide the latencies of the
// other, and one maximum, one vote and one rescale serve both.
constexpr int kBlockPages = 2;

// A thread's state: rows lane / 4 and lane / 4 + 8 of each of its warp's row groups.
template <int kRG>
struct RowsState {
  float o[kRG][16][4];
  float m[kRG][2], l[kRG][2];
  int eb;        // 8-bit pool: the exponent byte E that O is held against
  float inv_e;   // 2^(127 - E)
  uint32_t hot;  // E + 7 in every byte (0 while E is unset)
};

// Raises the running maxima to the block's (mx, in exp2 units) where they exceed them by 2^8, and,
// for an 8-bit pool, E to the block's largest exponent byte (vw: this thread's exponent words,
// invisible keys as 0) where that exceeds it by 7; O and l follow.
template <bool kKv8, int kRG>
__device__ __forceinline__ void raise(RowsState<kRG>& st, const float (&mx)[kRG][2],
                                      const uint32_t (&vw)[kBlockPages]) {
  bool up = false;
#pragma unroll
  for (int g = 0; g < kRG; ++g) up = up || mx[g][0] > st.m[g][0] + 8.f || mx[g][1] > st.m[g][1] + 8.f;
  // Any byte above E + 7 (an unset E lets everything through).
  if constexpr (kKv8) up = up || __vcmpgtu4(__vmaxu4(vw[0], vw[1]), st.hot) != 0;
  if (!__any_sync(0xffffffffu, up)) return;
  float f = 1.f;
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
      f = d <= 0 ? 0.f : __int_as_float(d << 23);
      st.eb = top;
      st.inv_e = __int_as_float((2 * kExpBias - top) << 23);
      st.hot = static_cast<uint32_t>(min(top + 7, 255)) * 0x01010101u;
    }
  }
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    float al[2] = {1.f, 1.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (mx[g][h] > st.m[g][h] + 8.f) {
        al[h] = fast_exp2(st.m[g][h] - mx[g][h]);
        st.m[g][h] = mx[g][h];
      }
      st.l[g][h] *= al[h];
      al[h] *= f;
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      st.o[g][n][0] *= al[0];
      st.o[g][n][1] *= al[0];
      st.o[g][n][2] *= al[1];
      st.o[g][n][3] *= al[1];
    }
  }
}

// Row maxima of a row group's block over the quad that holds a row.
__device__ __forceinline__ void block_max(const float (&s)[2 * kBlockPages][4], float (&mx)[2]) {
  mx[0] = fmaxf(s[0][0], s[0][1]);
  mx[1] = fmaxf(s[0][2], s[0][3]);
#pragma unroll
  for (int t = 1; t < 2 * kBlockPages; ++t) {
    mx[0] = fmaxf(mx[0], fmaxf(s[t][0], s[t][1]));
    mx[1] = fmaxf(mx[1], fmaxf(s[t][2], s[t][3]));
  }
#pragma unroll
  for (int off = 1; off <= 2; ++off) {
    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
  }
}

// p = 2^(s c - m) in place, and its sums into l.
__device__ __forceinline__ void block_exp(float (&s)[2 * kBlockPages][4], const float (&c)[2],
                                          const float (&m)[2], float (&l)[2]) {
  const float mu0 = m[0] == -INFINITY ? 0.f : m[0];
  const float mu1 = m[1] == -INFINITY ? 0.f : m[1];
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int t = 0; t < 2 * kBlockPages; ++t) {
    s[t][0] = fast_exp2(__fmaf_rn(s[t][0], c[0], -mu0));
    s[t][1] = fast_exp2(__fmaf_rn(s[t][1], c[0], -mu0));
    s[t][2] = fast_exp2(__fmaf_rn(s[t][2], c[1], -mu1));
    s[t][3] = fast_exp2(__fmaf_rn(s[t][3], c[1], -mu1));
    l0 += s[t][0] + s[t][1];
    l1 += s[t][2] + s[t][3];
  }
  l[0] += l0;
  l[1] += l1;
}

// Scores of key column col (0..15) of page t that a row does not see become -infinity.
// vis[g][h]: bit 16 t + k: row (g, h) sees key k of page t.  kCol1: the second column tile's first key.
template <int kCol1>
__device__ __forceinline__ void mask_block(float (&s)[2 * kBlockPages][4], const uint32_t (&vis)[2],
                                           int col0) {
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = vis[i >> 1] >> (16 * t + col0);
      if (!(v >> (i & 1) & 1u)) s[2 * t][i] = -INFINITY;
      if (!(v >> (kCol1 + (i & 1)) & 1u)) s[2 * t + 1][i] = -INFINITY;
    }
  }
}

// Keys that some row of the warp sees, both pages.
template <int kRG>
__device__ __forceinline__ uint32_t seen_by_any(const uint32_t (&vis)[kRG][2]) {
  uint32_t v = 0;
#pragma unroll
  for (int g = 0; g < kRG; ++g) v |= vis[g][0] | vis[g][1];
  return __reduce_or_sync(0xffffffffu, v);
}

// ---- two pages, 8-bit pool ----------------------------------------------------------------------

// q: shared address of this lane's ldmatrix row of the warp's first row group (f16, the dims of a
// 16-dim chunk in the order 0 1 4 5 8 9 12 13 2 3 6 7 10 11 14 15, so that a lane's fragment is the dims
// 4 (lane % 4) .. + 3 that its word of codes holds).  c: scale log2(e) times the rows' query scale.
// Key column j of tile t (of two per page) is token 4 (j / 2) + j % 2 + 2 t, so a thread's four
// keys of a page are neighbours (4 (lane % 4) .. + 3) and their exponent bytes one word.  Accumulator
// tile 2u + p holds columns 16u + 2j + p, so a thread's o[2u][0], o[2u + 1][0], o[2u][1],
// o[2u + 1][1] are four neighbouring columns.
template <int kRG, bool kMask>
__device__ __forceinline__ void rows_block8(const uint32_t (&page)[kBlockPages], uint32_t q,
                                            RowsState<kRG>& st, const float (&c)[kRG][2],
                                            const uint32_t (&vis)[kRG][2], int lane) {
  const int mi = lane >> 3, t8 = lane & 7, q4 = 4 * (lane & 3);
  const int tok = 4 * (t8 >> 1) + (t8 & 1);  // this lane's ldmatrix row in tile 0
  const int sw = code_swizzle8(tok);         // the same for tok + 2
  float s[kRG][2 * kBlockPages][4];
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int t = 0; t < 2 * kBlockPages; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[g][t][i] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {  // 32 dims at a time
    uint32_t qa[kRG][2][4];
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        ldsm_x4(q + g * (16 * kHeadDim * 2) + (((2 * (2 * u + i) + (mi >> 1)) ^ t8) << 4),
                qa[g][i][0], qa[g][i][1], qa[g][i][2], qa[g][i][3]);
    }
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      // Both key tiles of the page, chunks 2u and 2u + 1.
      uint32_t b[4];
      ldsm_x4(page[t] + (tok + 2 * (mi >> 1)) * kRow8Bytes + (((2 * u + (mi & 1)) ^ sw) << 4), b[0],
              b[1], b[2], b[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b0 = e4m3x2_to_f16x2<0>(b[i]), b1 = e4m3x2_to_f16x2<1>(b[i]);
#pragma unroll
        for (int g = 0; g < kRG; ++g) mma_f16(s[g][2 * t + (i >> 1)], qa[g][i & 1], b0, b1);
      }
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
    for (int g = 0; g < kRG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[g][2 * t][i] *= f[i & 1];
        s[g][2 * t + 1][i] *= f[2 + (i & 1)];
      }
    }
  }
  if constexpr (kMask) {
    // Rows of keys no row here sees may hold anything (pages of a finished sequence, unused
    // drafts, a second page that is not there): their values and exponents become zero.
    const uint32_t any = seen_by_any<kRG>(vis) >> q4;
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      const uint32_t a = any >> (16 * t);
      keep[t][0] = (a & 1u ? 0xffffu : 0u) | (a & 2u ? 0xffff0000u : 0u);
      keep[t][1] = (a & 4u ? 0xffffu : 0u) | (a & 8u ? 0xffff0000u : 0u);
      vw[t] &= (a & 1u ? 0xffu : 0u) | (a & 2u ? 0xff00u : 0u) | (a & 4u ? 0xff0000u : 0u) |
               (a & 8u ? 0xff000000u : 0u);
    }
#pragma unroll
    for (int g = 0; g < kRG; ++g) mask_block<2>(s[g], vis[g], q4);
  }
  float mx[kRG][2];
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    block_max(s[g], mx[g]);
    mx[g][0] *= c[g][0];
    mx[g][1] *= c[g][1];
  }
  raise<true, kRG>(st, mx, vw);
  uint32_t pa[kRG][kBlockPages][4];
#pragma unroll
  for (int g = 0; g < kRG; ++g) block_exp(s[g], c[g], st.m[g], st.l[g]);
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    const float f[4] = {scale_of_byte<0>(vw[t]) * st.inv_e, scale_of_byte<1>(vw[t]) * st.inv_e,
                        scale_of_byte<2>(vw[t]) * st.inv_e, scale_of_byte<3>(vw[t]) * st.inv_e};
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      float p[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[0][i] = s[g][2 * t][i] * f[i & 1];
        p[1][i] = s[g][2 * t + 1][i] * f[2 + (i & 1)];
        if constexpr (kMask) {
          // A key this row does not see contributes nothing, whatever its exponent byte.
          const uint32_t v = vis[g][i >> 1] >> (16 * t + q4);
          if (!(v >> (i & 1) & 1u)) p[0][i] = 0.f;
          if (!(v >> (2 + (i & 1)) & 1u)) p[1][i] = 0.f;
        }
      }
      pa[g][t][0] = pack_f16(p[0][0], p[0][1]);
      pa[g][t][1] = pack_f16(p[0][2], p[0][3]);
      pa[g][t][2] = pack_f16(p[1][0], p[1][1]);
      pa[g][t][3] = pack_f16(p[1][2], p[1][3]);
    }
  }
  const int vtok = tok + 2 * (mi & 1);
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
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
        const uint32_t a0 = e4m3x2_to_f16x2<0>(a), b0 = e4m3x2_to_f16x2<0>(b);
        const uint32_t a1 = e4m3x2_to_f16x2<1>(a), b1 = e4m3x2_to_f16x2<1>(b);
#pragma unroll
        for (int g = 0; g < kRG; ++g) {
          mma_f16(st.o[g][4 * u + 2 * h], pa[g][t], a0, b0);
          mma_f16(st.o[g][4 * u + 2 * h + 1], pa[g][t], a1, b1);
        }
      }
    }
  }
}

// ---- two pages, bf16 pool -----------------------------------------------------------------------

__device__ __forceinline__ bool bf16_pair_bad(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// A thread's keys of a page are 2q, 2q + 1, 2q + 8, 2q + 9 (q = lane % 4).  Accumulator tile n holds
// columns 8n + 2q, 8n + 2q + 1.
template <int kRG, bool kMask>
__device__ __forceinline__ void rows_block16(const uint32_t (&page)[kBlockPages], uint32_t q,
                                             RowsState<kRG>& st, const float (&c)[kRG][2],
                                             const uint32_t (&vis)[kRG][2], int lane) {
  const int mi = lane >> 3, t8 = lane & 7, q2 = 2 * (lane & 3);
  float s[kRG][2 * kBlockPages][4];
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int t = 0; t < 2 * kBlockPages; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[g][t][i] = 0.f;
    }
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t qa[kRG][4];
#pragma unroll
    for (int g = 0; g < kRG; ++g)
      ldsm_x4(q + g * (16 * kHeadDim * 2) + (((2 * ks + (mi >> 1)) ^ t8) << 4), qa[g][0], qa[g][1],
              qa[g][2], qa[g][3]);
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      uint32_t b0, b1, b2, b3;
      ldsm_x4(page[t] + swz_off(t8 + (mi >> 1) * 8, ks * 16 + (mi & 1) * 8, 16), b0, b1, b2, b3);
#pragma unroll
      for (int g = 0; g < kRG; ++g) {
        mma_bf16(s[g][2 * t], qa[g], b0, b1);
        mma_bf16(s[g][2 * t + 1], qa[g], b2, b3);
      }
    }
  }
  uint32_t any = 0;
  if constexpr (kMask) {
    any = seen_by_any<kRG>(vis) >> q2;
#pragma unroll
    for (int g = 0; g < kRG; ++g) mask_block<8>(s[g], vis[g], q2);
  }
  float mx[kRG][2];
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    block_max(s[g], mx[g]);
    mx[g][0] *= c[g][0];
    mx[g][1] *= c[g][1];
  }
  const uint32_t none[kBlockPages] = {};
  raise<false, kRG>(st, mx, none);
#pragma unroll
  for (int g = 0; g < kRG; ++g) block_exp(s[g], c[g], st.m[g], st.l[g]);
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    // p is rounded to bf16 for the product (half a step of 2^-8), as in kernels B and D.
    uint32_t pa[kRG][4];
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      const float(&p0)[4] = s[g][2 * t];
      const float(&p1)[4] = s[g][2 * t + 1];
      pa[g][0] = pack_bf16(p0[0], p0[1]);
      pa[g][1] = pack_bf16(p0[2], p0[3]);
      pa[g][2] = pack_bf16(p1[0], p1[1]);
      pa[g][3] = pack_bf16(p1[2], p1[3]);
    }
    const uint32_t a = any >> (16 * t);
    const uint32_t keep0 = (a & 1u ? 0xffffu : 0u) | (a & 2u ? 0xffff0000u : 0u);
    const uint32_t keep1 = (a & 0x100u ? 0xffffu : 0u) | (a & 0x200u ? 0xffff0000u : 0u);
    const int key = t8 + (mi & 1) * 8;
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
          b[i] &= (i & 1) ? keep1 : keep0;
          if (bf16_pair_bad(b[i])) {
            bad = true;
            if ((b[i] & 0x7f80u) == 0x7f80u) b[i] &= 0xffff0000u;
            if ((b[i] & 0x7f800000u) == 0x7f800000u) b[i] &= 0xffffu;
          }
        }
      }
#pragma unroll
      for (int g = 0; g < kRG; ++g) {
        mma_bf16(st.o[g][2 * np], pa[g], b[0], b[1]);
        mma_bf16(st.o[g][2 * np + 1], pa[g], b[2], b[3]);
      }
    }
    if constexpr (kMask) {
      if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const int src = (lane & ~3) | ((k & 7) >> 1);
#pragma unroll
          for (int g = 0; g < kRG; ++g) {
            const float(&p0)[4] = s[g][2 * t];
            const float(&p1)[4] = s[g][2 * t + 1];
            const float a0 = (k & 8) ? ((k & 1) ? p1[1] : p1[0]) : ((k & 1) ? p0[1] : p0[0]);
            const float a1 = (k & 8) ? ((k & 1) ? p1[3] : p1[2]) : ((k & 1) ? p0[3] : p0[2]);
            const float w0 = __shfl_sync(0xffffffffu, a0, src);
            const float w1 = __shfl_sync(0xffffffffu, a1, src);
            const bool see0 = vis[g][0] >> (16 * t + k) & 1u, see1 = vis[g][1] >> (16 * t + k) & 1u;
#pragma unroll
            for (int n = 0; n < 16; ++n) {
              const uint32_t w = lds32(vbase + swz_off(k, n * 8 + q2, 16));
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t bits = i == 0 ? w << 16 : w & 0xffff0000u;
                if ((bits & 0x7f800000u) != 0x7f800000u) continue;
                const float v = __uint_as_float(bits);
                if (see0) st.o[g][n][i] += w0 * v;
                if (see1) st.o[g][n][2 + i] += w1 * v;
              }
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

// The last CTA of a split tile merges the splits' partial rows: out = sum_s 2^(lse_s - M) O_s /
// sum_s 2^(lse_s - M), s in order, so the result does not depend on which CTA came last.  The
// partial rows come through shared memory (the idle ring, `bytes` of it) by asynchronous copies, as many
// splits at a time as fit, so that one latency covers them all (through registers the merge took 4-8
// us of a short call); the rows' M and sums are formed from global memory meanwhile.  A warp
// takes rows warp, warp + 4, ..., a lane four columns.
template <int kRows>
__device__ __forceinline__ void merge_splits(const AttnArgs& a, uint8_t* smem, int bytes, int row0,
                                             int n_splits, int rows, int kvh, int flat_tok) {
  constexpr int kT = kRowsWarps * 32, kPer = kRows / kRowsWarps, kLanes = kT / kRows;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* top = reinterpret_cast<float*>(smem);  // [kRows] M, then [kRows] 1 / sum
  float* lse_s = top + 2 * kRows;               // [splits of a chunk][rows], then their O rows
  const int chunk = max(1, min(n_splits, (bytes - 2 * kRows * 4) / (rows * (kHeadDim + 1) * 4 + 16)));
  float* o_s = lse_s + (chunk * rows + 3) / 4 * 4;
  auto at = [&](int s, int r) {
    return (static_cast<long long>(row0) + static_cast<long long>(s) * rows + r) * a.num_kv + kvh;
  };
  float4 acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n_splits; s0 += chunk) {
    const int cnt = min(chunk, n_splits - s0);
    if (s0 > 0) asm volatile("bar.sync 1, %0;" ::"r"(kT) : "memory");  // the last chunk was read
    for (int i = warp; i < cnt * rows; i += kRowsWarps) {
      const float* src = a.ws_o + at(s0, 0) * kHeadDim +
                         static_cast<long long>(i) * a.num_kv * kHeadDim + lane * 4;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       smem_u32(o_s + i * kHeadDim + lane * 4)),
                   "l"(src)
                   : "memory");
    }
    for (int i = tid; i < cnt * rows; i += kT) lse_s[i] = __ldcg(a.ws_lse + at(s0, 0) + static_cast<long long>(i) * a.num_kv);
    if (s0 == 0) {
      // kLanes neighbouring threads per row, over all splits.
      const int r = tid / kLanes;
      float m = -INFINITY, l = 0.f;
      if (r < rows) {
#pragma unroll 4
        for (int s = tid % kLanes; s < n_splits; s += kLanes) {
          const float x = __ldcg(a.ws_lse + at(s, r));
          if (x == -INFINITY) continue;
          const float mn = fmaxf(m, x);
          l = l * fast_exp2(m - mn) + fast_exp2(x - mn);  // a NaN stays in l
          m = mn;
        }
      }
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m, off);
        const float lo = __shfl_xor_sync(0xffffffffu, l, off);
        const float mn = fmaxf(m, mo);
        l = (m == -INFINITY ? l : l * fast_exp2(m - mn)) + (mo == -INFINITY ? lo : lo * fast_exp2(mo - mn));
        m = mn;
      }
      if (r < kRows && tid % kLanes == 0) {
        top[r] = m;
        top[kRows + r] = l != 0.f ? 1.f / l : 0.f;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"r"(kT) : "memory");
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int r = warp + k * kRowsWarps;
      if (r < rows) {
        const float m = top[r];
        for (int i = 0; i < cnt; ++i) {
          const float x = lse_s[i * rows + r];
          const float w = x == -INFINITY ? 0.f : fast_exp2(x - m);
          const float4 v = *reinterpret_cast<const float4*>(o_s + (i * rows + r) * kHeadDim + lane * 4);
          acc[k].x += w * v.x;
          acc[k].y += w * v.y;
          acc[k].z += w * v.z;
          acc[k].w += w * v.w;
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int r = warp + k * kRowsWarps;
    if (r >= rows) break;
    const float inv = top[kRows + r];
    __nv_bfloat16* dst = a.out + static_cast<long long>(flat_tok + (r >> 1)) * a.out_row_stride +
                         (kvh * kGroup + (r & 1)) * kHeadDim + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc[k].x * inv, acc[k].y * inv),
                                                pack_bf16(acc[k].z * inv, acc[k].w * inv));
  }
}

template <bool kKv8, bool kTree, int kRG>
__global__ void __launch_bounds__(RowsCfg<kKv8, kRG>::kThreads, RowsCfg<kKv8, kRG>::kCtasPerSm)
    rows_attn_kernel(const __grid_constant__ CUtensorMap kv_map, const RowsArgs ra) {
  using Cfg = RowsCfg<kKv8, kRG>;
  constexpr int kStages = Cfg::kStages, kBatch = Cfg::kBatch;
  const AttnArgs& a = ra.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem;
  uint8_t* qtile = smem + Cfg::kQOffset;
  float* qscale = reinterpret_cast<float*>(smem + Cfg::kScaleOffset);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kStages);
  volatile int* last_flag = abort_flag + 1;
  static_assert(2 * (kRG == 1 ? kRowsNarrowTokens : kRowsTokens) == Cfg::kRows, "rows of a tile");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int item_idx = blockIdx.x / a.num_kv;
  const int kvh = blockIdx.x - item_idx * a.num_kv;
  // The plan was copied in before the previous kernel started, so it is read before the wait.
  const int* it = a.items + static_cast<long long>(item_idx) * kRec;
  const int seq = it[0], tok0 = it[1], n_q = it[2], page_begin = it[3], part_row = it[5];
  const int merge_row = it[7] == 1 ? it[6] : -1;
  const int* sr = a.seqs + static_cast<long long>(seq) * kRec;
  const int flat_start = sr[0], num_cached = sr[2], table_off = sr[4];
  const int npages = it[4] - page_begin;
  if (part_row >= 0 && threadIdx.x == 0) {
    // What the end of a split needs: its combine record and arrival counter.
    asm volatile("prefetch.global.L2 [%0];" ::"l"(ra.combines + static_cast<long long>(it[6]) * kRec));
    asm volatile("prefetch.global.L2 [%0];" ::"l"(ra.arrived + static_cast<long long>(it[6]) * a.num_kv + kvh));
  }

  const int sets = n_q * kGroup > 16 * kRG ? 2 : 1;
  const int phases = kRowsWarps / sets;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], sets);  // one warp of each row set reads a page
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();

  if (warp >= kRowsWarps) {
    if constexpr (kRG == 2) setmaxnreg_dec<Cfg::kProducerRegs>();
    const int* table = a.tables + table_off + page_begin;
    int mine = lane < npages ? table[lane] : 0;
    pdl_wait();
    pdl_trigger();
    if (warp != kRowsWarps) return;
    // ---------------- producer warp ----------------
    // Lane i of the first kBatch takes the pages j with j % kBatch == i: the lanes wait for their
    // slots and issue their copies side by side.  (One lane issuing every page takes a chain of
    // several hundred cycles per page, which three CTAs of 4 KiB pages per SM cannot afford: 256
    // decode rows 287 us that way, 219 with four lanes.)
    const uint64_t policy = l2_policy_evict_first();
    int issued = 0;  // by this lane
    bool stop = false;
    for (int j0 = 0; j0 < npages && !stop; j0 += 32) {
      if (j0 > 0) mine = j0 + lane < npages ? table[j0 + lane] : 0;
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
  if constexpr (kRG == 2) setmaxnreg_inc<Cfg::kConsumerRegs>();
  pdl_wait();
  pdl_trigger();
  // Query rows to shared memory, half a warp per row: bf16 as they are; for an 8-bit pool scaled
  // into f16 and in the order of dims that rows_block8 wants.  Rows without a token are zeros.
  const uint32_t q_u32 = smem_u32(qtile);
  {
    const int l16 = lane & 15;
    constexpr int kPer = Cfg::kRows / (2 * kRowsWarps);
    uint4 x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = (i * kRowsWarps + warp) * 2 + (lane >> 4);
      x[i] = make_uint4(0u, 0u, 0u, 0u);
      if ((r >> 1) < n_q)
        x[i] = __ldg(reinterpret_cast<const uint4*>(
            a.q + static_cast<long long>(flat_start + tok0 + (r >> 1)) * a.q_row_stride +
            (kvh * kGroup + (r & 1)) * kHeadDim + l16 * 8));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = (i * kRowsWarps + warp) * 2 + (lane >> 4);
      const uint32_t row = q_u32 + r * (kHeadDim * 2);
      if constexpr (kKv8) {
        unsigned top = __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1)
          top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, off));
        const int b = exp_byte8(max(top & 0xffffu, top >> 16));
        const float inv = inv_scale8(b);
        // A row with a NaN or an infinity gets the scale NaN: it scores NaN.
        if (l16 == 0) qscale[r] = row_scale8(b);
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = pack_f16(bf16_lo(w[k]) * inv, bf16_hi(w[k]) * inv);
        // Dims 8 l .. + 7: words (0, 1), (4, 5) go to the chunk's first half, (2, 3), (6, 7) to
        // its second.
        const int chunk = l16 & ~1;
        const int off = (l16 & 1) * 8;
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(row + ((chunk ^ (r & 7)) << 4) + off),
                     "r"(h[0]), "r"(h[2])
                     : "memory");
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(row + (((chunk + 1) ^ (r & 7)) << 4) + off),
                     "r"(h[1]), "r"(h[3])
                     : "memory");
      } else {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((l16 ^ (r & 7)) << 4)),
                     "r"(x[i].x), "r"(x[i].y), "r"(x[i].z), "r"(x[i].w)
                     : "memory");
      }
    }
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
  }

  const int set = warp % sets, phase = warp / sets;
  const int row_base = set * 16 * kRG;  // of this warp's rows
  const bool warp_active = (row_base >> 1) < n_q;
  const int q2 = 2 * (lane & 3);
  // This thread's rows row(g, h) = row_base + 16 g + lane / 4 + 8 h and their facts.
  const int row00 = row_base + (lane >> 2);
  float c[kRG][2];
  bool live[kRG][2];
  int words = 0;
  const int* masks = nullptr;  // tree: mask rows of the sequence
  if constexpr (kTree) {
    words = sr[7];
    masks = ra.plan + sr[6];
  }
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row00 + 16 * g + 8 * h;
      c[g][h] = a.scale_log2;
      if constexpr (kKv8) c[g][h] *= qscale[r];
      live[g][h] = (r >> 1) < n_q;
      if constexpr (kTree) {
        // A token whose mask misses itself sees nothing.
        if (live[g][h]) {
          const int k = tok0 + (r >> 1);
          live[g][h] = masks[static_cast<long long>(k) * words + (k >> 5)] >> (k & 31) & 1;
        }
      }
    }
  }

  RowsState<kRG> st;
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int n = 0; n < 16; ++n)
      st.o[g][n][0] = st.o[g][n][1] = st.o[g][n][2] = st.o[g][n][3] = 0.f;
    st.m[g][0] = st.m[g][1] = -INFINITY;
    st.l[g][0] = st.l[g][1] = 0.f;
  }
  st.eb = -1000;
  st.inv_e = 0.f;
  st.hot = 0;
  // First key position that some row of the warp may not see.
  const int first_masked = kTree ? num_cached : num_cached + tok0 + (row_base >> 1) + 1;
  const uint32_t ring_u32 = smem_u32(ring);
  // This lane's ldmatrix row of the query tile.
  const uint32_t q_row = q_u32 + (row_base + (lane & 7) + ((lane >> 3) & 1) * 8) * (kHeadDim * 2);
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
      uint32_t vis[kRG][2];
      if (cnt < kBlockPages || key0 + kBlockPages * kBlockTokens > first_masked) {
#pragma unroll
        for (int g = 0; g < kRG; ++g) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = tok0 + ((row00 + 16 * g + 8 * h) >> 1);  // the row's new token
            uint32_t v = 0;
            if (live[g][h]) {
#pragma unroll
              for (int t = 0; t < kBlockPages; ++t) {
                const int k0 = key0 + t * kBlockTokens;
                uint32_t bits;
                if constexpr (kTree) {
                  bits = k0 + kBlockTokens <= num_cached
                             ? 0xffffu
                             : tree_bits(masks + static_cast<long long>(k) * words, words, k0 - num_cached);
                } else {
                  bits = causal_bits(num_cached + k, k0);
                }
                if (t < cnt) v |= bits << (16 * t);
              }
            }
            vis[g][h] = v;
          }
        }
        if constexpr (kKv8)
          rows_block8<kRG, true>(page, q_row, st, c, vis, lane);
        else
          rows_block16<kRG, true>(page, q_row, st, c, vis, lane);
      } else {
#pragma unroll
        for (int g = 0; g < kRG; ++g) vis[g][0] = vis[g][1] = 0xffffffffu;
        if constexpr (kKv8)
          rows_block8<kRG, false>(page, q_row, st, c, vis, lane);
        else
          rows_block16<kRG, false>(page, q_row, st, c, vis, lane);
      }
    }
    __syncwarp();
    if (lane < cnt) mbar_arrive(&empty[(j + lane) % kStages]);
  }

  const float fe = st.eb < 0 ? 0.f : scale8(st.eb);  // O back to the values the codes stand for
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st.l[g][h] += __shfl_xor_sync(0xffffffffu, st.l[g][h], 1);
      st.l[g][h] += __shfl_xor_sync(0xffffffffu, st.l[g][h], 2);
    }
    if constexpr (kKv8) {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[g][n][i] *= fe;
      }
    }
  }

  // Merge of the page phases, one row group at a time: every warp leaves its (O, m, l) in the idle
  // ring (each page has been read once all consumer warps reach the barrier; a copy that was
  // abandoned on a timeout is drained by the producer before the CTA ends), and each warp merges
  // and writes 16 / phases of its row set's column tiles.
  float4* scratch = reinterpret_cast<float4*>(ring);
  const int per = 16 / phases;
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
#pragma unroll
    for (int n = 0; n < 16; ++n)
      scratch[(warp * 17 + n) * 32 + lane] =
          make_float4(st.o[g][n][0], st.o[g][n][1], st.o[g][n][2], st.o[g][n][3]);
    scratch[(warp * 17 + 16) * 32 + lane] =
        make_float4(st.m[g][0], st.m[g][1], st.l[g][0], st.l[g][1]);
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
    float mx[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f}, wt[kRowsWarps][2];
#pragma unroll
    for (int p = 0; p < kRowsWarps; ++p) {
      if (p < phases) {
        const float4 ml = scratch[((p * sets + set) * 17 + 16) * 32 + lane];
        mx[0] = fmaxf(mx[0], ml.x);
        mx[1] = fmaxf(mx[1], ml.y);
      }
    }
#pragma unroll
    for (int p = 0; p < kRowsWarps; ++p) {
      wt[p][0] = wt[p][1] = 0.f;
      if (p < phases) {
        const float4 ml = scratch[((p * sets + set) * 17 + 16) * 32 + lane];
        wt[p][0] = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mx[0]);
        wt[p][1] = ml.y == -INFINITY ? 0.f : fast_exp2(ml.y - mx[1]);
        // A phase whose scores were all NaN never raised its maximum: its sum is kept as it is.
        if (ml.z != ml.z) wt[p][0] = 1.f;
        if (ml.w != ml.w) wt[p][1] = 1.f;
        L[0] += ml.z * wt[p][0];
        L[1] += ml.w * wt[p][1];
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row00 + 16 * g + 8 * h;
      const int tok = r >> 1;
      if (tok >= n_q) continue;
      const RowOut out = row_out(a, r, tok, live[g][h], mx[h], L[h], kvh, part_row, merge_row,
                                 flat_start + tok0, phase == 0 && q2 == 0);
      for (int n = phase * per; n < (phase + 1) * per; n += 2) {
        float x0[2] = {0.f, 0.f}, x1[2] = {0.f, 0.f};  // tiles n and n + 1
#pragma unroll
        for (int p = 0; p < kRowsWarps; ++p) {
          if (p < phases) {
            const float2* base = reinterpret_cast<const float2*>(
                scratch + ((p * sets + set) * 17 + n) * 32 + lane);
            const float2 y0 = base[h], y1 = base[64 + h];
            x0[0] += y0.x * wt[p][h];
            x0[1] += y0.y * wt[p][h];
            x1[0] += y1.x * wt[p][h];
            x1[1] += y1.y * wt[p][h];
          }
        }
        if constexpr (kKv8) {
          const float x[4] = {x0[0], x1[0], x0[1], x1[1]};
          put_cols<4>(out, 8 * n + 2 * q2, x, live[g][h]);
        } else {
          put_cols<2>(out, 8 * n + q2, x0, live[g][h]);
          put_cols<2>(out, 8 * n + 8 + q2, x1, live[g][h]);
        }
      }
    }
  }

  if (part_row >= 0) {
    // A split of a tile: the last one to arrive merges them all.
    __threadfence();
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
    const int* cr = ra.combines + static_cast<long long>(it[6]) * kRec;
    if (threadIdx.x == 0) {
      int* counter = ra.arrived + static_cast<long long>(it[6]) * a.num_kv + kvh;
      const bool last = atomicAdd(counter, 1) == cr[4] - 1;
      if (last) *counter = 0;  // ready for the next call
      *last_flag = last ? 1 : 0;
    }
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
    if (*last_flag) {
      __threadfence();
      merge_splits<Cfg::kRows>(a, ring, Cfg::kStageBytes, cr[3], cr[4], n_q * kGroup, kvh,
                               flat_start + tok0);
    }
  }
}

}  // namespace ms
