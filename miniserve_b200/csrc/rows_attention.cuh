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
// bf16 pool: mma.sync m16n8k16 with bf16 operands, as in kernel B.  As there, p reaches 2^8 before the
// maximum follows, so V rows beyond 2^119 may overflow where they are seen.
//
// 8-bit pool: mma.sync m16n8k16 with f16 operands.  e4m3 codes are f16 values, so they are converted
// exactly, two codes per instruction, after ldmatrix has brought them (16-bit units of two codes)
// to the lanes.  K: a lane's word is four neighbouring dims of one key; the query rows lie in shared
// memory in that order of dims, so two conversions give a B operand.  V: ldmatrix.trans
// leaves two neighbouring columns of two neighbouring tokens in a word; one byte permute and two
// conversions give the operands of two column tiles (even and odd columns).  The query row (bf16, 8
// significant bits) is scaled by a power of two into f16's range: exact down to 2^-25 of its
// largest value, and below that off by at most 2^-32 of it.  (mma.sync on e4m3 operands would need no conversion, but it runs at less than
// half the rate per product here: 256 decode rows took 431 us with K multiplied that way.)
// The row exponents of K multiply S's columns in fp32; those of V multiply p before it is rounded
// to f16, which keeps 11 bits of a product, three more than the bf16 form, as long as it lies between
// 2^-14 and 2^16.  So O needs a reference of its own.  While the V exponents that a warp meets lie within
// 10 of each other, it is the running maximum of the scores times one power of two, placed so that
// p 2^e is at most 2^15 and a row's largest at least 2.  A warp that meets others gives every row a power of
// two of its own from there on, from the largest s c + e over the keys that the row sees, which holds the
// row's largest product between 1 and 2^15 whatever the values are (see raise8).  Either way f16's range
// costs a key at most 2^-25 in units in which the row's largest p 2^e is at least 1.  (Scores are formed in
// fp32 from a query row scaled to at most 448: K rows beyond 2^100 may overflow there.)
//
// Why this shape.  A decode row needs its bytes and little else: up to 32 rows per CTA, three CTAs per SM
// at 128 registers (the query rows stay in shared memory and are read again for every pair of pages).
// Tiles of more than 16 tokens are bound by the conversions and the products, so a warp holds two row
// groups (kRG = 2) and uses each converted operand twice; that takes more than 168 registers, which
// two CTAs of two warpgroups have once the producer's warpgroup hands its share to the consumers.
//
// What it measures (cold L2, 8 KV heads unless said): 256 decode rows over 1.2 GB of 8-bit pages 196 to
// 219 us by GPU and by where the pool lies (0.94 to 0.85 of the copy rate), 64 trees of 16 drafts over 562 MB
// of bf16 pages 102 to 109 us (0.84 to 0.79), 3 rows over 100k tokens 50 to 52 us (0.62; 8 us of it merge
// 36 splits); the short forms, 8 decode rows or one tree of 8 drafts, 15 to 18 us, which is latency.  48
// trees of 32 drafts (wide tiles, 8-bit pages) 123 to 130 us (0.27): mma.sync keeps the tensor pipe 48 %
// busy, and two warps per scheduler at 232 registers do not cover their own latencies; another order of the
// products changes nothing.  Where V rows spread over 2^24 in size, so that rows have factors of their own
// and every pair of pages takes the masked loop: 256 decode rows 292 us (219 beside it), 3 rows 73 (50), 48
// trees 215 (130).
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
  // Combine records {seq, tok0, n_q, first partial row, partials per row, rows between them, CTAs of
  // this kernel that arrive} of tiles with several partials; an item names its record in field 6.
  const int* combines;
  unsigned* arrived;    // [record][KVH] splits that have finished: zero between calls
  // The kernel before this one belongs to the same call and lets this one start only once its own
  // predecessor has completed (every CTA of it waits before it triggers), and nothing before the merge
  // reads what it writes: the wait for it moves from the start to the merge, so this kernel's pages fill the SMs
  // that its longest CTAs leave idle.  Every CTA still waits, so that whoever waits for this kernel has
  // waited for that one too.
  int behind;
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
  // Merge scratch in the ring: per warp 16 rows of a row group, padded, and their (m, l).
  static_assert(kRowsWarps * 16 * (kHeadDim + 4 + 2) * 4 <= kStageBytes, "merge scratch reuses the ring");
  static constexpr int kRows = kRG == 1 ? 32 : 64;
  static constexpr int kQOffset = (kStageBytes + 127) / 128 * 128;
  static constexpr int kScaleOffset = kQOffset + kRows * kHeadDim * 2;  // the rows' query scales
  static constexpr int kFactorOffset = kScaleOffset + kRows * 4;  // 8-bit pool: the rows' factors, per warp
  static constexpr int kBarOffset = kFactorOffset + (kKv8 ? kRowsWarps * 16 * kRG * 4 : 0);
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
  // 8-bit pool: what p 2^e is multiplied by before it is rounded, for all rows of the warp, and the middle
  // of the V exponent bytes that this serves, in every byte (see raise8).
  float unit;
  uint32_t mid;
};

// Multiplies a row's O.
template <int kRG>
__device__ __forceinline__ void scale_o(RowsState<kRG>& st, int g, const float (&f)[2]) {
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    st.o[g][n][0] *= f[0];
    st.o[g][n][1] *= f[0];
    st.o[g][n][2] *= f[1];
    st.o[g][n][3] *= f[1];
  }
}

// 8-bit pool.  p 2^e is multiplied by a power of two, x = 2^-d, before it is rounded, so O stands for O 2^d.
// The rows of a warp share x (`unit`) while its V exponent bytes lie within kReach of a middle: p is at
// most 2^kSlack8 and 2^(e - d) between 2 and 2^(2 kReach + 1), so a product is at most 2^kTop8 and a
// row's largest at least 2.
constexpr float kSlack8 = 4.f;
constexpr int kReach = 5;
constexpr int kTop8 = 15;
static_assert(kSlack8 + 2 * kReach + 1 == kTop8, "largest product");
// Values of `mid` before the first V row that is not zero (unit 0), and once the bytes have spread.
constexpr uint32_t kUnset = 0, kSpread = 1;
constexpr int kLeastMid = kReach + 1;
// Beyond this 2^d a row's sums may leave fp32 (products below 2^15, codes below 2^9, up to 2^30 keys).
constexpr float kLargeBack = 9.223372036854775808e18f;  // 2^63
constexpr int kFirstProduct = 8;  // log2 of what a row's largest product is when its own d is set

// 2^k: 0 below fp32's normal range.
__device__ __forceinline__ float pow2i(int k) {
  return k < -126 ? 0.f : __int_as_float((min(k, 127) + kExpBias) << 23);
}

// Whether one of this thread's V exponent bytes (vw) lies further than kReach from the middle (a carry out
// of a byte above 133 only adds to what is found).
template <int kRG>
__device__ __forceinline__ bool bytes_out(const RowsState<kRG>& st, const uint32_t (&vw)[kBlockPages]) {
  constexpr uint32_t kOver = (127 - kReach) * 0x01010101u;
  const uint32_t far0 = __vabsdiffu4(vw[0], st.mid), far1 = __vabsdiffu4(vw[1], st.mid);
  return st.mid <= kSpread || ((far0 + kOver | far0 | far1 + kOver | far1) & 0x80808080u) != 0;
}
template <int kRG>
__device__ __forceinline__ bool max_up(const RowsState<kRG>& st, const float (&mx)[kRG][2], float slack) {
  bool up = false;
#pragma unroll
  for (int g = 0; g < kRG; ++g) up = up || mx[g][0] > st.m[g][0] + slack || mx[g][1] > st.m[g][1] + slack;
  return up;
}

// Sets the middle for a warp that has none, around the block's bytes (but zeros, which any middle serves) with
// room for 4 larger ones if there is.  False: they have spread already.
template <int kRG>
__device__ __forceinline__ bool set_mid(RowsState<kRG>& st, const uint32_t (&vw)[kBlockPages]) {
  int top = 0, bottom = 255;
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = static_cast<int>(vw[t] >> (8 * i) & 255u);
      top = max(top, b);
      if (b != 0) bottom = min(bottom, b);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  bottom = __reduce_min_sync(0xffffffffu, bottom);
  if (st.mid != kUnset || top == static_cast<int>(kExpNan) || top - bottom > 2 * kReach) return false;
  if (top > 0) {
    const int mid = max(top + min(4, 2 * kReach - (top - bottom)) - kReach, kLeastMid);
    st.mid = static_cast<uint32_t>(mid) * 0x01010101u;
    st.unit = pow2i(kExpBias + kReach + 1 - mid);
  }
  return true;
}

// Brings the running maxima up to a block (mx, in exp2 units) where it exceeds them by `slack`; O and l
// follow.
template <int kRG>
__device__ __forceinline__ void raise(RowsState<kRG>& st, const float (&mx)[kRG][2], float slack) {
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    float al[2] = {1.f, 1.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (mx[g][h] > st.m[g][h] + slack) {
        al[h] = fast_exp2(st.m[g][h] - mx[g][h]);
        st.m[g][h] = mx[g][h];
      }
      st.l[g][h] *= al[h];
    }
    scale_o(st, g, al);
  }
}

// The same for a block of an 8-bit pool in the form that serves any bytes: s its scores (invisible keys
// -infinity), vw this thread's V exponent words, x this thread's first row among its warp's factors in
// shared memory (all lanes of a quad hold, read and write the same; 0 until a row has one).
//
// Once the bytes have spread, every row has a d of its own.  It grows where the block's largest
// s c - m + e over the keys that the row sees exceeds d + 15, to 8 below it; when m is raised by y, it
// falls by y rounded up and O keeps its size.  So products stay below 2^15, and a row's largest at least 1.
// d is whole: values that are held with another exponent, or beside other rows, round alike.  Zero rows
// (byte 0) and NaN rows (255) are left out: the one adds nothing, the other is NaN at any d.
template <int kRG>
__device__ __forceinline__ void raise8(RowsState<kRG>& st, const float (&s)[kRG][2 * kBlockPages][4],
                                       const float (&c)[kRG][2], const float (&mx)[kRG][2],
                                       const uint32_t (&vw)[kBlockPages], float* x, int lane) {
  // Zero bytes, those of scrubbed rows among them, are inside.
  const uint32_t in[kBlockPages] = {vw[0] | (__vcmpeq4(vw[0], 0u) & st.mid),
                                    vw[1] | (__vcmpeq4(vw[1], 0u) & st.mid)};
  const bool out = bytes_out(st, in);
  if (!__any_sync(0xffffffffu, out || max_up(st, mx, kSlack8))) return;
  if (st.mid != kSpread && __any_sync(0xffffffffu, out) && !set_mid(st, vw)) {
    st.mid = kSpread;
#pragma unroll
    for (int g = 0; g < kRG; ++g) x[16 * g] = x[16 * g + 8] = st.unit;
  }
  if (st.mid != kSpread) {
    raise(st, mx, kSlack8);
    return;
  }
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    float al[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float by = mx[g][h] - st.m[g][h];
      const float old = x[16 * g + 8 * h];
      int d = kExpBias - (__float_as_int(old) >> 23);
      al[h] = 1.f;
      if (by > kSlack8) {
        st.m[g][h] = mx[g][h];
        st.l[g][h] *= fast_exp2(-by);
        const int y = min(static_cast<int>(ceilf(fminf(by, 500.f))), d + 126);
        al[h] = fast_exp2(static_cast<float>(y) - by);
        d -= y;
      }
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b = vw[t] >> (8 * i) & 255u;
          // b - 127 as a float: b in the low bits of 2^23.
          const float e = b - 1u < kExpNan - 1u ? __uint_as_float(0x4b000000u | b) - (8388608.f + kExpBias)
                                                : -INFINITY;
          top = fmaxf(top, __fmaf_rn(s[g][2 * t + (i >> 1)][2 * h + (i & 1)], c[g][h], e));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top -= st.m[g][h];
      if (old == 0.f ? top > -INFINITY : top > static_cast<float>(d + kTop8)) {
        const int grown = static_cast<int>(ceilf(fminf(top, 200.f))) - kFirstProduct;
        al[h] = old == 0.f ? 1.f : al[h] * pow2i(d - grown);
        d = grown;
        x[16 * g + 8 * h] = pow2i(-d);
      } else if (old != 0.f) {
        x[16 * g + 8 * h] = pow2i(-d);
      }
    }
    scale_o(st, g, al);
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

// A thread's keys of a page are key0, key0 + 1, key0 + kNext, key0 + kNext + 1.  Whether row (g, h) sees
// key i (0..3) of page t; vis[g][h]: bit 16 t + k for key k.
template <int kNext>
__device__ __forceinline__ bool sees(uint32_t vis, int t, int key0, int i) {
  return vis >> (16 * t + key0 + (i >> 1) * kNext + (i & 1)) & 1u;
}

// Scores a row does not see become -infinity.
template <int kNext>
__device__ __forceinline__ void mask_block(float (&s)[2 * kBlockPages][4], const uint32_t (&vis)[2],
                                           int key0) {
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!sees<kNext>(vis[h], t, key0, i)) s[2 * t + (i >> 1)][2 * h + (i & 1)] = -INFINITY;
    }
  }
}

// Rows of keys that no row of the tile sees (behind a sequence's end, unused drafts) may hold anything,
// and 0 times NaN is NaN: their V rows (`dead`: bit k) become zeros in shared memory.  Each warp that
// reads the page does it for itself, with the same result.  row_bytes of V rows start at v;
// the 8-bit pool's exponent bytes at `exps` (0: none) go too.
__device__ __forceinline__ void scrub_keys(uint32_t dead, uint32_t v, bool kv8, uint32_t exps,
                                           bool refilled, int lane) {
  // Two lanes per key: half of its 128 (8-bit) or 256 bytes each (a bf16 row lies in two halves).
  const int k = lane >> 1, h = lane & 1;
  if (dead >> k & 1u) {
    const uint32_t row = kv8 ? v + k * kRow8Bytes + h * 64 : v + h * (kBlockTokens * 128) + k * 128;
    for (int i = 0; i < (kv8 ? 64 : 128); i += 16)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + i), "r"(0) : "memory");
    if (kv8 && h == 0) asm volatile("st.shared.u8 [%0], %1;" ::"r"(exps + k), "r"(0) : "memory");
  }
  // A later copy into the slot goes through the async proxy.
  if (refilled) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// ---- two pages, 8-bit pool ----------------------------------------------------------------------

// q: shared address of this lane's ldmatrix row of the warp's first row group (f16, the dims of a
// 16-dim chunk in the order 0 1 4 5 8 9 12 13 2 3 6 7 10 11 14 15, so that a lane's fragment is the dims
// 4 (lane % 4) .. + 3 that its word of codes holds).  c: scale log2(e) times the rows' query scale.
// Key column j of tile t (of two per page) is token 4 (j / 2) + j % 2 + 2 t, so a thread's four
// keys of a page are neighbours (4 (lane % 4) .. + 3) and their exponent bytes one word.  Accumulator
// tile 2u + p holds columns 16u + 2j + p, so a thread's o[2u][0], o[2u + 1][0], o[2u][1],
// o[2u + 1][1] are four neighbouring columns.
// The unmasked form serves the common unit only: it returns false, with nothing done, for a block whose V
// exponents leave it.
template <int kRG, bool kMask>
__device__ __forceinline__ bool rows_block8(const uint32_t (&page)[kBlockPages], uint32_t q,
                                            RowsState<kRG>& st, const float (&c)[kRG][2],
                                            const uint32_t (&vis)[kRG][2], float* x_rows, int lane) {
  const int mi = lane >> 3, t8 = lane & 7, q4 = 4 * (lane & 3);
  const int tok = 4 * (t8 >> 1) + (t8 & 1);  // this lane's ldmatrix row in tile 0
  const int sw = code_swizzle8(tok);         // the same for tok + 2
  // Unmasked pairs lie side by side in the ring: the second page is an offset in the load.
  auto at_page = [&](uint32_t addr, int t) {
    return t == 0 ? addr : addr + (kMask ? page[1] - page[0] : static_cast<uint32_t>(kPage8Bytes));
  };
  const uint32_t k_row = page[0] + (tok + 2 * (mi >> 1)) * kRow8Bytes;
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
        ldsm_x4((q + (((2 * (2 * u + i) + (mi >> 1)) ^ t8) << 4)) + g * (16 * kHeadDim * 2),
                qa[g][i][0], qa[g][i][1], qa[g][i][2], qa[g][i][3]);
    }
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      // Both key tiles of the page, chunks 2u and 2u + 1.
      uint32_t b[4];
      ldsm_x4(at_page(k_row + (((2 * u + (mi & 1)) ^ sw) << 4), t), b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b0 = e4m3x2_to_f16x2<0>(b[i]), b1 = e4m3x2_to_f16x2<1>(b[i]);
#pragma unroll
        for (int g = 0; g < kRG; ++g) mma_f16(s[g][2 * t + (i >> 1)], qa[g][i & 1], b0, b1);
      }
    }
  }
  uint32_t vw[kBlockPages];
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    const uint32_t kw = lds32(at_page(page[0] + kExp8Off + q4, t));
    vw[t] = lds32(at_page(page[0] + kExp8Off + kBlockTokens + q4, t));
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
  if constexpr (kMask) {
    raise8(st, s, c, mx, vw, x_rows, lane);
  } else {
    const bool out = bytes_out(st, vw);
    if (__any_sync(0xffffffffu, out || max_up(st, mx, kSlack8))) {
      if (__any_sync(0xffffffffu, out) && !set_mid(st, vw)) return false;
      raise(st, mx, kSlack8);
    }
  }
#pragma unroll
  for (int g = 0; g < kRG; ++g) block_exp(s[g], c[g], st.m[g], st.l[g]);
  // p times the scale of its V row and the row's factor.  A NaN row's scale is infinite, and infinity
  // times its zero codes NaN; what a row does not see is 0 whatever the scale.
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
    const float unit = kMask ? 1.f : st.unit;
    const float f[4] = {scale_of_byte<0>(vw[t]) * unit, scale_of_byte<1>(vw[t]) * unit,
                        scale_of_byte<2>(vw[t]) * unit, scale_of_byte<3>(vw[t]) * unit};
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
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = st.mid == kSpread ? x_rows[16 * g + 8 * h] : st.unit;
#pragma unroll
        for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& w = s[g][2 * t + (i >> 1)][2 * h + (i & 1)];
            w = sees<2>(vis[g][h], t, q4, i) ? w * x : 0.f;
          }
        }
      }
    }
  }
  uint32_t pa[kRG][kBlockPages][4];
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t) {
      pa[g][t][0] = pack_f16(s[g][2 * t][0], s[g][2 * t][1]);
      pa[g][t][1] = pack_f16(s[g][2 * t][2], s[g][2 * t][3]);
      pa[g][t][2] = pack_f16(s[g][2 * t + 1][0], s[g][2 * t + 1][1]);
      pa[g][t][3] = pack_f16(s[g][2 * t + 1][2], s[g][2 * t + 1][3]);
    }
  }
  const uint32_t v_row = page[0] + kCodes8Bytes + (tok + 2 * (mi & 1)) * kRow8Bytes;
#pragma unroll
  for (int t = 0; t < kBlockPages; ++t) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t w[4];
      ldsm_x4_t(at_page(v_row + (((2 * u + (mi >> 1)) ^ sw) << 4), t), w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t a = w[2 * h], b = w[2 * h + 1];
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
  return true;
}

// ---- two pages, bf16 pool -----------------------------------------------------------------------

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
  if constexpr (kMask) {
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
  if (__any_sync(0xffffffffu, max_up(st, mx, 8.f))) raise(st, mx, 8.f);
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
#pragma unroll
    for (int np = 0; np < 8; ++np) {
      uint32_t b[4];
      ldsm_x4_t(page[t] + kPageBytes + swz_off(t8 + (mi & 1) * 8, np * 16 + (mi >> 1) * 8, 16), b[0],
                b[1], b[2], b[3]);
#pragma unroll
      for (int g = 0; g < kRG; ++g) {
        mma_bf16(st.o[g][2 * np], pa[g], b[0], b[1]);
        mma_bf16(st.o[g][2 * np + 1], pa[g], b[2], b[3]);
      }
    }
  }
}

// Whether a page's V rows hold an infinity or a NaN (all 32 lanes; a page with masked keys only).
__device__ __forceinline__ bool page_has_special16(uint32_t page, int lane) {
  bool bad = false;
#pragma unroll 1
  for (int i = 0; i < kPageBytes / (32 * 16); ++i) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(page + kPageBytes + (i * 32 + lane) * 16));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      bad = bad || (w[k] & 0x7f80u) == 0x7f80u || (w[k] & 0x7f800000u) == 0x7f800000u;
  }
  return __any_sync(0xffffffffu, bad);
}

// A page whose V rows hold an infinity or a NaN that only some rows see: a product with 0 would bring
// it to the others, so the page is attended key by key in fp32, each row with the keys it sees.
template <int kRG>
__device__ __forceinline__ void rows_page16_special(uint32_t page, int t, uint32_t q_tile,
                                                    int row00, RowsState<kRG>& st,
                                                    const float (&c)[kRG][2],
                                                    const uint32_t (&vis)[kRG][2], int lane) {
  const int q = lane & 3;
#pragma unroll 1
  for (int k = 0; k < kBlockTokens; ++k) {
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row00 + 16 * g + 8 * h;
        float s = 0.f;  // a quarter of the dims per lane of the quad
#pragma unroll 1
        for (int d = 32 * q; d < 32 * q + 32; d += 2) {
          const uint32_t a = lds32(q_tile + r * (kHeadDim * 2) + (((d >> 3) ^ (r & 7)) << 4) + (d & 7) * 2);
          const uint32_t b = lds32(page + swz_off(k, d, 16));
          s += bf16_lo(a) * bf16_lo(b) + bf16_hi(a) * bf16_hi(b);
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s *= c[g][h];
        const bool see = vis[g][h] >> (16 * t + k) & 1u;
        float al = 1.f;
        if (see && s > st.m[g][h]) {
          al = fast_exp2(st.m[g][h] - s);
          st.m[g][h] = s;
        }
        const float p = see ? fast_exp2(s - (st.m[g][h] == -INFINITY ? 0.f : st.m[g][h])) : 0.f;
        st.l[g][h] = st.l[g][h] * al + (q == 0 ? p : 0.f);
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const uint32_t w = lds32(page + kPageBytes + swz_off(k, n * 8 + 2 * q, 16));
          st.o[g][n][2 * h] = st.o[g][n][2 * h] * al + (see ? p * bf16_lo(w) : 0.f);
          st.o[g][n][2 * h + 1] = st.o[g][n][2 * h + 1] * al + (see ? p * bf16_hi(w) : 0.f);
        }
      }
    }
  }
}

// ---- the kernel ---------------------------------------------------------------------------------

// Rows of a split tile from their M and 1 / sum in `top`: warp w takes rows w, w + 4, ..., kR at a time, a
// lane four columns; the partial rows of kS splits are fetched at once, their weights with them (lane
// kS h + i forms that of split i of row h).
template <int kR, int kS>
__device__ __forceinline__ void merge_rows(const AttnArgs& a, const float* top, int row0,
                                           int n_splits, int stride, int rows, int kvh, int flat_tok,
                                           const int* masks, int words, int tok0) {
  static_assert(kR * kS <= 32 && (kS & (kS - 1)) == 0 && (kR & (kR - 1)) == 0, "a lane per weight");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long split_rows = static_cast<long long>(stride) * a.num_kv;
  const long long row_step = static_cast<long long>(kRowsWarps) * a.num_kv;
  const int wh = lane / kS & (kR - 1), wi = lane & (kS - 1);
#pragma unroll 1
  for (int r0 = warp; r0 < rows; r0 += kR * kRowsWarps) {
    const int n_r = min(kR, (rows - r0 + kRowsWarps - 1) / kRowsWarps);
    const long long first = static_cast<long long>(row0 + r0) * a.num_kv + kvh;
    const float* o = a.ws_o + first * kHeadDim + lane * 4;
    const int my_h = min(wh, n_r - 1);
    const float* lse = a.ws_lse + first + my_h * row_step;
    const float m = top[r0 + my_h * kRowsWarps], inv = top[rows + r0 + my_h * kRowsWarps];
    float4 acc[kR] = {};
#pragma unroll 1
    for (int s = 0; s < n_splits; s += kS) {
      float4 x[kR][kS];
      const float w_lse = s + wi < n_splits ? __ldcg(lse + (s + wi) * split_rows) : -INFINITY;
#pragma unroll
      for (int i = 0; i < kS; ++i) {
#pragma unroll
        for (int h = 0; h < kR; ++h) {
          x[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s + i < n_splits && h < n_r)
            x[h][i] = __ldcg(reinterpret_cast<const float4*>(
                o + ((s + i) * split_rows + h * row_step) * kHeadDim));
        }
      }
      const float w = (w_lse == -INFINITY ? 0.f : fast_exp2(w_lse - m)) * inv;
#pragma unroll
      for (int i = 0; i < kS; ++i) {
#pragma unroll
        for (int h = 0; h < kR; ++h) {
          const float u = __shfl_sync(0xffffffffu, w, kS * h + i);
          acc[h].x += u * x[h][i].x;
          acc[h].y += u * x[h][i].y;
          acc[h].z += u * x[h][i].z;
          acc[h].w += u * x[h][i].w;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kR; ++h) {
      if (h >= n_r) break;
      const int r = r0 + h * kRowsWarps, tok = tok0 + (r >> 1);
      const bool live = masks == nullptr ||
                        (masks[static_cast<long long>(r >> 1) * words + (tok >> 5)] >> (tok & 31) & 1);
      __nv_bfloat16* dst = a.out + static_cast<long long>(flat_tok + (r >> 1)) * a.out_row_stride +
                           (kvh * kGroup + (r & 1)) * kHeadDim + lane * 4;
      *reinterpret_cast<uint2*>(dst) =
          live ? make_uint2(pack_bf16(acc[h].x, acc[h].y), pack_bf16(acc[h].z, acc[h].w))
               : make_uint2(0u, 0u);
    }
  }
}

// The last CTA of a split tile merges the splits' partial rows: out = sum_s (2^(lse_s - M) /
// sum_t 2^(lse_t - M)) O_s, s in order, so the result does not depend on which CTA came last.  It runs alone
// and is bound by latencies, so it has few of them: L neighbouring threads per row form its M and sum,
// then the rows are merged with 16 loads in flight per lane (3 rows over 100k tokens in 36 splits: 51 us;
// 57 with the partial rows copied to shared memory first), spread over the splits where there are many,
// else over the rows (48 trees of 32 drafts: 131 us, 135 with two rows at a time).  Every load
// goes past L1, whose lines may be older than the other CTAs' rows.  masks: the tile's first mask row of
// a tree (a draft that sees nothing writes zeros: the tensor-core kernel does not know it), else null.
// top: 2 x rows floats.
__device__ __forceinline__ void merge_splits(const AttnArgs& a, float* top, int row0, int n_splits,
                                             int stride, int rows, int kvh, int flat_tok,
                                             const int* masks, int words, int tok0) {
  const int tid = threadIdx.x;
  const long long split_rows = static_cast<long long>(stride) * a.num_kv;
  {
    const int log_l = min(5, 7 - (32 - __clz(rows - 1)));  // 128 threads over the rows, L <= 32
    const int r = tid >> log_l, l_step = 1 << log_l;
    const float* lse = a.ws_lse + static_cast<long long>(row0 + r) * a.num_kv + kvh;
    float m = -INFINITY, l = 0.f;
    if (r < rows) {
#pragma unroll 4
      for (int s = tid & (l_step - 1); s < n_splits; s += l_step) {
        const float x = __ldcg(lse + s * split_rows);
        if (x == -INFINITY) continue;
        const float mn = fmaxf(m, x);
        l = l * fast_exp2(m - mn) + fast_exp2(x - mn);  // a NaN stays in l
        m = mn;
      }
    }
    for (int off = 1; off < l_step; off <<= 1) {
      const float mo = __shfl_xor_sync(0xffffffffu, m, off);
      const float lo = __shfl_xor_sync(0xffffffffu, l, off);
      const float mn = fmaxf(m, mo);
      l = (m == -INFINITY ? l : l * fast_exp2(m - mn)) + (mo == -INFINITY ? lo : lo * fast_exp2(mo - mn));
      m = mn;
    }
    if (r < rows && (tid & (l_step - 1)) == 0) {
      top[r] = m;
      top[rows + r] = l != 0.f ? 1.f / l : 0.f;  // a NaN sum stays NaN
    }
  }
  asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
  if (n_splits <= 4)
    merge_rows<4, 4>(a, top, row0, n_splits, stride, rows, kvh, flat_tok, masks, words, tok0);
  else
    merge_rows<2, 8>(a, top, row0, n_splits, stride, rows, kvh, flat_tok, masks, words, tok0);
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

  // Row sets of 16 kRG rows; each holds at least one token (two only where the rows exceed one).
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
    if (!ra.behind) pdl_wait();
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
  if (!ra.behind) pdl_wait();
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
        x[i] = __ldcg(reinterpret_cast<const uint4*>(
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
  const int q2 = 2 * (lane & 3);
  // This thread's rows row(g, h) = row_base + 16 g + lane / 4 + 8 h and their facts.
  const int row00 = row_base + (lane >> 2);
  float c[kRG][2];
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
      c[g][h] = a.scale_log2;
      if constexpr (kKv8) c[g][h] *= qscale[row00 + 16 * g + 8 * h];
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
  st.unit = 0.f;
  st.mid = kUnset;
  // This thread's first row among its warp's factors (see raise8).
  float* const x_rows = reinterpret_cast<float*>(smem + Cfg::kFactorOffset) + warp * 16 * kRG + (lane >> 2);
  // First key position that some row of the warp may not see.
  const int first_masked = kTree ? num_cached : num_cached + tok0 + (row_base >> 1) + 1;
  const uint32_t ring_u32 = smem_u32(ring);
  // This lane's ldmatrix row of the query tile.
  const uint32_t q_row = q_u32 + (row_base + (lane & 7) + ((lane >> 3) & 1) * 8) * (kHeadDim * 2);
  // Waits for the pages j .. j + cnt - 1 (cnt warp-uniform).  The warp leaves its loop only as a whole: the
  // tensor-core operations are warp-collective.
  auto wait_pages = [&](int j, int cnt) -> bool {
    bool ok = true;
#pragma unroll
    for (int t = 0; t < kBlockPages; ++t)
      if (t < cnt)
        ok = ok && mbar_wait_fast(&full[(j + t) % kStages], ((j + t) / kStages) & 1, abort_flag);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0) {
      atomicOr(&g_status_word, kErrTimeout);
      *abort_flag = 1;
    }
    return false;
  };
  // Whole pairs whose keys every row sees, then the rest (the end of the tile's pages, and in an 8-bit pool
  // everything from a pair on whose V exponents spread), with masks: what only the rest needs is kept out
  // of the registers of the first loop.
  const int n_full = min(npages & ~(kBlockPages - 1),
                         max(0, first_masked - page_begin * kBlockTokens) / (kBlockPages * kBlockTokens) * kBlockPages);
  int j = phase * kBlockPages;
  bool ok = true;
  for (; j < n_full; j += phases * kBlockPages) {
    if (!(ok = wait_pages(j, kBlockPages))) break;
    const uint32_t page[kBlockPages] = {ring_u32 + (j % kStages) * Cfg::kPage,
                                        ring_u32 + (j % kStages + 1) * Cfg::kPage};
    const uint32_t vis[kRG][2] = {};
    if constexpr (kKv8) {
      if (!rows_block8<kRG, false>(page, q_row, st, c, vis, x_rows, lane)) break;
    } else {
      rows_block16<kRG, false>(page, q_row, st, c, vis, lane);
    }
    __syncwarp();
    if (lane < kBlockPages) mbar_arrive(&empty[(j + lane) % kStages]);
  }
  for (; ok && j < npages; j += phases * kBlockPages) {
    const int cnt = min(kBlockPages, npages - j);
    if (!(ok = wait_pages(j, cnt))) break;
    // A second page that is not there is the first one again, with every key masked.
    uint32_t page[kBlockPages] = {ring_u32 + (j % kStages) * Cfg::kPage,
                                  ring_u32 + ((j + cnt - 1) % kStages) * Cfg::kPage};
    // The plan's records again (volatile loads: nothing of them lives through the loop above).
    auto reload = [](const int* p) {
      int v;
      asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
      return v;
    };
    const int* itm = a.items + static_cast<long long>(item_idx) * kRec;
    const int t0 = reload(itm + 1), nq = reload(itm + 2);
    const int* rec = a.seqs + static_cast<long long>(reload(itm)) * kRec;
    const int cached = reload(rec + 2);
    const int* mrows = nullptr;
    int mwords = 0;
    if constexpr (kTree) {
      mwords = reload(rec + 7);
      mrows = ra.plan + reload(rec + 6);
    }
    const int key0 = (reload(itm + 3) + j) * kBlockTokens;
    // Which of the pages' keys token k of the sequence's new ones sees.
    auto seen = [&](int k) {
      uint32_t v = 0;
#pragma unroll
      for (int t = 0; t < kBlockPages; ++t) {
        const int k0 = key0 + t * kBlockTokens;
        uint32_t bits;
        if constexpr (kTree) {
          const int* row = mrows + static_cast<long long>(k) * mwords;
          bits = 0u;
          if (row[k >> 5] >> (k & 31) & 1)
            bits = k0 + kBlockTokens <= cached ? 0xffffu : tree_bits(row, mwords, k0 - cached);
        } else {
          bits = causal_bits(cached + k, k0);
        }
        if (t < cnt) v |= bits << (16 * t);
      }
      return v;
    };
    // A lane per token of the tile (at most 32), handed to the rows; and all of them together.
    const uint32_t mine = lane < nq ? seen(t0 + lane) : 0u;
    const uint32_t any = __reduce_or_sync(0xffffffffu, mine);
    uint32_t vis[kRG][2];
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = (row00 + 16 * g + 8 * h) >> 1;  // rows past the last token see nothing
        vis[g][h] = __shfl_sync(0xffffffffu, mine, tok & 31);
      }
    }
#pragma unroll 1
    for (int t = 0; t < cnt; ++t) {
      const uint32_t dead = ~(any >> (16 * t)) & 0xffffu;
      if (dead != 0)
        scrub_keys(dead, page[t] + Cfg::kPage / 2 - (kKv8 ? kBlockTokens : 0), kKv8,
                   kKv8 ? page[t] + kExp8Off + kBlockTokens : 0u, j + t + kStages < npages, lane);
    }
    bool run = true;
    if constexpr (!kKv8) {
      bool special[kBlockPages];
#pragma unroll
      for (int t = 0; t < kBlockPages; ++t)
        special[t] = t < cnt && page_has_special16(page[t], lane);
      if (special[0] || special[1]) {
#pragma unroll 1
        for (int t = 0; t < kBlockPages; ++t)
          if (t == 0 ? special[0] : special[1])
            rows_page16_special<kRG>(page[t], t, q_u32, row00, st, c, vis, lane);
        // The other page, if it has none, goes the usual way, in both places.
        const uint32_t keep_bits = (special[0] ? 0u : 0xffffu) | (special[1] ? 0u : 0xffff0000u);
        run = keep_bits != 0u && !(special[0] && cnt < kBlockPages);
        if (special[0]) page[0] = page[1];
        if (special[1]) page[1] = page[0];
#pragma unroll
        for (int g = 0; g < kRG; ++g) {
          vis[g][0] &= keep_bits;
          vis[g][1] &= keep_bits;
        }
      }
    }
    if (run) {
      if constexpr (kKv8)
        rows_block8<kRG, true>(page, q_row, st, c, vis, x_rows, lane);
      else
        rows_block16<kRG, true>(page, q_row, st, c, vis, lane);
    }
    __syncwarp();
    if (lane < cnt) mbar_arrive(&empty[(j + lane) % kStages]);
  }

#pragma unroll
  for (int g = 0; g < kRG; ++g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st.l[g][h] += __shfl_xor_sync(0xffffffffu, st.l[g][h], 1);
      st.l[g][h] += __shfl_xor_sync(0xffffffffu, st.l[g][h], 2);
    }
    if constexpr (kKv8) {  // O back to the values the codes stand for
      float back[2];
      bool large = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = st.mid == kSpread ? x_rows[16 * g + 8 * h] : st.unit;
        back[h] = x == 0.f ? 0.f : __int_as_float((2 * kExpBias << 23) - __float_as_int(x));
        large = large || back[h] > kLargeBack;
      }
      if (__any_sync(0xffffffffu, large)) {
        // Rows near the end of the range have finite means, but no finite sums: a quarter of their mean
        // (four of them are added), with the weight in m.
        float inv[2] = {1.f, 1.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(back[h] > kLargeBack && st.l[g][h] > 0.f)) continue;
          inv[h] = 0.25f / st.l[g][h];
          st.m[g][h] += __log2f(4.f * st.l[g][h]);
          st.l[g][h] = 0.25f;
        }
        scale_o(st, g, inv);
      }
      scale_o(st, g, back);
    }
  }

  // Merge of the page phases, one row group at a time: every warp leaves its (O, m, l) in the idle
  // ring (each page has been read once all consumer warps reach the barrier; a copy that was
  // abandoned on a timeout is drained by the producer before the CTA ends), rows of 128 columns, and
  // the threads share the rows out in chunks of 8 columns.  Loops, not unrolled: this runs once, and
  // a longer form costs more in instruction fetches than it saves.
  constexpr int kPitch = kHeadDim + 4;
  float* so = reinterpret_cast<float*>(ring);                     // [warp][16 rows][kPitch]
  float* sm = so + kRowsWarps * 16 * kPitch;                      // [warp][16 rows] m, then l
  float* sl = sm + kRowsWarps * 16;
#pragma unroll
  for (int g = 0; g < kRG; ++g) {
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (lane >> 2) + 8 * h;
      float* row = so + (warp * 16 + r) * kPitch;
      if constexpr (kKv8) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<float4*>(row + 16 * u + 2 * q2) =
              make_float4(st.o[g][2 * u][2 * h], st.o[g][2 * u + 1][2 * h],
                          st.o[g][2 * u][2 * h + 1], st.o[g][2 * u + 1][2 * h + 1]);
      } else {
#pragma unroll
        for (int n = 0; n < 16; ++n)
          *reinterpret_cast<float2*>(row + 8 * n + q2) =
              make_float2(st.o[g][n][2 * h], st.o[g][n][2 * h + 1]);
      }
      if (q2 == 0) {
        sm[warp * 16 + r] = st.m[g][h];
        sl[warp * 16 + r] = st.l[g][h];
      }
    }
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
#pragma unroll 1
    for (int e = threadIdx.x; e < sets * 16 * 16; e += kRowsWarps * 32) {
      const int sr_ = e >> 4, d = (e & 15) * 8;          // row among the sets' rows of this group
      const int set_ = sr_ >> 4, rr = sr_ & 15;
      const int r = set_ * 16 * kRG + 16 * g + rr;       // row of the tile
      const int tok = r >> 1;
      if (tok >= n_q) continue;
      bool alive = true;
      if constexpr (kTree) {
        const int k = tok0 + tok;
        alive = masks[static_cast<long long>(k) * words + (k >> 5)] >> (k & 31) & 1;
      }
      float M = -INFINITY, L = 0.f, x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      for (int p = 0; p < phases; ++p) M = fmaxf(M, sm[(p * sets + set_) * 16 + rr]);
#pragma unroll 1
      for (int p = 0; p < phases; ++p) {
        const int w = (p * sets + set_) * 16 + rr;
        const float mw = sm[w], lw = sl[w];
        float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
        if (lw != lw) f = 1.f;  // a phase whose scores were all NaN never raised its maximum
        L += lw * f;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(so + w * kPitch + d + i);
          x[i] += v.x * f;
          x[i + 1] += v.y * f;
          x[i + 2] += v.z * f;
          x[i + 3] += v.w * f;
        }
      }
      float scale = L != 0.f ? 1.f / L : 0.f;  // a NaN sum stays NaN
      const float lse = alive && L != 0.f ? M + __log2f(L) : -INFINITY;
      if (part_row >= 0) {
        const long long prow = static_cast<long long>(part_row + r) * a.num_kv + kvh;
        float* dst = a.ws_o + prow * kHeadDim + d;
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *reinterpret_cast<float4*>(dst + i) =
              alive ? make_float4(x[i] * scale, x[i + 1] * scale, x[i + 2] * scale, x[i + 3] * scale)
                    : make_float4(0.f, 0.f, 0.f, 0.f);
        if (d == 0) a.ws_lse[prow] = lse;
        continue;
      }
      if constexpr (kKv8 && !kTree) {
        if (merge_row >= 0) {  // a cascade row: with the shared-prefix partial
          const long long prow = static_cast<long long>(merge_row + r) * a.num_kv + kvh;
          const float lse_p = a.ws_lse[prow];
          const float top = fmaxf(lse, lse_p);
          const float wu = lse == -INFINITY ? 0.f : fast_exp2(lse - top);
          const float wp = lse_p == -INFINITY ? 0.f : fast_exp2(lse_p - top);
          const float n = wu + wp != 0.f ? 1.f / (wu + wp) : 0.f;
          scale *= wu * n;
          const float* op = a.ws_o + prow * kHeadDim + d;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * scale + op[i] * (wp * n);
          scale = 1.f;
        }
      }
      __nv_bfloat16* dst = a.out + static_cast<long long>(flat_start + tok0 + tok) * a.out_row_stride +
                           (kvh * kGroup + (r & 1)) * kHeadDim + d;
      uint4 y = make_uint4(0u, 0u, 0u, 0u);
      if (alive)
        y = make_uint4(pack_bf16(x[0] * scale, x[1] * scale), pack_bf16(x[2] * scale, x[3] * scale),
                       pack_bf16(x[4] * scale, x[5] * scale), pack_bf16(x[6] * scale, x[7] * scale));
      *reinterpret_cast<uint4*>(dst) = y;
    }
  }

  if (ra.behind) pdl_wait();
  if (part_row >= 0) {
    // A split of a tile, or the last pages of one whose cached blocks the tensor-core kernel read
    // before this launch: the last one to arrive merges them all.
    __threadfence();
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
    const int* cr = ra.combines + static_cast<long long>(it[6]) * kRec;
    if (threadIdx.x == 0) {
      unsigned* counter = ra.arrived + static_cast<long long>(it[6]) * a.num_kv + kvh;
      // Wraps to 0 with the last arrival: ready for the next call.
      *last_flag = atomicInc(counter, static_cast<unsigned>(cr[6] - 1)) == static_cast<unsigned>(cr[6] - 1);
    }
    asm volatile("bar.sync 1, %0;" ::"r"(kRowsWarps * 32) : "memory");
    if (*last_flag) {
      __threadfence();
      merge_splits(a, reinterpret_cast<float*>(ring), cr[3], cr[4], cr[5], n_q * kGroup, kvh,
                   flat_start + tok0,
                   kTree ? masks + static_cast<long long>(tok0) * words : nullptr, words, tok0);
    }
  }
}

}  // namespace ms
