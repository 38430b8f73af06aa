// Sparse attention over selected pages: the key bounds of pages, the selection of the pages whose keys
// could score highest, and attention over the keys of the selected pages.
//
// A page is the 16 tokens of one block, of one KV head.  Its bounds are, per channel d, the smallest and
// the largest key value lo_d, hi_d over its tokens (bf16 values, or what 8-bit rows stand for, which are
// bf16 values too: nothing is rounded).  For a query q no key within the bounds has a product above
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d,
// and a page's score is the larger one of that for the two query heads of the KV head.  The two sums are the same
// where the bounds are finite.  The second one, which is computed, is infinite or NaN for every q where a bound is
// not finite (0 times infinity on the side that q_d rules out): such a page holds a key that is not finite, and
// counts as one of infinite score.
#pragma once

#include <cstddef>

#include "kv8.cuh"
#include "paged_attention.cuh"
#include "qkv_proj_tc.cuh"
#include "rows_attention.cuh"

namespace ms {

constexpr int kShortQuery = 8;                    // rows of sequences with more new tokens are not sparse
constexpr int kBoundsBytes = 2 * kHeadDim * 2;    // lo, hi: [2][128] bf16 of one page
constexpr int kMaxSelectPages = 49152;            // pages a row may see: its scores lie in shared memory
constexpr int kMaxBudget = 4096;                  // pages a row may keep
constexpr int kMaxCluster = 8;                    // CTAs that share a row

// Fields of a plan's sequence records (8 ints each).
struct SeqRec {
  int flat_start, num_new, num_cached, context_len, table_off;
};
__device__ __forceinline__ SeqRec load_seq(const int* seqs, int s) {
  const int4 a = *reinterpret_cast<const int4*>(seqs + 8 * s);
  return {a.x, a.y, a.z, a.w, seqs[8 * s + 4]};
}

// ---- key bounds ----------------------------------------------------------------------------------

struct BoundsArgs {
  const uint8_t* pool;  // first byte of the layer
  uint8_t* bounds;      // [num_blocks][kv_heads][2][128] bf16
  const int* seqs;      // a step's plan: the pages that its new tokens lie on ...
  const int* tables;
  const long long* blocks;  // ... or pages by block, with the number of their tokens
  const long long* rows;
  int num;  // sequences, or pages
  int num_kv;
  int num_blocks;
};

__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                 *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                 *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

// Launch latency bounds a decode step (61 rows: 2.3 us), memory a prompt (16384 tokens of an 8-bit pool: 7.0 us of
// which 21 MB take 3.2).
//
// Bounds of the first `rows` tokens of one page, by one warp.  Lane l reads 16-byte pieces: piece l % 8 of
// tokens l / 8, + 4, + 8, + 12, so each load of the warp covers 512 contiguous bytes; NaN keys give NaN
// bounds.  Every lane ends with 16 channels and stores a quarter of them.
template <bool kKv8>
__device__ __forceinline__ void page_bounds(const BoundsArgs& a, int block, int head, int rows,
                                            int lane) {
  constexpr uint32_t kPosInf = 0x7f807f80u, kNegInf = 0xff80ff80u;
  const long long page = static_cast<long long>(block) * a.num_kv + head;
  const int piece = lane & 7, group = lane >> 3;
  uint32_t lo[8], hi[8];  // bf16: pieces of the two halves of a row; 8-bit: 16 neighbouring channels
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = kPosInf, hi[i] = kNegInf;
  uint4 x[4][kKv8 ? 1 : 2];
  int b[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int tok = 4 * p + group;
    if constexpr (kKv8) {
      const uint8_t* at = a.pool + page * kPage8Bytes;
      x[p][0] = make_uint4(0u, 0u, 0u, 0u);
      b[p] = 0;
      if (tok < rows) {
        x[p][0] = *reinterpret_cast<const uint4*>(at + code_off8(tok, piece));
        b[p] = at[kExp8Off + tok];
      }
    } else {
      const uint8_t* at = a.pool + page * kPageKVBytes + tok * 128 + piece * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[p][h] = make_uint4(0u, 0u, 0u, 0u);
        if (tok < rows) x[p][h] = *reinterpret_cast<const uint4*>(at + h * (kPageBytes / 2));
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    if (4 * p + group >= rows) continue;
    uint32_t w[8];
    if constexpr (kKv8) {
      const float s = row_scale8(b[p]);
      expand4(x[p][0].x, s, w[0], w[1]);
      expand4(x[p][0].y, s, w[2], w[3]);
      expand4(x[p][0].z, s, w[4], w[5]);
      expand4(x[p][0].w, s, w[6], w[7]);
    } else {
      w[0] = x[p][0].x, w[1] = x[p][0].y, w[2] = x[p][0].z, w[3] = x[p][0].w;
      w[4] = x[p][1].x, w[5] = x[p][1].y, w[6] = x[p][1].z, w[7] = x[p][1].w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = min2_nan(lo[i], w[i]), hi[i] = max2_nan(hi[i], w[i]);
  }
#pragma unroll
  for (int off = 8; off <= 16; off <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = min2_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], off));
      hi[i] = max2_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], off));
    }
  uint4 y;
  if (group < 2) {
    y = group == 0 ? make_uint4(lo[0], lo[1], lo[2], lo[3]) : make_uint4(lo[4], lo[5], lo[6], lo[7]);
  } else {
    y = group == 2 ? make_uint4(hi[0], hi[1], hi[2], hi[3]) : make_uint4(hi[4], hi[5], hi[6], hi[7]);
  }
  const int part = group & 1;
  const int channel = kKv8 ? piece * 16 + part * 8 : part * 64 + piece * 8;
  *reinterpret_cast<uint4*>(a.bounds + page * kBoundsBytes + (group >> 1) * kHeadDim * 2 +
                            channel * 2) = y;
}

// Of a step: CTAs (x: sequence, y: share of its pages), a warp per (page, KV head).
template <bool kKv8, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) key_bounds_step_kernel(const BoundsArgs a,
                                                                      unsigned* status) {
  pdl_wait();
  pdl_trigger();
  const SeqRec s = load_seq(a.seqs, blockIdx.x);
  if (s.num_new <= 0) return;
  const int lane = threadIdx.x & 31;
  const int first = s.num_cached / kBlockTokens;
  const int units = ((s.context_len - 1) / kBlockTokens + 1 - first) * a.num_kv;
  for (int u = blockIdx.y * kWarps + (threadIdx.x >> 5); u < units; u += gridDim.y * kWarps) {
    const int page = first + u / a.num_kv;
    const int block = a.tables[s.table_off + page];
    if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.num_blocks)) {
      if (lane == 0) atomicOr(status, kErrBlock);
      continue;
    }
    page_bounds<kKv8>(a, block, u % a.num_kv, min(kBlockTokens, s.context_len - page * kBlockTokens),
                      lane);
  }
}

// Of a list of blocks: a warp per (block, KV head).  Blocks below 0 and blocks without tokens are skipped.
template <bool kKv8, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) key_bounds_kernel(const BoundsArgs a,
                                                                 unsigned* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long u = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const long long i = u / a.num_kv;
  if (i >= a.num) return;
  const long long block = a.blocks[i], rows = a.rows[i];
  if (block < 0 || rows <= 0) return;
  if (block >= a.num_blocks) {
    if (lane == 0) atomicOr(status, kErrBlock);
    return;
  }
  page_bounds<kKv8>(a, static_cast<int>(block), static_cast<int>(u - i * a.num_kv),
                    static_cast<int>(min(rows, static_cast<long long>(kBlockTokens))), lane);
}

// ---- selection -------------------------------------------------------------------------------------

struct SelectArgs {
  const __nv_bfloat16* q;
  long long q_row_stride;
  const uint8_t* bounds;
  const int* seqs;
  const int* tables;
  int* pages;  // [T][kv_heads][budget]
  int max_new;
  int num_kv;
  int num_blocks;
  int budget, first, last;
  // Of each (sequence, new token, KV head): the scores of `capacity` pages (a multiple of 64), and of each 16
  // of them the largest sum of magnitudes, as bits.
  int capacity;
  float* scores;
  uint32_t* sums;
};

// The block-wide pieces below are called by every thread of a CTA of kThreads.
template <int kThreads>
__device__ __forceinline__ int block_exclusive_scan(int x, int* total, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += y;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  // Every warp scans the warps' sums: a load each and five steps, not a load for every warp.
  int sums = lane < kThreads / 32 ? scratch[lane] : 0;
#pragma unroll
  for (int off = 1; off < kThreads / 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sums, off);
    if (lane >= off) sums += y;
  }
  *total = __shfl_sync(0xffffffffu, sums, kThreads / 32 - 1);
  const int before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
  return (warp > 0 ? before : 0) + v - x;
}

// The want-th largest (want >= 1) of the keys whose bit in `among` is set (null: all of m), eight bits a
// pass; *above gets how many of them are larger, *same how many are equal.
template <int kThreads>
__device__ uint32_t radix_select(const uint32_t* keys, const uint32_t* among, int m, int want,
                                 int* above, int* same, int* hist) {
  uint32_t prefix = 0, mask = 0;
  int larger = 0, equal = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix && (among == nullptr || (among[i >> 5] >> (i & 31) & 1u)))
        atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // bins from the top: lane l has 255 - 8 l .. 248 - 8 l
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - 8 * threadIdx.x - i];
      int run = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, off);
        if (static_cast<int>(threadIdx.x) >= off) run += y;
      }
      int over = larger + run - sum;
      if (over < want && over + sum >= want) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (over < want && over + c[i] >= want) {
            hist[256] = 255 - 8 * threadIdx.x - i;
            hist[257] = over;
            hist[258] = c[i];
          }
          over += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(hist[256]) << shift;
    mask |= 255u << shift;
    larger = hist[257];
    equal = hist[258];
  }
  *above = larger;
  *same = equal;
  __syncthreads();
  return prefix;
}

// Scores in 64 bits, where every product of two bf16 values is exact and 256 of them lose nothing that
// ordinary keys differ by: selections are those of the definition, not of a summation's order.  One warp:
// lanes 0-15 hold lo and min(q, 0), lanes 16-31 hi and max(q, 0), 8 channels each.
struct ExactQuery {
  double q[kGroup][8];
};
__device__ __forceinline__ ExactQuery exact_query(const __nv_bfloat16* q, int lane) {
  ExactQuery e;
#pragma unroll
  for (int g = 0; g < kGroup; ++g) {
    const uint4 x = *reinterpret_cast<const uint4*>(q + g * kHeadDim + (lane & 15) * 8);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
      // Not fminf and fmaxf: a NaN stays one.
      e.q[g][i] = (lane < 16 ? v > 0.f : v < 0.f) ? 0.0 : static_cast<double>(v);
    }
  }
  return e;
}
// The score as a number that orders like it: not finite counts as infinite, -0 as 0.
__device__ __forceinline__ unsigned long long exact_key(const ExactQuery& e, const uint8_t* bounds,
                                                        int lane) {
  const uint4 x = *reinterpret_cast<const uint4*>(bounds + lane * 16);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  double s[kGroup] = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double v = (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
#pragma unroll
    for (int g = 0; g < kGroup; ++g) s[g] = fma(e.q[g][i], v, s[g]);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
    for (int g = 0; g < kGroup; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], off);
  double top = s[0] > s[1] ? s[0] : s[1];
  if (isnan(s[0]) || isnan(s[1]) || isinf(top)) top = __longlong_as_double(0x7ff0000000000000LL);
  const long long b = __double_as_longlong(top + 0.0);
  return static_cast<unsigned long long>(b < 0 ? ~b : b ^ (1LL << 63));
}

// What a CTA of kThreads keeps in shared memory beside the scores.
template <int kThreads>
struct SelectShared {
  static constexpr int kBins = kThreads > 256 ? kThreads : 256;
  static constexpr int kClose = kThreads >= 256 ? 256 : 64;  // pages near the border: scored in 64 bits
  int bins[kBins + 4];  // also the radix passes' and the scans' scratch
  unsigned long long close_key[kClose];
  int close[kClose];
  int scratch[kThreads / 32];
  int found, sure, n_close;
  // Of the scores: the largest negated one, the largest one (both as ordered_bits), the largest sum of magnitudes.
  uint32_t low, high, most;
};

// fp32 numbers (no NaN) as unsigned ones of the same order, and back; none is 0.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered_bits(uint32_t b) {
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// Marks in `taken` the `want` pages (1 <= want <= m) with the highest scores by scoring every page in 64
// bits and two radix selections, of the upper and of the lower half of what orders them.  For scores that
// fp32 cannot tell apart or hold.
template <int kThreads, typename Bounds>
__device__ __noinline__ void take_exactly(uint32_t* keys, uint32_t* taken, uint32_t* ties, int m, int want,
                                          int* hist, const __nv_bfloat16* q, const Bounds& bounds_of) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int words = (m + 31) / 32;
  const ExactQuery e = exact_query(q, lane);
  __syncthreads();
  for (int i = warp; i < m; i += kThreads / 32) {
    const unsigned long long k = exact_key(e, bounds_of(i), lane);
    if (lane == 0) keys[i] = static_cast<uint32_t>(k >> 32);
  }
  __syncthreads();
  int above, same;
  const uint32_t border = radix_select<kThreads>(keys, nullptr, m, want, &above, &same, hist);
  for (int w = warp; w < words; w += kThreads / 32) {
    const int i = 32 * w + lane;
    const uint32_t k = i < m ? keys[i] : 0u;
    const unsigned t = __ballot_sync(0xffffffffu, i < m && k > border);
    const unsigned u = __ballot_sync(0xffffffffu, i < m && k == border);
    if (lane == 0) taken[w] = t, ties[w] = u;
  }
  __syncthreads();
  int left = want - above;
  if (left < same) {  // more pages share the border's upper half than are left to take
    for (int i = warp; i < m; i += kThreads / 32)
      if (ties[i >> 5] >> (i & 31) & 1u) {
        const unsigned long long k = exact_key(e, bounds_of(i), lane);
        if (lane == 0) keys[i] = static_cast<uint32_t>(k);
      }
    __syncthreads();
    const uint32_t low = radix_select<kThreads>(keys, ties, m, left, &above, &same, hist);
    left -= above;
    for (int w = warp; w < words; w += kThreads / 32) {
      const int i = 32 * w + lane;
      const bool tie = i < m && (ties[w] >> lane & 1u);
      const unsigned t = __ballot_sync(0xffffffffu, tie && keys[i] > low);
      const unsigned u = __ballot_sync(0xffffffffu, tie && keys[i] == low);
      if (lane == 0) taken[w] |= t, ties[w] = u;
    }
    __syncthreads();
  }
  // The first `left` ties, by index.
  const int per = (words + kThreads - 1) / kThreads, w0 = threadIdx.x * per;
  int mine = 0, total;
  for (int w = w0; w < min(words, w0 + per); ++w) mine += __popc(ties[w]);
  int before = block_exclusive_scan<kThreads>(mine, &total, hist);
  for (int w = w0; w < min(words, w0 + per); ++w)
    for (unsigned u = ties[w]; u != 0u && before < left; u &= u - 1, ++before) taken[w] |= u & (0u - u);
  __syncthreads();
}

// The same from fp32 scores in [low, high] that are off by at most `error` each.  A histogram finds the bin of
// the want-th largest score, between lo and hi.  The true border is within `error` of that, so a page whose
// score is over hi + 2 error is taken and one below lo - 2 error is not, and the few between are scored in 64
// bits and ranked, ties by index.  (2.5 for 2: the ends of the bin and the sums round, by less than 2^-20 of the
// scores' bound, of which `error` is 2^-14.)  Where more than kClose are between, they are divided again.
// False: they do not part in fp32.
template <int kThreads, typename Bounds>
__device__ __forceinline__ bool take_by_scores(const float* scores, uint32_t* taken, int m, int want,
                                               float low, float high, float error,
                                               SelectShared<kThreads>& sh,
                                               const __nv_bfloat16* q, const Bounds& bounds_of) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kBins = SelectShared<kThreads>::kBins, kClose = SelectShared<kThreads>::kClose;
  const float slack = 2.5f * error;
  int above = 0;  // scores over `high`
#pragma unroll 1
  for (int level = 0; level < 4; ++level) {
    if (level > 0) {  // the first time the caller has cleared them
      for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
      if (threadIdx.x == 0) sh.n_close = sh.sure = 0;
      __syncthreads();
    }
    const float per = high > low ? kBins / (high - low) : 0.f;
#pragma unroll 4
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const float s = scores[i];
      if (s >= low && s <= high)
        atomicAdd(&sh.bins[min(kBins - 1, static_cast<int>((s - low) * per))], 1);
    }
    __syncthreads();
    {  // bins from the top: each thread a run of them
      constexpr int kRun = kBins / kThreads;
      int c[kRun], sum = 0, total;
#pragma unroll
      for (int i = 0; i < kRun; ++i) sum += c[i] = sh.bins[kBins - 1 - kRun * threadIdx.x - i];
      int over = above + block_exclusive_scan<kThreads>(sum, &total, sh.scratch);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if (over < want && over + c[i] >= want) sh.found = kBins - 1 - kRun * threadIdx.x - i;
        over += c[i];
      }
    }
    __syncthreads();
    const float width = (high - low) * (1.f / kBins);
    const float lo = low + sh.found * width, hi = low + (sh.found + 1) * width;
    // Taken, between, or neither.
    const float sure_from = hi + slack, close_from = lo - slack;
    int sure = 0;
#pragma unroll 4
    for (int i0 = warp * 32; i0 < m; i0 += kThreads) {
      const int i = i0 + lane;
      const float s = i < m ? scores[i] : -INFINITY;
      const unsigned t = __ballot_sync(0xffffffffu, s > sure_from);
      const unsigned u = __ballot_sync(0xffffffffu, s >= close_from) & ~t;
      if (lane == 0) taken[i0 >> 5] = t;
      sure += __popc(t);
      if (u >> lane & 1u) {
        const int at = atomicAdd(&sh.n_close, 1);
        if (at < kClose) sh.close[at] = i;
      }
    }
    if (lane == 0) atomicAdd(&sh.sure, sure);
    __syncthreads();
    const int n = sh.n_close, left = want - sh.sure;
    if (n <= kClose) {
      if (left < n) {
        if (warp < n) {
          const ExactQuery e = exact_query(q, lane);
          for (int j = warp; j < n; j += kThreads / 32) {
            const unsigned long long k = exact_key(e, bounds_of(sh.close[j]), lane);
            if (lane == 0) sh.close_key[j] = k;
          }
        }
        __syncthreads();
      }
      // A warp places a page among the others.
      for (int j = warp; j < n; j += kThreads / 32) {
        const int i = sh.close[j];
        int place = 0;
        if (left < n) {
          const unsigned long long k = sh.close_key[j];
          for (int o = lane; o < n; o += 32)
            place += sh.close_key[o] > k || (sh.close_key[o] == k && sh.close[o] < i);
          place = __reduce_add_sync(0xffffffffu, place);
        }
        if (lane == 0 && place < left) atomicOr(&taken[i >> 5], 1u << (i & 31));
      }
      __syncthreads();
      return true;
    }
    low = close_from, high = sure_from, above = sh.sure;
    if (!(high - low > 16.f * error)) return false;
    __syncthreads();
  }
  return false;
}

// ---- scores ------------------------------------------------------------------------------------
//
// Scoring is a product of the pages' bounds [lo, hi] with the queries' [min(q, 0), max(q, 0)], 256 deep, on
// mma.sync: 16 pages are the rows of A, and the columns of B are the query heads of four tokens, so that a
// lane ends with both heads of one token and two pages.  The order of the 256 is free as long as A and B
// agree, so that a lane's 16-byte piece of a page is its share of two products.  A second product, of the
// magnitudes, gives sum_d |q_d bound_d|: an fp32 score is off by less than 2^-14 of that.  (Each of the 16
// products adds 16 exact products to its running sum, and loses from each of these 17 at most 2^-23 of the
// largest, 16 * 17 2^-23 < 2^-14.9 in all; then two sums are added.)
//
// The loads bound it, 512 bytes a page and head.  One CTA per SM takes an equal run of all the work, in items
// of 16 pages x 8 heads (or as many pages more as there are heads fewer); one warp keeps bulk copies of whole
// items in flight through a ring, a warp per head multiplies.  Copies of all heads of a block are contiguous:
// with heads in different CTAs, DRAM gave 3.5 TB/s to pieces of 512 bytes (32 rows over 8000-32000 tokens, 144 MB:
// 40 us; in this form 29, where the copy rate allows 22).

constexpr int kScoreWarps = 8;
constexpr int kScoreStages = 3;
constexpr int kTilePages = 16;

// How the heads of a block are shared out: `heads` neighbouring ones per item (a divisor of the KV heads) and
// `tiles` tiles of 16 pages, at most kScoreWarps products in all.
struct ScoreShape {
  int heads, tiles;
  __host__ __device__ int pitch() const { return heads * kBoundsBytes + 64; }  // 64: no bank conflicts
  __host__ __device__ int pages() const { return tiles * kTilePages; }
  __host__ __device__ int stage_bytes() const { return pages() * pitch(); }
};

struct ScoreArgs {
  SelectArgs s;
  ScoreShape shape;
  int num_seqs;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Pages of a sequence that are scored: those between the first and the last ones of its last token.
__device__ __forceinline__ int scored_pages(const SelectArgs& a, int num_new, int num_cached) {
  if (num_new < 1 || num_new > kShortQuery || num_new > a.max_new) return 0;
  const int n = (num_cached + num_new - 1) / kBlockTokens + 1;
  return n > a.budget && a.budget > a.first + a.last ? min(n - a.first - a.last, a.capacity) : 0;
}

// The work of one CTA: items lo .. hi of all, head group by head group and sequence by sequence.  Every warp
// walks it by itself.
struct ScoreWalk {
  int seq, item, items;  // the present sequence, the item in it, how many it has
  int group;
  int most, table_off;
};
__device__ __forceinline__ int items_of(const ScoreArgs& a, int seq, int* most, int* table_off) {
  const int4 x = *reinterpret_cast<const int4*>(a.s.seqs + 8 * seq);
  *table_off = a.s.seqs[8 * seq + 4];
  *most = scored_pages(a.s, x.y, x.z);
  return (*most + a.shape.pages() - 1) / a.shape.pages();
}
// To the first sequence from `from` on that has items, or the first one of the next group.
__device__ __forceinline__ void walk_to(const ScoreArgs& a, ScoreWalk& w, int from, int lane) {
  for (; w.group < a.s.num_kv / a.shape.heads; ++w.group) {
    for (int s0 = from; s0 < a.num_seqs; s0 += 32) {
      int most = 0, off = 0, items = 0;
      if (s0 + lane < a.num_seqs) items = items_of(a, s0 + lane, &most, &off);
      const unsigned some = __ballot_sync(0xffffffffu, items > 0);
      if (some != 0u) {
        const int l = __ffs(some) - 1;
        w.seq = s0 + l;
        w.items = __shfl_sync(0xffffffffu, items, l);
        w.most = __shfl_sync(0xffffffffu, most, l);
        w.table_off = __shfl_sync(0xffffffffu, off, l);
        w.item = 0;
        return;
      }
    }
    from = 0;
  }
}
// The CTA's first item; returns how many it has.
__device__ __forceinline__ int walk_start(const ScoreArgs& a, ScoreWalk& w, int lane) {
  int all = 0, most, off;
  for (int s = lane; s < a.num_seqs; s += 32) all += items_of(a, s, &most, &off);
  all = __reduce_add_sync(0xffffffffu, all);
  const long long total = static_cast<long long>(all) * (a.s.num_kv / a.shape.heads);
  const long long lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
  if (lo >= hi) return 0;
  w.group = static_cast<int>(lo / all);
  int left = static_cast<int>(lo - static_cast<long long>(w.group) * all);
  for (int s0 = 0; s0 < a.num_seqs; s0 += 32) {
    int items = 0;
    if (s0 + lane < a.num_seqs) items = items_of(a, s0 + lane, &most, &off);
    int run = items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    const unsigned here = __ballot_sync(0xffffffffu, run > left);
    if (here != 0u) {
      const int l = __ffs(here) - 1;
      w.seq = s0 + l;
      w.items = __shfl_sync(0xffffffffu, items, l);
      w.most = __shfl_sync(0xffffffffu, most, l);
      w.table_off = __shfl_sync(0xffffffffu, off, l);
      w.item = left - __shfl_sync(0xffffffffu, run - items, l);
      return static_cast<int>(hi - lo);
    }
    left -= __shfl_sync(0xffffffffu, run, 31);
  }
  return 0;
}
__device__ __forceinline__ void walk_on(const ScoreArgs& a, ScoreWalk& w, int lane) {
  if (++w.item == w.items) walk_to(a, w, w.seq + 1, lane);
}

__device__ __forceinline__ uint32_t magnitudes(uint32_t x) { return x & 0x7fff7fffu; }

// B: column n of part x is query head n % 2 of token 4 x + n / 2; lane l has n = l / 4 and of each 64-byte run of
// the 512 its l % 4th 16 bytes.  q: the first token's first of the two heads.
template <int kTiles>
__device__ __forceinline__ void score_queries(const __nv_bfloat16* q, long long row_stride, int tokens,
                                              int lane, uint32_t (&b)[kTiles][8][4]) {
  const int r = lane >> 2, c = lane & 3;
#pragma unroll
  for (int x = 0; x < kTiles; ++x) {
    const int tok = 4 * x + (r >> 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 y = make_uint4(0u, 0u, 0u, 0u);
      if (tok < tokens)
        y = *reinterpret_cast<const uint4*>(q + tok * row_stride + (r & 1) * kHeadDim + (4 * j + c) * 8);
      const uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[x][j][i] = min2_nan(v[i], 0u);
        b[x][4 + j][i] = max2_nan(v[i], 0u);
      }
    }
  }
}

// Scores of the 16 pages of a tile for token 4 x + lane % 4, of pages lane / 4 and 8 + lane / 4, and the larger of
// their heads' sums of magnitudes, as bits (a NaN is the largest).  low, high: the lane's pieces of the two.
template <int kTiles>
__device__ __forceinline__ void score_tile(const uint8_t* low, const uint8_t* high,
                                           const uint32_t (&b)[kTiles][8][4], float (&score)[kTiles][2],
                                           uint32_t (&most)[kTiles]) {
  float acc[kTiles][2][4], mag[kTiles][2][4];  // two chains each: a product waits for the one before it
#pragma unroll
  for (int x = 0; x < kTiles; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[x][0][i] = acc[x][1][i] = mag[x][0][i] = mag[x][1][i] = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 u = *reinterpret_cast<const uint4*>(low + 64 * j);
    const uint4 v = *reinterpret_cast<const uint4*>(high + 64 * j);
    const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
    uint32_t m0[4], m1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m0[i] = magnitudes(a0[i]), m1[i] = magnitudes(a1[i]);
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      mma_bf16(acc[x][0], a0, b[x][j][0], b[x][j][1]);
      mma_bf16(acc[x][1], a1, b[x][j][2], b[x][j][3]);
      mma_bf16(mag[x][0], m0, magnitudes(b[x][j][0]), magnitudes(b[x][j][1]));
      mma_bf16(mag[x][1], m1, magnitudes(b[x][j][2]), magnitudes(b[x][j][3]));
    }
  }
#pragma unroll
  for (int x = 0; x < kTiles; ++x) {
    most[x] = 0u;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      score[x][half] = fmaxf(acc[x][0][2 * half] + acc[x][1][2 * half],
                             acc[x][0][2 * half + 1] + acc[x][1][2 * half + 1]);
#pragma unroll
      for (int g = 0; g < kGroup; ++g)
        most[x] = max(most[x], __float_as_uint(mag[x][0][2 * half + g] + mag[x][1][2 * half + g]));
    }
  }
}

template <int kTiles>
__global__ void __launch_bounds__((kScoreWarps + 1) * 32, 1)
    score_pages_kernel(const __grid_constant__ ScoreArgs a, unsigned* status) {
  extern __shared__ __align__(128) uint8_t score_smem[];
  __shared__ uint64_t full[kScoreStages], empty[kScoreStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const ScoreShape shape = a.shape;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < kScoreStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], shape.heads * shape.tiles);
    }
    fence_barrier_init();
  }
  __syncthreads();
  // The plan was uploaded before the kernel in front of this one started.
  ScoreWalk w;
  const int count = walk_start(a, w, lane);
  pdl_wait();
  pdl_trigger();
  if (count == 0) return;
  if (warp == kScoreWarps) {
    constexpr int kMost = kScoreWarps * kTilePages / 32;  // pages of an item per lane, at most
    const uint32_t bytes = shape.heads * kBoundsBytes;
    int blocks[kMost];  // of the next item: read before the wait for its stage
    auto look = [&] {
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int p = lane + 32 * i;
        if (p < shape.pages())
          blocks[i] = a.s.tables[w.table_off + a.s.first + min(w.item * shape.pages() + p, w.most - 1)];
      }
    };
    look();
    int k = 0;
    for (; k < count; ++k) {
      const int stage = k % kScoreStages;
      bool ok = true;
      if (k >= kScoreStages) ok = mbar_wait(&empty[stage], (k / kScoreStages - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) atomicOr(status, kErrTimeout);
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], shape.pages() * bytes);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int p = lane + 32 * i;
        if (p >= shape.pages()) continue;
        int block = blocks[i];
        if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.s.num_blocks)) {
          atomicOr(status, kErrBlock);
          block = 0;
        }
        const long long row = static_cast<long long>(block) * a.s.num_kv + w.group * shape.heads;
        bulk_load(score_smem + stage * shape.stage_bytes() + p * shape.pitch(),
                  a.s.bounds + row * kBoundsBytes, bytes, &full[stage]);
      }
      __syncwarp();
      if (k + 1 < count) {
        walk_on(a, w, lane);
        look();
      }
    }
    for (int i = max(0, k - kScoreStages); i < k; ++i)  // no copy is in flight when the CTA ends
      mbar_wait(&full[i % kScoreStages], (i / kScoreStages) & 1);
    return;
  }
  if (warp >= shape.heads * shape.tiles) return;
  const int mine = warp % shape.heads, tile = warp / shape.heads;
  const int r = lane >> 2, c = lane & 3;
  uint32_t b[kTiles][8][4];
  int seq = -1, group = -1, tokens = 0;
  for (int k = 0; k < count; ++k) {
    if (w.seq != seq || w.group != group) {
      seq = w.seq, group = w.group;
      const SeqRec rec = load_seq(a.s.seqs, seq);
      tokens = rec.num_new;
      score_queries<kTiles>(a.s.q + static_cast<long long>(rec.flat_start) * a.s.q_row_stride +
                                (group * shape.heads + mine) * kGroup * kHeadDim,
                            a.s.q_row_stride, tokens, lane, b);
    }
    const int stage = k % kScoreStages;
    const bool ok = mbar_wait(&full[stage], (k / kScoreStages) & 1);
    if (!__all_sync(0xffffffffu, ok)) {
      if (lane == 0) atomicOr(status, kErrTimeout);
      return;
    }
    const uint8_t* at = score_smem + stage * shape.stage_bytes() + (tile * kTilePages + r) * shape.pitch() +
                        mine * kBoundsBytes + c * 16;
    float score[kTiles][2];
    uint32_t most[kTiles];
    score_tile<kTiles>(at, at + 8 * shape.pitch(), b, score, most);
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    const int first = w.item * shape.pages() + tile * kTilePages;
    const int head = group * shape.heads + mine;
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      const int tok = 4 * x + c;
      const long long row = (static_cast<long long>(seq) * a.s.max_new + tok) * a.s.num_kv + head;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = first + 8 * half + r;
        if (tok < tokens && i < w.most) a.s.scores[row * a.s.capacity + i] = score[x][half];
      }
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1)
        most[x] = max(most[x], __shfl_xor_sync(0xffffffffu, most[x], off));
      if (r == 0 && tok < tokens && first < w.most)
        a.s.sums[(row * a.s.capacity + first) / kTilePages] = most[x];
    }
    if (k + 1 < count) walk_on(a, w, lane);
  }
}

// One CTA per (sequence, new token, KV head): the pages of the largest scores, in order.  kScore: it computes the
// scores too, a tile per warp with the bounds straight from memory.  That saves a launch where there are few pages.
// Latency bounds it, of about ten barriers and of code that every launch fetches anew: 5 us for 256 rows and heads of
// 1100 pages, 7 for 24 of 6250; 5.4 with the scores for 64 of up to 128.
template <int kThreads, bool kScore>
__global__ void __launch_bounds__(kThreads, kScore ? 2 : 1024 / kThreads)
    select_pages_kernel(const __grid_constant__ SelectArgs a, unsigned* status) {
  extern __shared__ __align__(16) uint32_t select_smem[];
  __shared__ SelectShared<kThreads> sh;
  // The plan was uploaded before the kernel in front of this one started.
  const int head = blockIdx.x % a.num_kv;
  const int tok = blockIdx.x / a.num_kv % a.max_new;
  const SeqRec seq = load_seq(a.seqs, blockIdx.x / (a.num_kv * a.max_new));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < SelectShared<kThreads>::kBins; i += kThreads) sh.bins[i] = 0;
  if (threadIdx.x == 0) sh.n_close = sh.sure = 0, sh.low = sh.high = sh.most = 0u;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  if (tok >= seq.num_new || seq.num_new > kShortQuery) return;
  const int n = (seq.num_cached + tok) / kBlockTokens + 1;
  int* out = a.pages + (static_cast<long long>(seq.flat_start + tok) * a.num_kv + head) * a.budget;
  if (n <= a.budget) {
    for (int i = threadIdx.x; i < a.budget; i += kThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int want = a.budget - a.first - a.last;
  for (int i = threadIdx.x; i < a.first; i += kThreads) out[i] = i;
  for (int i = threadIdx.x; i < a.last; i += kThreads) out[a.budget - a.last + i] = n - a.last + i;
  if (want == 0) return;
  const int m = min(n - a.first - a.last, a.capacity), words = (m + 31) / 32;
  float* scores = reinterpret_cast<float*>(select_smem);
  uint32_t* taken = select_smem + a.capacity;
  uint32_t* ties = taken + (a.capacity + 31) / 32;
  const int* table = a.tables + seq.table_off + a.first;
  const __nv_bfloat16* q = a.q + static_cast<long long>(seq.flat_start + tok) * a.q_row_stride +
                           head * kGroup * kHeadDim;
  auto bounds_of = [&](int i) {
    int block = table[i];
    if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.num_blocks)) {
      if (kScore) atomicOr(status, kErrBlock);
      block = 0;
    }
    return a.bounds + (static_cast<long long>(block) * a.num_kv + head) * kBoundsBytes;
  };
  // Scores to shared memory, their span, and the largest sum of magnitudes.
  uint32_t low = 0, high = 0, most = 0;
  if constexpr (kScore) {
    uint32_t b[1][8][4];
    const int r = lane >> 2, c = lane & 3;
    bool loaded = false;
    for (int t = warp * kTilePages; t < m; t += kThreads / 32 * kTilePages) {
      const uint8_t* at[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) at[half] = bounds_of(min(t + 8 * half + r, m - 1)) + c * 16;
      if (!loaded) score_queries<1>(q, a.q_row_stride, 1, lane, b);
      loaded = true;
      float score[1][2];
      uint32_t sum[1];
      score_tile<1>(at[0], at[1], b, score, sum);
      if (c == 0) {  // columns 0 and 1: the token's two heads
        most = max(most, sum[0]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = t + 8 * half + r;
          if (i < m) {
            scores[i] = score[0][half];
            low = max(low, ordered_bits(-score[0][half])), high = max(high, ordered_bits(score[0][half]));
          }
        }
      }
      __syncwarp();
    }
  } else {
    const uint32_t* sums = a.sums + static_cast<long long>(blockIdx.x) * (a.capacity / kTilePages);
    for (int i = threadIdx.x; i < (m + kTilePages - 1) / kTilePages; i += kThreads)
      most = max(most, __ldcg(sums + i));
    const float4* from = reinterpret_cast<const float4*>(a.scores + static_cast<long long>(blockIdx.x) * a.capacity);
#pragma unroll 4
    for (int i = threadIdx.x; i < (m + 3) / 4; i += kThreads) {
      const float4 x = __ldcg(from + i);
      reinterpret_cast<float4*>(scores)[i] = x;
      const float s[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * i + e < m) low = max(low, ordered_bits(-s[e])), high = max(high, ordered_bits(s[e]));
    }
  }
  low = __reduce_max_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) atomicMax(&sh.low, low), atomicMax(&sh.high, high), atomicMax(&sh.most, most);
  __syncthreads();
  low = sh.low, high = sh.high, most = sh.most;
  const float error = 0x1p-14f * __uint_as_float(most);
  // Values that are not finite, sums that could overflow, products that could be flushed: nothing that fp32
  // says holds.
  bool done = error > 0x1p-80f && error < 0x1p100f;
  if (most == 0u) {  // queries of zeros (padded rows), or products that vanished
    const uint4 x = *reinterpret_cast<const uint4*>(q + lane * 8);
    done = !__any_sync(0xffffffffu, magnitudes(x.x | x.y | x.z | x.w) != 0u);
    for (int w = threadIdx.x; done && w < words; w += kThreads)
      taken[w] = want >= 32 * (w + 1) ? 0xffffffffu : want > 32 * w ? (1u << (want - 32 * w)) - 1u : 0u;
    __syncthreads();
  } else if (done)
    done = take_by_scores<kThreads>(scores, taken, m, want, -from_ordered_bits(low), from_ordered_bits(high),
                                    error, sh, q, bounds_of);
  if (!done) take_exactly<kThreads>(select_smem, taken, ties, m, want, sh.bins, q, bounds_of);
  // Each page's place: the pages taken in the words before it (over the ties, which are done with), and in its own.
  for (int w0 = 0, run = a.first; w0 < words; w0 += kThreads) {
    const int w = w0 + threadIdx.x;
    int total;
    const int before = block_exclusive_scan<kThreads>(w < words ? __popc(taken[w]) : 0, &total, sh.scratch);
    if (w < words) ties[w] = run + before;
    run += total;
  }
  __syncthreads();
#pragma unroll 2
  for (int i = threadIdx.x; i < m; i += kThreads) {
    const uint32_t bits = taken[i >> 5], below = (1u << (i & 31)) - 1u;
    if (bits >> (i & 31) & 1u) {
      const int at = static_cast<int>(ties[i >> 5]) + __popc(bits & below);
      if (at < a.budget) out[at] = a.first + i;
    }
  }
}

// ---- attention over selected pages ------------------------------------------------------------------

struct PagesArgs {
  const __nv_bfloat16* q;
  long long q_row_stride;
  __nv_bfloat16* out;
  long long out_row_stride;
  const uint8_t* pool;  // first byte of the layer
  const int* seqs;
  const int* tables;
  const int* pages;  // [T][kv_heads][budget]
  int max_new;
  int num_kv;
  int num_blocks;
  int budget;
  int cluster;  // CTAs of a row and head
  int stages;   // of a warp's ring
  float scale_log2;
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t x) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}

// A warp takes a page at a time out of its own ring in shared memory, with mma.sync:
// * S = Q K^T, 16 channels deep and 8 keys wide a product.  A holds the two query heads in turn in its first
//   eight rows, so that lane 4 r + c ends with the scores of head r % 2 for four keys: page_key(., i, c).
// * O^T = V^T P^T, 16 channels by 16 keys by 8 columns a product.  B are the weights of just these four keys:
//   P moves nowhere.  A are two keys' values at a time, interleaved after their loads.
// The order of the channels in the first product and of its rows in the second is free, and so is that of the
// keys.  They are taken so that the 16-byte loads of eight lanes hit eight different banks' worth of the
// page: a bf16 page has the 128-byte swizzle of its TMA load, an 8-bit one its own (code_swizzle8).
//
// Key of column n of the g-th product of eight keys.
template <bool kKv8>
__host__ __device__ constexpr int column_key(int n, int g) {
  if constexpr (kKv8) return n + 8 * ((g ^ (n >> 1) ^ n) & 1);
  return ((n & 1) ? ((n - 1) ^ 4) + 1 : n) + 8 * g;
}
// Key of a lane's i-th score.
template <bool kKv8>
__host__ __device__ constexpr int page_key(int i, int c) {
  return column_key<kKv8>(2 * c + (i & 1), i >> 1);
}
// Byte offset in K (or V) of 16-byte piece `piece` of a key: of its 8 (8-bit), or of its 16 in two halves.
template <bool kKv8>
__host__ __device__ constexpr int piece_off(int key, int piece) {
  if constexpr (kKv8) return code_off8(key, piece);
  return (piece >> 3) * (kPageBytes / 2) + key * 128 + (((piece & 7) ^ (key & 7)) << 4);
}
// What the above has to hold: every key is met once, and the loads of eight lanes meet eight different 16 bytes of
// the 128 that the banks serve at a time.
template <bool kKv8>
constexpr bool page_layout_holds() {
  unsigned columns = 0, scores = 0;
  for (int i = 0; i < 16; ++i) {
    columns |= 1u << column_key<kKv8>(i & 7, i >> 3);
    scores |= 1u << page_key<kKv8>(i & 3, i >> 2);
  }
  bool apart = true;
  for (int first = 0; first < 32; first += 8)
    for (int i = 0; i < 4; ++i)
      for (int g = 0; g < 2; ++g) {
        unsigned keys = 0, values = 0;
        for (int lane = first; lane < first + 8; ++lane) {
          const int r = lane >> 2, c = lane & 3;
          keys |= 1u << (piece_off<kKv8>(column_key<kKv8>(r, g), kKv8 ? 4 * (i & 1) + c : 4 * i + c) >> 4 & 7);
          values |= 1u << (piece_off<kKv8>(page_key<kKv8>(i, c), kKv8 ? r : 8 * g + r) >> 4 & 7);
        }
        apart = apart && keys == 0xffu && values == 0xffu;
      }
  return columns == 0xffffu && scores == 0xffffu && apart;
}
static_assert(page_layout_holds<false>() && page_layout_holds<true>(), "layout of the products over a page");

// A warp's ring: `stages` pages in flight.
template <bool kKv8>
constexpr int kStageBytes = kKv8 ? kPage8Bytes : kPageKVBytes;
constexpr int kMaxPageStages = 4;

// Queries as A: the channels of a lane's key pieces, of head r % 2.  For an 8-bit pool in f16, times 2^-shift
// so that the row's largest value is near 2^13: exact but for values 2^-27 of it (and in rows below 2^-87, which are
// scaled by 2^100).  2^shift goes to the score before the key row's scale where it is below 1 and after it where it is
// above: the two may be near opposite ends of fp32's range.
template <bool kKv8>
struct PageQuery {
  uint32_t x[16];
  float unit;  // of a score, in the exponent of 2
  float after;
  __device__ __forceinline__ void load(const __nv_bfloat16* q, float scale_log2, int lane) {
    const int c = lane & 3;
    q += ((lane >> 2) & 1) * kHeadDim;
    unit = scale_log2;
    if constexpr (!kKv8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 y = *reinterpret_cast<const uint4*>(q + (4 * j + c) * 8);
        x[4 * j] = y.x, x[4 * j + 1] = y.y, x[4 * j + 2] = y.z, x[4 * j + 3] = y.w;
      }
    } else {
      uint4 y[2][2];
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[j][i] = *reinterpret_cast<const uint4*>(q + (4 * j + c) * 16 + i * 8);
          top = __vmaxu2(top, amax8(y[j][i]));
        }
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int shift = min(max(static_cast<int>(top >> 7) - 127 - 13, -100), 254 - 127 - 13);
      const float down = __int_as_float((127 - shift) << 23);
      unit *= __int_as_float((127 + min(shift, 0)) << 23);
      after = __int_as_float((127 + max(shift, 0)) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w[4] = {y[j][i].x, y[j][i].y, y[j][i].z, y[j][i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __half2 h = __floats2half2_rn(bf16_lo(w[k]) * down, bf16_hi(w[k]) * down);
            x[8 * j + 4 * i + k] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
    }
  }
};

// One warp's share of a row, for head r % 2: running maximum m of the scores, sum of 2^(s - m), and the sum of
// 2^(s - m + e - lead) c over keys with values c 2^e.
// * bf16 (e = 0): lead = 24, so that the sum of 2^16 values of any size stays in fp32's range (the shares of values
//   below 2^-100 reach its smallest numbers).
// * 8-bit: codes c, and lead follows the largest s - m + e, so that values of any size do not overflow, and rows whose
//   2^(s + e) is within 2^-14 of the largest one keep their weight; below that it loses bits, and a share below 2^-36 of
//   the largest 2^(s + e) is lost (f16's smallest number, 2^-24, of a second part that is held 2^12 larger).
// Both move only when they grow by more than 8 (weights up to 2^8), which few pages do.  Scores enter as differences
// from m alone: beside a score beyond 2^24, fp32 does not hold the 24 or an e that is added to it.
// A weight is two bf16 or f16 numbers, itself and what its rounding lost (f16: times 2^12), in columns 0-1
// and 2-3 of B, which a product with eight columns has room for: weights are exact to 2^-17 (f16 2^-22).
template <bool kKv8>
struct RowState {
  float m, lead, sum;  // lead: 8-bit
  float acc[8][4];  // product t: channels of rows r and r + 8, columns 2 c and 2 c + 1
};
// Channel of acc[t][0] (head 0) and acc[t][1] (head 1); acc[t][2], [3] are the next one's.
template <bool kKv8>
__device__ __forceinline__ int row_channel(int r, int t) {
  return kKv8 ? r * 16 + 2 * t : (t >> 2) * 64 + r * 8 + 2 * (t & 3);
}

template <bool kKv8>
__device__ __forceinline__ void page_scores(const PageQuery<kKv8>& q, const uint8_t* page, int lane,
                                            float (&s)[4]) {
  const int r = lane >> 2, c = lane & 3;
  float acc[2][2][4];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[g][0][i] = acc[g][1][i] = 0.f;
    const int key = column_key<kKv8>(r, g);
#pragma unroll
    for (int j = 0; j < (kKv8 ? 2 : 4); ++j) {
      const uint4 x = *reinterpret_cast<const uint4*>(page + piece_off<kKv8>(key, 4 * j + c));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      if constexpr (kKv8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a[4] = {q.x[8 * j + 2 * i], 0u, q.x[8 * j + 2 * i + 1], 0u};
          mma_f16(acc[g][i & 1], a, e4m3x2_to_f16x2<0>(w[i]), e4m3x2_to_f16x2<1>(w[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a[4] = {q.x[4 * j + 2 * i], 0u, q.x[4 * j + 2 * i + 1], 0u};
          mma_bf16(acc[g][i], a, w[2 * i], w[2 * i + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = (acc[i >> 1][0][i & 1] + acc[i >> 1][1][i & 1]) * q.unit;
    if constexpr (kKv8) s[i] = s[i] * row_scale8(page[kExp8Off + page_key<kKv8>(i, c)]) * q.after;
  }
}

// visible: keys of the page up to the query's position; what lies behind is no value, and 0 times it could be
// NaN.
template <bool kKv8>
__device__ __forceinline__ void page_update(const uint8_t* page, float (&s)[4], int visible, int lane,
                                            RowState<kKv8>& st) {
  const int r = lane >> 2, c = lane & 3;
  // Exponent of a key's share over 2^m, from d = s - m.
  auto share = [&](int i, float d) {
    const int key = page_key<kKv8>(i, c), b = page[kExp8Off + kBlockTokens + key];
    if (key >= visible) return -INFINITY;
    return d + (b == static_cast<int>(kExpNan) ? __int_as_float(0x7fc00000) : static_cast<float>(b - kExpBias));
  };
  float m = st.m == -INFINITY ? 0.f : st.m;
  float d[4], e[4], top = -INFINITY, most = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (page_key<kKv8>(i, c) >= visible) s[i] = -INFINITY;
    top = fmaxf(top, s[i]);
    d[i] = s[i] - m;
    if constexpr (kKv8) most = fmaxf(most, e[i] = share(i, d[i]));
  }
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if constexpr (kKv8) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
  }
  bool grow = top - st.m > 8.f;
  if constexpr (kKv8) grow = grow || most - st.lead > 8.f;
  if (__any_sync(0xffffffffu, grow)) {
    const float old = st.m;
    st.m = fmaxf(old, top);
    m = st.m == -INFINITY ? 0.f : st.m;
    const float down = old == -INFINITY ? -INFINITY : old - st.m;
    st.sum *= fast_exp2(down);
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d[i] = s[i] - m;
      if constexpr (kKv8) most = fmaxf(most, e[i] = share(i, d[i]));
    }
    float fix = fast_exp2(down);
    if constexpr (kKv8) {
#pragma unroll
      for (int off = 1; off <= 2; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
      const float was = st.lead == -INFINITY ? -INFINITY : st.lead + down;
      st.lead = fmaxf(was, most);
      fix = was == -INFINITY ? 0.f : fast_exp2(was - st.lead);
    }
    const float other = __shfl_xor_sync(0xffffffffu, fix, 4);
    const float f0 = lane & 4 ? other : fix, f1 = lane & 4 ? fix : other;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      st.acc[t][0] *= f0, st.acc[t][2] *= f0;
      st.acc[t][1] *= f1, st.acc[t][3] *= f1;
    }
  }
  const float lead = st.lead == -INFINITY ? 0.f : st.lead;
  const bool rest = lane & 8;  // columns 2 and 3, and what nobody reads
  uint32_t b[2];
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = fast_exp2(d[i]);
    st.sum += x;
    if constexpr (kKv8)
      w[i] = fast_exp2(e[i] - lead);
    else
      w[i] = x * 0x1p-24f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (kKv8) {
      const __half2 h = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
      const float2 f = __half22float2(h);
      const __half2 l = __floats2half2_rn((w[2 * i] - f.x) * 4096.f, (w[2 * i + 1] - f.y) * 4096.f);
      b[i] = rest ? *reinterpret_cast<const uint32_t*>(&l) : *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const uint32_t h = pack_bf16(w[2 * i], w[2 * i + 1]);
      const uint32_t l = pack_bf16(w[2 * i] - bf16_lo(h), w[2 * i + 1] - bf16_hi(h));
      b[i] = rest ? l : h;
    }
  }
#pragma unroll
  for (int h = 0; h < (kKv8 ? 1 : 2); ++h) {
    uint32_t y[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = page_key<kKv8>(i, c);
      uint4 x = *reinterpret_cast<const uint4*>(
          page + (kKv8 ? kCodes8Bytes : kPageBytes) + piece_off<kKv8>(key, 8 * h + r));
      if (key >= visible) x = make_uint4(0u, 0u, 0u, 0u);
      y[i][0] = x.x, y[i][1] = x.y, y[i][2] = x.z, y[i][3] = x.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kKv8) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t u = __byte_perm(y[0][i], y[1][i], o == 0 ? 0x5140 : 0x7362);
          const uint32_t v = __byte_perm(y[2][i], y[3][i], o == 0 ? 0x5140 : 0x7362);
          const uint32_t a[4] = {e4m3x2_to_f16x2<0>(u), e4m3x2_to_f16x2<1>(u), e4m3x2_to_f16x2<0>(v),
                                 e4m3x2_to_f16x2<1>(v)};
          mma_f16(st.acc[2 * i + o], a, b[0], b[1]);
        }
      } else {
        const uint32_t a[4] = {__byte_perm(y[0][i], y[1][i], 0x5410), __byte_perm(y[0][i], y[1][i], 0x7632),
                               __byte_perm(y[2][i], y[3][i], 0x5410), __byte_perm(y[2][i], y[3][i], 0x7632)};
        mma_bf16(st.acc[4 * h + i], a, b[0], b[1]);
      }
    }
  }
}

// What warps and CTAs pass on of their share of a row.
struct RowPart {
  float m[kGroup], lead[kGroup], sum[kGroup];
  float pad[2];
  float acc[kGroup][kHeadDim];
};

constexpr int kPagesWarps = 4;

// Without a suspend-time hint (see mbar_try_wait_nohint).
__device__ __forceinline__ bool mbar_wait_nohint(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < kSpinLimit; ++i)
    if (mbar_try_wait_nohint(bar, parity)) return true;
  return false;
}

// One cluster of CTAs (or one CTA) per (sequence, new token, KV head); their warps take the listed pages in
// turn, each through its own ring, and the first CTA merges.  Memory bounds it where the CTAs fill the GPU: 256
// rows of 64 bf16 pages 145 us (6.9 TB/s, the copy rate), of 64 8-bit pages 85 (0.78 of it); 48 rows of 128 8-bit
// pages are two or three CTAs per SM, 43 us (0.73).  Four warps share one row and head: with one or two each 166 and
// 150 us, 88 and 57.  Few rows are a chain of latencies: 8 rows of 16 pages 5.0 us.
template <bool kKv8>
__global__ void __launch_bounds__(kPagesWarps * 32, kKv8 ? 4 : 3)
    attend_pages_kernel(const __grid_constant__ PagesArgs a, const __grid_constant__ CUtensorMap map,
                        unsigned* status) {
  // A ring for each warp, which holds its part in the end; behind them the parts of a cluster's CTAs.
  extern __shared__ __align__(1024) uint8_t pages_smem[];
  __shared__ uint64_t bars[kPagesWarps][kMaxPageStages];
  const int ring_bytes = a.stages * kStageBytes<kKv8>;
  RowPart* peers = reinterpret_cast<RowPart*>(pages_smem + kPagesWarps * ring_bytes);
  auto part_of = [&](int w) { return reinterpret_cast<RowPart*>(pages_smem + w * ring_bytes); };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&bars[warp][i], 1);
    fence_barrier_init();
    if (!kKv8) tma_prefetch_desc(&map);
  }
  __syncwarp();
  if (a.cluster > 1) cluster_arrive_relaxed();
  // The plan was uploaded before the kernel in front of this one started.
  const int rank = blockIdx.x % a.cluster, job = blockIdx.x / a.cluster;
  const int head = job % a.num_kv, tok = job / a.num_kv % a.max_new;
  const SeqRec seq = load_seq(a.seqs, job / (a.num_kv * a.max_new));
  const bool live = tok < seq.num_new && seq.num_new <= kShortQuery;
  pdl_wait();
  pdl_trigger();
  const long long row = seq.flat_start + tok;
  const int position = seq.num_cached + tok;
  const int n = live ? position / kBlockTokens + 1 : 0;
  RowState<kKv8> st;
  st.m = st.lead = -INFINITY;
  st.sum = 0.f;
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) st.acc[t][i] = 0.f;
  if (live) {
    PageQuery<kKv8> q;
    const int* list = a.pages + (row * a.num_kv + head) * a.budget;
    uint8_t* ring = pages_smem + warp * ring_bytes;
    const uint64_t policy = l2_policy_evict_first();
    const int step = kPagesWarps * a.cluster;
    int put = 0, get = 0;  // stages that the next copy goes to and comes from
    uint32_t phase = 0;    // of `get`
    bool ok = true, loaded = false;
    for (int j0 = rank * kPagesWarps + warp; j0 < a.budget && ok; j0 += 32 * step) {
      // The blocks of the warp's next 32 pages, one per lane, those that it sees in front.
      const int j = j0 + lane * step;
      int page = j < a.budget ? list[j] : -1;
      int block = -1;
      if (page >= 0 && page < n) {
        block = a.tables[seq.table_off + page];
        if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.num_blocks)) {
          atomicOr(status, kErrBlock);
          block = -1;
        }
      }
      const unsigned todo = __ballot_sync(0xffffffffu, block >= 0);
      const int count = __popc(todo);
      if (todo & (todo + 1)) {
        const int from = static_cast<int>(__fns(todo, 0, lane + 1)) & 31;
        block = __shfl_sync(0xffffffffu, block, from);
        page = __shfl_sync(0xffffffffu, page, from);
      }
      auto fetch = [&](int i) {  // the i-th of them
        const int b = __shfl_sync(0xffffffffu, block, i);
        uint64_t* bar = &bars[warp][put];
        uint8_t* to = ring + put * kStageBytes<kKv8>;
        put = put + 1 == a.stages ? 0 : put + 1;
        if (lane != 0) return;
        mbar_arrive_expect_tx(bar, kStageBytes<kKv8>);
        if constexpr (kKv8)
          bulk_load(to, a.pool + (static_cast<long long>(b) * a.num_kv + head) * kPage8Bytes, kPage8Bytes, bar);
        else
          tma_load_5d(to, &map, bar, 0, 0, 0, head, b, policy);
      };
      auto next = [&] {
        get = get + 1 == a.stages ? 0 : get + 1;
        phase ^= get == 0;
      };
      for (int i = 0; i < min(count, a.stages); ++i) fetch(i);
      if (!loaded) {
        q.load(a.q + row * a.q_row_stride + head * kGroup * kHeadDim, a.scale_log2, lane);
        loaded = true;
      }
      for (int i = 0; i < count; ++i, next()) {
        ok = __all_sync(0xffffffffu, mbar_wait_nohint(&bars[warp][get], phase));
        if (!ok) {
          if (lane == 0) atomicOr(status, kErrTimeout);
          // No copy is in flight when the CTA ends.
          for (int o = i; o < min(count, i + a.stages); ++o, next()) mbar_wait(&bars[warp][get], phase);
          break;
        }
        const uint8_t* stage = ring + get * kStageBytes<kKv8>;
        float score[4];
        page_scores<kKv8>(q, stage, lane, score);
        page_update<kKv8>(stage, score, position - __shfl_sync(0xffffffffu, page, i) * kBlockTokens + 1, lane,
                          st);
        __syncwarp();
        if (i + a.stages < count) fetch(i + a.stages);
      }
    }
  }
  // The warp's result: sums over the lanes of a head; columns 0-1 and 2-3 of the products.
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) st.sum += __shfl_xor_sync(0xffffffffu, st.sum, off);
  __syncwarp();
  RowPart& mine = *part_of(warp);
  if ((lane & ~4) == 0) mine.m[lane >> 2] = st.m, mine.lead[lane >> 2] = st.lead, mine.sum[lane >> 2] = st.sum;
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lost = __shfl_xor_sync(0xffffffffu, st.acc[t][i], 1) * (kKv8 ? 1.f / 4096.f : 1.f);
      // An infinity among the values: what its weight lost may be zero, and zero times it NaN.
      const float both = st.acc[t][i] + lost, y = isnan(both) && !isnan(st.acc[t][i]) ? st.acc[t][i] : both;
      if ((lane & 3) == 0) mine.acc[i & 1][row_channel<kKv8>(lane >> 2, t) + (i >> 1)] = y;
    }
  __syncthreads();
  // Merges `count` parts: a thread has two neighbouring channels of a head.
  constexpr int kPer = kGroup * kHeadDim / (kPagesWarps * 32);
  const int at = threadIdx.x * kPer, g = at / kHeadDim, d = at % kHeadDim;
  float m, lead, sum, acc[kPer];
  auto merge = [&](auto of, int count) {
    m = lead = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
    for (int w = 0; w < count; ++w) m = fmaxf(m, of(w)->m[g]);
    if constexpr (kKv8)  // without keys neither: minus infinity less itself is NaN, which fmaxf passes over
      for (int w = 0; w < count; ++w) lead = fmaxf(lead, of(w)->lead[g] + (of(w)->m[g] - m));
    for (int w = 0; w < count; ++w) {
      const RowPart* p = of(w);
      float f = p->m[g] == -INFINITY ? 1.f : fast_exp2(p->m[g] - m);
      sum += p->sum[g] * f;
      if constexpr (kKv8) f = p->lead[g] == -INFINITY ? 1.f : fast_exp2(p->lead[g] + (p->m[g] - m) - lead);
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] += p->acc[g][d + i] * f;
    }
  };
  merge(part_of, kPagesWarps);
  if (a.cluster > 1) {
    cluster_wait();  // all CTAs have started
    const uint32_t to = peer_smem(smem_u32(&peers[rank]), 0);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      store_cluster(to + offsetof(RowPart, acc) + (at + i) * 4, __float_as_uint(acc[i]));
    if (d == 0) {
      store_cluster(to + offsetof(RowPart, m) + g * 4, __float_as_uint(m));
      store_cluster(to + offsetof(RowPart, lead) + g * 4, __float_as_uint(lead));
      store_cluster(to + offsetof(RowPart, sum) + g * 4, __float_as_uint(sum));
    }
    __syncwarp();
    cluster_arrive();  // and all parts have come
    cluster_wait();
    if (rank != 0) return;
    merge([&](int w) { return peers + w; }, a.cluster);
  }
  if (!live) return;
  // 2^lead in two steps: it may be beyond fp32 where the values are near the end of their range.  No key at all:
  // zero; NaN goes through.
  const float half = fast_exp2(0.5f * (kKv8 ? lead : 24.f)), part = half / sum;
  *reinterpret_cast<uint32_t*>(a.out + row * a.out_row_stride + head * kGroup * kHeadDim + at) =
      sum == 0.f ? 0u : pack_bf16(acc[0] * part * half, acc[1] * part * half);
}

}  // namespace ms
