// The 8-bit KV pool: quantising rows as they are written, reading them back, and expanding pages
// for the tensor-core prefill kernel.
//
// A row is one token's K or V of one KV head: 128 values x.  It is held as e4m3 codes c and one
// exponent byte b, and stands for c 2^(b - 127):
//   b - 127 = the smallest integer e in [-100, 120] with max|x| 2^-e <= 448 (e4m3's largest value),
//   c = e4m3(x 2^-e), ties to even (at e = 120 clamped to +-240, so that c 2^e stays a bf16 value).
// A power-of-two scale costs no precision (e4m3 is a floating-point format, only the range of small
// values moves) and makes every product exact: c 2^e is a bf16 value, so reading back rounds
// nothing, and writing a row that was read back stores the same values again.  A row with a NaN or an
// infinity gets b = 255 and zero codes, and stands for NaN (2^128 overflows to infinity, and
// infinity times a zero code is NaN, so the kernels need no extra case for it).  A zero-filled pool
// (b = 0) stands for zeros.
//
// Layout of a layer: [num_blocks][kv_heads][4128 bytes]; the 4128 bytes of a (block, head) are K's
// 16 rows of 128 codes, V's 16 rows, K's 16 exponent bytes, V's 16.  One copy of 4128 contiguous bytes brings
// everything an attention step needs, and the 16-byte chunks of row t are stored XOR-swizzled (chunk
// i at position i ^ (t % 2 + 2 (t / 4))), so the copy needs no tensor map and ldmatrix reads it
// without bank conflicts, in the order of tokens that gives a lane four neighbouring ones.
#pragma once

#include <cuda_fp16.h>

#include "norm_rope_scatter.cuh"

namespace ms {

constexpr int kRow8Bytes = kHeadDim;                          // codes of one row
constexpr int kCodes8Bytes = kBlockTokens * kRow8Bytes;       // K or V codes of a (block, head)
constexpr int kExp8Off = 2 * kCodes8Bytes;                    // exponent bytes: K's, then V's
constexpr int kPage8Bytes = kExp8Off + 2 * kBlockTokens;      // 4128
constexpr int kExpBias = 127, kExpMin = -100, kExpMax = 120;
constexpr unsigned kExpNan = 255;

// What the chunk positions of token `tok` are XORed with: distinct over the tokens 0, 1, 4, 5, 8, 9,
// 12, 13 that one ldmatrix reads, and the same for tok and tok + 2 there.
__device__ __forceinline__ int code_swizzle8(int tok) { return (tok & 1) | ((tok >> 1) & 6); }

// Byte offset of 16-byte chunk `chunk` of token `tok` inside one K or V code block.
__device__ __forceinline__ int code_off8(int tok, int chunk) {
  return tok * kRow8Bytes + ((chunk ^ code_swizzle8(tok)) << 4);
}

// Exponent byte of a row from the largest magnitude's bf16 bits (NaN and infinity >= 0x7f80).
// amax = 1.m 2^(E - 127) and 448 = 1.75 2^8, so e = E - 135, plus one when 1.m > 1.75 (m > 96).
__device__ __forceinline__ int exp_byte8(unsigned amax) {
  if (amax >= 0x7f80u) return static_cast<int>(kExpNan);
  const int e = static_cast<int>(amax >> 7) - 135 + ((amax & 127u) > 96u ? 1 : 0);
  return min(max(e, kExpMin), kExpMax) + kExpBias;
}

// 2^-(b - 127) in fp32; 0 for a NaN row (its codes become zero).
__device__ __forceinline__ float inv_scale8(int b) {
  return b == static_cast<int>(kExpNan) ? 0.f : __int_as_float((2 * kExpBias - b) << 23);
}
// 2^(b - 127): 0 for b = 0, infinity for b = 255.
__device__ __forceinline__ float scale8(int b) { return __int_as_float(b << 23); }

__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Two e4m3 codes (bits 0-7 and 8-15 of the half that kHalf names) to an f16 pair, exactly.
template <int kHalf>
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
  uint32_t r;
  if constexpr (kHalf == 0)
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
        : "=r"(r)
        : "r"(w));
  else
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
        : "=r"(r)
        : "r"(w));
  return r;
}

// Eight bf16 values to eight codes at the row's scale.  |x 2^-e| <= 448 except at the largest exponent,
// whose codes stop at 240 (256 2^120 is no bf16 value), and a NaN row's codes are zero: a branch that no
// ordinary row takes clears both cases first.
__device__ __forceinline__ uint2 quantise8(uint4 x, int b) {
  if (b >= kExpMax + kExpBias) {
    constexpr uint32_t kTop = 0x7f707f70u;  // 240 2^120
    auto fix = [&](uint32_t w) {
      if (b == static_cast<int>(kExpNan)) return 0u;
      return (w & 0x80008000u) | __vminu2(w & 0x7fff7fffu, kTop);
    };
    x = make_uint4(fix(x.x), fix(x.y), fix(x.z), fix(x.w));
  }
  const float inv = inv_scale8(b);
  auto four = [&](uint32_t w0, uint32_t w1) {
    return cvt_e4m3x4(bf16_lo(w0) * inv, bf16_hi(w0) * inv, bf16_lo(w1) * inv, bf16_hi(w1) * inv);
  };
  return make_uint2(four(x.x, x.y), four(x.z, x.w));
}

// Largest magnitudes (bf16 bits) of the even and the odd values of a lane's eight.
__device__ __forceinline__ unsigned amax8(const uint4& x) {
  return __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                  __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
}

// Four codes to four bf16 values (two words), exact; `scale` is NaN for a NaN row.
__device__ __forceinline__ void expand4(uint32_t codes, float scale, uint32_t& w0, uint32_t& w1) {
  const uint32_t h0 = e4m3x2_to_f16x2<0>(codes), h1 = e4m3x2_to_f16x2<1>(codes);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0));
  const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h1));
  w0 = pack_bf16(a.x * scale, a.y * scale);
  w1 = pack_bf16(c.x * scale, c.y * scale);
}
__device__ __forceinline__ float row_scale8(int b) {
  return b == static_cast<int>(kExpNan) ? __int_as_float(0x7fc00000) : scale8(b);
}

// Row (slot, head) of K or V: its page, then codes and exponent at fixed places.
__device__ __forceinline__ long long page8_off(long long slot, int head, int num_kv) {
  return ((slot >> 4) * num_kv + head) * kPage8Bytes;
}

// Stores one row held by the 16 lanes of a half-warp, 8 values (16 bytes of bf16) per lane.  Every
// lane of the warp calls it (the shuffles are warp-wide); `ok` says whether this half-warp's row is
// stored.
__device__ __forceinline__ void store_row8_l16(uint8_t* page, bool is_v, int tok, const uint4& x,
                                               int l16, bool ok) {
  unsigned a = amax8(x);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, off));
  const int b = exp_byte8(max(a & 0xffffu, a >> 16));
  if (!ok) return;
  const uint2 c = quantise8(x, b);
  *reinterpret_cast<uint2*>(page + (is_v ? kCodes8Bytes : 0) + code_off8(tok, l16 >> 1) +
                            (l16 & 1) * 8) = c;
  if (l16 == 0) page[kExp8Off + (is_v ? kBlockTokens : 0) + tok] = static_cast<uint8_t>(b);
}

// The same for a row held by a whole warp, 4 values (8 bytes) per lane.
__device__ __forceinline__ void store_row8_l32(uint8_t* page, bool is_v, int tok, const uint2& x,
                                               int lane) {
  unsigned a = __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, off));
  const int b = exp_byte8(max(a & 0xffffu, a >> 16));
  *reinterpret_cast<uint32_t*>(page + (is_v ? kCodes8Bytes : 0) + code_off8(tok, lane >> 2) +
                               (lane & 3) * 4) = quantise8(make_uint4(x.x, x.y, 0u, 0u), b).x;
  if (lane == 0) page[kExp8Off + (is_v ? kBlockTokens : 0) + tok] = static_cast<uint8_t>(b);
}

// Kernel A's rows into an 8-bit pool (a.k_pool is the layer's first byte).
struct Kv8Rows {
  static __device__ __forceinline__ uint8_t* page(const NormRopeArgs& a, long long slot, int head) {
    return reinterpret_cast<uint8_t*>(a.k_pool) + page8_off(slot, head, a.num_kv);
  }
  static __device__ __forceinline__ void store4(const NormRopeArgs& a, bool is_v, long long slot,
                                                int head, int lane, const uint2& x) {
    store_row8_l32(page(a, slot, head), is_v, static_cast<int>(slot & 15), x, lane);
  }
  static __device__ __forceinline__ void store8(const NormRopeArgs& a, bool is_v, long long slot,
                                                int head, int l16, const uint4& x) {
    store_row8_l16(page(a, slot, head), is_v, static_cast<int>(slot & 15), x, l16, true);
  }
};

// ---- write: kv_scatter into an 8-bit pool ----------------------------------------------------

struct Scatter8Args {
  const __nv_bfloat16* k;  // [T, KVH, 128] (row stride k_row_stride, head stride 128)
  long long k_row_stride;
  const __nv_bfloat16* v;
  long long v_row_stride;
  const long long* slots;
  uint8_t* pool;
  long long num_slots;
  int num_tokens;
  int num_kv;
};

// Which rows a warp of the row-copy kernels moves: rows r = 0 .. 2 KVH - 1 of a token are its K heads,
// then its V heads; a warp takes the same four neighbouring rows (8 lanes each) of kTokens consecutive
// tokens, so its index is divided once and its kTokens loads are in flight together.  A lane holds 16
// values of a row, dims 8 l .. + 7 of each half: the kernels are bound by the ALU pipe as much as by
// memory, and what every lane of a row computes alike (largest value, exponent, addresses) is computed
// by 8 lanes rather than 16 (16384 tokens of 8 heads written and read: 49 us with 16, 39 with 8, 0.66 of
// the copy rate; 65521 rows read: 82 and 78 us, 0.79).
struct RowGroup {
  long long t0;
  int h;
  bool is_v;
  int cnt;  // tokens; 0 for rows past the token's last one (the shuffles are warp-wide)
};
__device__ __forceinline__ RowGroup row_group(unsigned warp, int lane, int num_kv, int num_tokens,
                                              int tokens) {
  const unsigned groups = (2u * num_kv + 3u) / 4u;
  const unsigned tg = warp / groups;
  const int r = 4 * static_cast<int>(warp - tg * groups) + (lane >> 3);
  RowGroup g;
  g.t0 = static_cast<long long>(tg) * tokens;
  g.is_v = r >= num_kv;
  g.h = g.is_v ? r - num_kv : r;
  const long long left = num_tokens - g.t0;
  g.cnt = r < 2 * num_kv && left > 0 ? static_cast<int>(min(left, static_cast<long long>(tokens))) : 0;
  return g;
}

// kVec16: rows are 16-byte aligned; else each lane loads 8-byte words.
template <int kWarps, int kTokens, bool kVec16>
__global__ void __launch_bounds__(kWarps * 32) kv_scatter8_kernel(const Scatter8Args a,
                                                                  unsigned* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, l8 = lane & 7;
  const RowGroup g = row_group(blockIdx.x * kWarps + (threadIdx.x >> 5), lane, a.num_kv, a.num_tokens,
                               kTokens);
  const long long stride = g.is_v ? a.v_row_stride : a.k_row_stride;
  const __nv_bfloat16* src = (g.is_v ? a.v : a.k) + g.t0 * stride + g.h * kHeadDim + l8 * 8;
  uint4 x[kTokens][2];
  long long slot[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    slot[i] = -1;
    if (i >= g.cnt) continue;
    slot[i] = a.slots[g.t0 + i];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const __nv_bfloat16* at = src + i * stride + p * (kHeadDim / 2);
      if constexpr (kVec16) {
        x[i][p] = *reinterpret_cast<const uint4*>(at);
      } else {
        const uint2 lo = *reinterpret_cast<const uint2*>(at);
        const uint2 hi = *reinterpret_cast<const uint2*>(at + 4);
        x[i][p] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    const bool ok = slot[i] >= 0 && slot[i] < a.num_slots;
    if (i < g.cnt && !ok && l8 == 0) atomicOr(status, kErrSlot);
    unsigned m = __vmaxu2(amax8(x[i][0]), amax8(x[i][1]));
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, off));
    const int b = exp_byte8(max(m & 0xffffu, m >> 16));
    if (!ok) continue;
    const int tok = static_cast<int>(slot[i] & 15);
    uint8_t* page = a.pool + page8_off(slot[i], g.h, a.num_kv);
    uint8_t* codes = page + (g.is_v ? kCodes8Bytes : 0) + (l8 & 1) * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *reinterpret_cast<uint2*>(codes + code_off8(tok, 4 * p + (l8 >> 1))) = quantise8(x[i][p], b);
    if (l8 == 0) page[kExp8Off + (g.is_v ? kBlockTokens : 0) + tok] = static_cast<uint8_t>(b);
  }
}

// ---- read back: kv_gather ---------------------------------------------------------------------

struct GatherArgs {
  const long long* slots;
  const void* pool;  // k_cache (bf16 layout) or the 8-bit layer
  long long block_stride, head_stride;  // bf16 pool, elements
  long long num_slots;
  __nv_bfloat16* k;
  long long k_row_stride;
  __nv_bfloat16* v;
  long long v_row_stride;
  int num_tokens;
  int num_kv;
};

// Rows by slot to [T, KVH, 128] bf16; a slot outside the pool reads as zeros and sets the status bit.
template <bool kKv8, int kWarps, int kTokens>
__global__ void __launch_bounds__(kWarps * 32) kv_gather_kernel(const GatherArgs a,
                                                                unsigned* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, l8 = lane & 7;
  const RowGroup g = row_group(blockIdx.x * kWarps + (threadIdx.x >> 5), lane, a.num_kv, a.num_tokens,
                               kTokens);
  long long slot[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) slot[i] = i < g.cnt ? a.slots[g.t0 + i] : 0;
  uint4 x[kTokens][2];
  int b[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    b[i] = 0;
    if (i >= g.cnt) continue;
    if (slot[i] < 0 || slot[i] >= a.num_slots) {
      if (l8 == 0) atomicOr(status, kErrSlot);
      continue;
    }
    if constexpr (kKv8) {
      const uint8_t* page =
          static_cast<const uint8_t*>(a.pool) + page8_off(slot[i], g.h, a.num_kv);
      const int tok = static_cast<int>(slot[i] & 15);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint2 c = *reinterpret_cast<const uint2*>(page + (g.is_v ? kCodes8Bytes : 0) +
                                                        code_off8(tok, 4 * p + (l8 >> 1)) +
                                                        (l8 & 1) * 8);
        x[i][p].x = c.x;
        x[i][p].y = c.y;
      }
      b[i] = page[kExp8Off + (g.is_v ? kBlockTokens : 0) + tok];
    } else {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        x[i][p] = *reinterpret_cast<const uint4*>(
            static_cast<const __nv_bfloat16*>(a.pool) + (g.is_v ? 2 * kBlockTokens * 64 : 0) +
            pool_offset(slot[i], g.h, p * (kHeadDim / 2) + l8 * 8, a.block_stride, a.head_stride));
    }
  }
  const long long stride = g.is_v ? a.v_row_stride : a.k_row_stride;
  __nv_bfloat16* dst = (g.is_v ? a.v : a.k) + g.t0 * stride + g.h * kHeadDim + l8 * 8;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (i >= g.cnt) break;
    const float scale = row_scale8(b[i]);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint4 y = x[i][p];
      if constexpr (kKv8) {
        expand4(x[i][p].x, scale, y.x, y.y);
        expand4(x[i][p].y, scale, y.z, y.w);
      }
      *reinterpret_cast<uint4*>(dst + i * stride + p * (kHeadDim / 2)) = y;
    }
  }
}

// ---- pages for the tensor-core prefill kernel ---------------------------------------------------

// Workspace block w = the bf16 pool layout of 8-bit block map[w], one CTA of 8 warps per (w, head):
// the prefill kernel reads each key block once per 64-token query tile, so expanding its pages once
// costs less than expanding them in every CTA (a page: 4 KiB read, 8 KiB written; two chunks of 1000
// tokens over 512 cached ones: 41 us, 35 over a bf16 pool).
__global__ void __launch_bounds__(256) kv8_expand_kernel(const uint8_t* pool, const int* map,
                                                         int num_kv, int num_blocks,
                                                         __nv_bfloat16* out, unsigned* status) {
  pdl_wait();
  pdl_trigger();
  const int w = blockIdx.x / num_kv, h = blockIdx.x - w * num_kv;
  const int blk = map[w];
  const bool ok = static_cast<unsigned>(blk) < static_cast<unsigned>(num_blocks);
  if (!ok && threadIdx.x == 0) atomicOr(status, kErrBlock);
  const uint8_t* page =
      pool + (static_cast<long long>(ok ? blk : 0) * num_kv + h) * kPage8Bytes;
  uint8_t* dst = reinterpret_cast<uint8_t*>(out) + static_cast<long long>(blockIdx.x) * kPageKVBytes;
  const int l16 = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // K, then V: 16 half-warps, one row each
    const int tok = threadIdx.x >> 4;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (ok) {
      const uint2 c = *reinterpret_cast<const uint2*>(page + i * kCodes8Bytes +
                                                      code_off8(tok, l16 >> 1) + (l16 & 1) * 8);
      const float s = row_scale8(page[kExp8Off + i * kBlockTokens + tok]);
      expand4(c.x, s, x.x, x.y);
      expand4(c.y, s, x.z, x.w);
    }
    *reinterpret_cast<uint4*>(dst + i * kPageBytes + (l16 >> 3) * (kPageBytes / 2) + tok * 128 +
                              (l16 & 7) * 16) = x;
  }
}

}  // namespace ms
