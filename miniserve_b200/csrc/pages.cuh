// Whole pages of a paged tensor [layers][num_blocks][page_bytes]: copied to other places, or filled with
// zeros, in every layer by one launch.
//
// The lists come as kernel arguments (a launch carries up to 32 KiB of them), since a host that manages
// pages has them at hand: no copy to the device, nothing that a captured graph would have to keep alive.
// Memory bounds both: a page is read once and written once (1000 bf16 pages of 8 layers and 8 heads, 1.05 GB: 162 us, 0.99
// of the copy rate; 2000 8-bit pages cleared, 0.53 GB: 75 us).  One page copied three times in 28 layers takes 3.3 us.
// Either with the ordered launch that follows it, about 1 us of it.
#pragma once

#include "ms_common.cuh"

namespace ms {

// kMax pairs (pages to clear: kMax destinations and no sources).
template <int kMax>
struct PageList {
  int dst[kMax];
  int src[kMax];
};

struct PageArgs {
  uint8_t* base;
  long long layer_stride;  // bytes
  long long page_bytes;    // a multiple of 16
  int pieces;              // of a page: one CTA each
  int piece_bytes;         // a multiple of 16, at most kPagePiece: a page's pieces are as even as they can be
  int count;
};

constexpr int kPagePiece = 16384;  // bytes that a CTA moves, at most

// Grid: x = (entry, piece), y = layer.
template <bool kCopy, int kMax>
__global__ void __launch_bounds__(256) pages_kernel(const __grid_constant__ PageArgs a,
                                                    const __grid_constant__ PageList<kMax> list) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x / a.pieces;
  const long long from = static_cast<long long>(blockIdx.x - i * a.pieces) * a.piece_bytes;
  const int n = static_cast<int>(min(static_cast<long long>(a.piece_bytes), a.page_bytes - from)) / 16;
  uint8_t* layer = a.base + blockIdx.y * a.layer_stride + from;
  uint4* dst = reinterpret_cast<uint4*>(layer + list.dst[i] * a.page_bytes);
  const uint4* src = reinterpret_cast<const uint4*>(layer + (kCopy ? list.src[i] * a.page_bytes : 0));
  uint4 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + 256 * k;
    x[k] = make_uint4(0u, 0u, 0u, 0u);
    if (kCopy && at < n) x[k] = src[at];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + 256 * k;
    if (at < n) dst[at] = x[k];
  }
}

}  // namespace ms
