// C-ABI entry points of sparse attention over selected pages and of whole pages (declared in
// include/msattn.h).  Included at the end of msattn.cu, whose launch helpers they use.

namespace {

constexpr int kBoundsWarps = 8;

// A layer of either kind of pool by its first byte.
int check_layer(const char* what, const void* pool, int num_blocks, int num_kv) {
  if (pool == nullptr || num_blocks <= 0 || num_kv <= 0) {
    set_error(std::string(what) + ": null pointer or empty pool");
    return MS_ERR_ARG;
  }
  if (!aligned(pool, 16)) {
    set_error(std::string(what) + ": the layer must be 16-byte aligned");
    return MS_ERR_LAYOUT;
  }
  return MS_OK;
}

template <int kThreads>
using Threads = std::integral_constant<int, kThreads>;

// As many neighbouring heads per item as a CTA has warps for, and pages for the warps that are left.
ms::ScoreShape score_shape(int num_kv) {
  ms::ScoreShape shape;
  shape.heads = std::min(num_kv, ms::kScoreWarps);
  while (num_kv % shape.heads) --shape.heads;
  shape.tiles = ms::kScoreWarps / shape.heads;
  return shape;
}

int check_step(const char* what, const int32_t* plan_dev, const MsPlanInfo* plan) {
  if (plan != nullptr && plan_dev != nullptr && aligned(plan_dev, 16)) return MS_OK;
  set_error(std::string(what) + ": need a plan, uploaded to a 16-byte aligned address");
  return MS_ERR_ARG;
}

int check_short(const char* what, int max_new, int num_kv, const MsPlanInfo* plan, int budget) {
  if (plan->is_tree) {
    set_error(std::string(what) + ": need a plan of ms_plan_build (drafts of a tree see no run of pages)");
    return MS_ERR_ARG;
  }
  if (max_new < 1 || max_new > ms::kShortQuery || budget < 1 || budget > ms::kMaxBudget) {
    set_error(std::string(what) + ": need 1 <= max_new <= " + std::to_string(ms::kShortQuery) +
              " and 1 <= budget <= " + std::to_string(ms::kMaxBudget));
    return MS_ERR_ARG;
  }
  if (static_cast<int64_t>(plan->num_seqs) * ms::kShortQuery * num_kv > 0x7fffffffLL) {
    set_error(std::string(what) + ": plan too large for one launch");
    return MS_ERR_ARG;
  }
  return MS_OK;
}

int bounds_of_step(const char* what, bool kv8, const void* pool, int num_blocks, int num_kv,
                   const int32_t* plan_dev, const MsPlanInfo* plan, void* bounds, void* stream) {
  int rc = check_layer(what, pool, num_blocks, num_kv);
  if (rc == MS_OK) rc = check_step(what, plan_dev, plan);
  if (rc) return rc;
  if (bounds == nullptr || !aligned(bounds, 16)) {
    set_error(std::string(what) + ": bounds must be 16-byte aligned");
    return MS_ERR_ARG;
  }
  if (plan->num_seqs <= 0) return MS_OK;
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  ms::BoundsArgs a = {};
  a.pool = static_cast<const uint8_t*>(pool);
  a.bounds = static_cast<uint8_t*>(bounds);
  a.seqs = plan_dev + plan->off_seqs;
  a.tables = plan_dev + plan->off_tables;
  a.num = plan->num_seqs;
  a.num_kv = num_kv;
  a.num_blocks = num_blocks;
  // CTAs of a sequence: enough for its pages if it had all the new tokens, but no more than fill the GPU
  // eight times over when every sequence has as many.
  const int64_t pages = plan->num_tokens / ms::kBlockTokens + 2;
  const int64_t most = (pages * num_kv + kBoundsWarps - 1) / kBoundsWarps;
  const int64_t fill = std::max<int64_t>(1, static_cast<int64_t>(8) * sms / plan->num_seqs);
  const dim3 grid(plan->num_seqs, static_cast<unsigned>(std::min<int64_t>({most, fill, 65535})));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      kv8 ? launch(ms::key_bounds_step_kernel<true, kBoundsWarps>, grid, kBoundsWarps * 32, 0, s, a, st)
          : launch(ms::key_bounds_step_kernel<false, kBoundsWarps>, grid, kBoundsWarps * 32, 0, s, a, st);
  if (e != cudaSuccess) return cuda_fail((std::string(what) + " launch").c_str(), e);
  return MS_OK;
}

int bounds_of_blocks(const char* what, bool kv8, const void* pool, int num_blocks, int num_kv,
                     const int64_t* blocks, const int64_t* rows, int count, void* bounds, void* stream) {
  int rc = check_layer(what, pool, num_blocks, num_kv);
  if (rc) return rc;
  if (count < 0 || (count > 0 && (!blocks || !rows)) || bounds == nullptr || !aligned(bounds, 16)) {
    set_error(std::string(what) + ": null pointer, negative count, or bounds not 16-byte aligned");
    return MS_ERR_ARG;
  }
  if (count == 0) return MS_OK;
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  ms::BoundsArgs a = {};
  a.pool = static_cast<const uint8_t*>(pool);
  a.bounds = static_cast<uint8_t*>(bounds);
  a.blocks = reinterpret_cast<const long long*>(blocks);
  a.rows = reinterpret_cast<const long long*>(rows);
  a.num = count;
  a.num_kv = num_kv;
  a.num_blocks = num_blocks;
  const int64_t ctas = (static_cast<int64_t>(count) * num_kv + kBoundsWarps - 1) / kBoundsWarps;
  if (ctas > 0x7fffffffLL) {
    set_error(std::string(what) + ": too many blocks");
    return MS_ERR_ARG;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(ctas);
  const cudaError_t e =
      kv8 ? launch(ms::key_bounds_kernel<true, kBoundsWarps>, grid, kBoundsWarps * 32, 0, s, a, st)
          : launch(ms::key_bounds_kernel<false, kBoundsWarps>, grid, kBoundsWarps * 32, 0, s, a, st);
  if (e != cudaSuccess) return cuda_fail((std::string(what) + " launch").c_str(), e);
  return MS_OK;
}

int attend_selected(const char* what, bool kv8, const void* q, int64_t q_row_stride, void* out,
                    int64_t out_row_stride, int num_heads, int num_kv, const void* pool, int num_blocks,
                    const int32_t* plan_dev, const MsPlanInfo* plan, int max_new, const int32_t* pages,
                    int budget, float scale, void* stream) {
  int rc = check_layer(what, pool, num_blocks, num_kv);
  if (rc == MS_OK)
    rc = check_attention(what, q, q_row_stride, out, out_row_stride, num_heads, num_kv, plan_dev, plan,
                         nullptr, 0, 0, 0, scale);
  if (rc == MS_OK) rc = check_short(what, max_new, num_kv, plan, budget);
  if (rc) return rc;
  if (pages == nullptr) {
    set_error(std::string(what) + ": null pointer");
    return MS_ERR_ARG;
  }
  if (plan->num_seqs <= 0) return MS_OK;
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  ms::PagesArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_row_stride = q_row_stride;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_row_stride = out_row_stride;
  a.pool = static_cast<const uint8_t*>(pool);
  a.seqs = plan_dev + plan->off_seqs;
  a.tables = plan_dev + plan->off_tables;
  a.pages = pages;
  a.max_new = max_new;
  a.num_kv = num_kv;
  a.num_blocks = num_blocks;
  a.budget = budget;
  a.scale_log2 = scale * 1.4426950408889634f;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap map = {};
  if (!kv8) rc = kv_tensor_map(pool, num_blocks, num_kv, 0, &map);
  if (rc == MS_OK) rc = ensure_smem_attrs();
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  // A row and head is shared by more CTAs, as a cluster, while they all fit two per SM and a warp has two pages
  // (measured: 24 of 128 bf16 pages 21 us with one CTA each, 8.4 with eight; 64 of 300 8-bit pages 57 and 28
  // with four; 128 of 64 bf16 pages 14.4 and 15.4 with two).
  const int64_t units = static_cast<int64_t>(plan->num_seqs) * max_new * num_kv;
  a.cluster = 1;
  while (a.cluster < ms::kMaxCluster && units * a.cluster * 2 <= 2 * sms &&
         budget >= 2 * 2 * a.cluster * ms::kPagesWarps)
    a.cluster *= 2;
  // 8-bit: rings of four pages leave room for three CTAs per SM, of three for four.  CTAs that three per SM hold
  // spread better (384 of 128 pages: 43 us, 51 with four per SM); more of them want four (2048 of 64: 92 and 85).
  const int64_t ctas = units * a.cluster;
  a.stages = !kv8 ? 2 : ctas <= 3 * sms ? 4 : 3;
  const size_t smem = ms::kPagesWarps * a.stages * (kv8 ? ms::kStageBytes<true> : ms::kStageBytes<false>) +
                      (a.cluster > 1 ? sizeof(ms::RowPart) * ms::kMaxCluster : 0);
  auto go = [&](auto kernel) {
    const unsigned grid = static_cast<unsigned>(ctas);
    return a.cluster > 1 ? launch_clusters(kernel, grid, a.cluster, ms::kPagesWarps * 32, smem, s, a, map, st)
                         : launch(kernel, grid, ms::kPagesWarps * 32, smem, s, a, map, st);
  };
  const cudaError_t e = kv8 ? go(ms::attend_pages_kernel<true>) : go(ms::attend_pages_kernel<false>);
  if (e != cudaSuccess) return cuda_fail((std::string(what) + " launch").c_str(), e);
  return MS_OK;
}

}  // namespace

extern "C" int ms_key_bounds_step(const void* k_cache, int32_t num_blocks, int32_t num_kv_heads,
                                  const int32_t* plan_dev, const MsPlanInfo* plan, void* bounds,
                                  void* stream) {
  return bounds_of_step("ms_key_bounds_step", false, k_cache, num_blocks, num_kv_heads, plan_dev, plan,
                        bounds, stream);
}

extern "C" int ms_key_bounds_step_kv8(const void* pool, int32_t num_blocks, int32_t num_kv_heads,
                                      const int32_t* plan_dev, const MsPlanInfo* plan, void* bounds,
                                      void* stream) {
  return bounds_of_step("ms_key_bounds_step_kv8", true, pool, num_blocks, num_kv_heads, plan_dev, plan,
                        bounds, stream);
}

extern "C" int ms_key_bounds(const void* k_cache, int32_t num_blocks, int32_t num_kv_heads,
                             const int64_t* blocks, const int64_t* rows, int32_t count, void* bounds,
                             void* stream) {
  return bounds_of_blocks("ms_key_bounds", false, k_cache, num_blocks, num_kv_heads, blocks, rows, count,
                          bounds, stream);
}

extern "C" int ms_key_bounds_kv8(const void* pool, int32_t num_blocks, int32_t num_kv_heads,
                                 const int64_t* blocks, const int64_t* rows, int32_t count, void* bounds,
                                 void* stream) {
  return bounds_of_blocks("ms_key_bounds_kv8", true, pool, num_blocks, num_kv_heads, blocks, rows, count,
                          bounds, stream);
}

extern "C" int64_t ms_select_workspace_bytes(int32_t num_seqs, int32_t max_new, int32_t max_pages,
                                             int32_t num_kv_heads) {
  const int64_t pages = (static_cast<int64_t>(max_pages) + 63) / 64 * 64;
  return static_cast<int64_t>(num_seqs) * max_new * num_kv_heads * (pages + pages / ms::kTilePages) * 4;
}

extern "C" int ms_select_pages(const void* q, int64_t q_row_stride, int32_t num_heads,
                               int32_t num_kv_heads, const void* bounds, int32_t num_blocks,
                               const int32_t* plan_dev, const MsPlanInfo* plan, int32_t max_new,
                               int32_t max_pages, int32_t budget, int32_t first, int32_t last,
                               int32_t* pages, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "ms_select_pages";
  int rc = check_layer(what, bounds, num_blocks, num_kv_heads);
  if (rc == MS_OK) rc = check_step(what, plan_dev, plan);
  if (rc == MS_OK) rc = check_short(what, max_new, num_kv_heads, plan, budget);
  if (rc) return rc;
  if (num_heads != ms::kGroup * num_kv_heads || !q || !pages || !aligned(q, 16) ||
      q_row_stride < num_heads * ms::kHeadDim || q_row_stride % 8) {
    set_error("ms_select_pages: need num_heads == 2 * num_kv_heads, q rows 16-byte aligned, pages");
    return MS_ERR_ARG;
  }
  if (first < 0 || last < 1 || first > budget - last) {
    set_error("ms_select_pages: need first >= 0, last >= 1 and first + last <= budget");
    return MS_ERR_ARG;
  }
  if (max_pages < 1 || max_pages > ms::kMaxSelectPages) {
    set_error("ms_select_pages: rows see 1 to " + std::to_string(ms::kMaxSelectPages) + " pages, not " +
              std::to_string(max_pages));
    return MS_ERR_ARG;
  }
  if (plan->num_seqs <= 0) return MS_OK;
  max_pages = (max_pages + 63) / 64 * 64;
  const int64_t rows = static_cast<int64_t>(plan->num_seqs) * max_new * num_kv_heads;
  const int64_t need = ms_select_workspace_bytes(plan->num_seqs, max_new, max_pages, num_kv_heads);
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)) {
    set_error("ms_select_pages: workspace of " + std::to_string(need) + " bytes (16-byte aligned) required");
    return MS_ERR_ARG;
  }
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  rc = ensure_smem_attrs();
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  ms::SelectArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_row_stride = q_row_stride;
  a.bounds = static_cast<const uint8_t*>(bounds);
  a.seqs = plan_dev + plan->off_seqs;
  a.tables = plan_dev + plan->off_tables;
  a.pages = pages;
  a.max_new = max_new;
  a.num_kv = num_kv_heads;
  a.num_blocks = num_blocks;
  a.budget = budget;
  a.first = first;
  a.last = last;
  a.capacity = max_pages;
  a.scores = static_cast<float*>(workspace);
  a.sums = reinterpret_cast<uint32_t*>(a.scores + rows * max_pages);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(plan->num_seqs * max_new * num_kv_heads);
  const size_t smem = 4 * (static_cast<size_t>(max_pages) + 2 * ((max_pages + 31) / 32));
  auto select = [&](auto threads, auto with_scores) {
    return launch(ms::select_pages_kernel<threads.value, with_scores.value>, grid, threads.value, smem, s, a, st);
  };
  cudaError_t e = cudaSuccess;
  if (max_pages > budget && max_pages <= 256 && grid <= 256) {
    // Few rows of few pages in one launch.  Measured with one launch and with two, on the device: 64 rows and heads of
    // 128 pages 5.7 and 9.4 us (on the host 10.7 and 13.0), 256 of 256 pages 11.8 and 15.2; beyond the border 512 of
    // 256 pages 23.0 and 21.8, 1024 of 128 29.4 and 22.9, 128 of 512 15.0 and 15.2.
    e = select(Threads<256>(), std::true_type());
    if (e != cudaSuccess) return cuda_fail("select_pages launch", e);
    return MS_OK;
  }
  ms::ScoreArgs score;
  score.s = a;
  score.shape = score_shape(num_kv_heads);
  score.num_seqs = plan->num_seqs;
  const size_t ring = static_cast<size_t>(ms::kScoreStages) * score.shape.stage_bytes();
  if (max_pages > budget && budget > first + last)
    e = max_new <= 4 ? launch(ms::score_pages_kernel<1>, sms, (ms::kScoreWarps + 1) * 32, ring, s, score, st)
                     : launch(ms::score_pages_kernel<2>, sms, (ms::kScoreWarps + 1) * 32, ring, s, score, st);
  if (e != cudaSuccess) return cuda_fail("score_pages launch", e);
  // Threads of a row and head: as many as fill the GPU with 131072 (measured with 32 to 1024: 10240 rows of
  // 156 pages take 50 us with 32 and 117 with 256, 24 of 6250 take 17 with 1024 and 21 with 256), but not more
  // than it has pages.
  const int64_t threads = std::min<int64_t>(131072 / grid, max_pages);
  const std::false_type scored;
  e = threads >= 1024  ? select(Threads<1024>(), scored)
      : threads >= 512 ? select(Threads<512>(), scored)
      : threads >= 256 ? select(Threads<256>(), scored)
      : threads >= 128 ? select(Threads<128>(), scored)
      : threads >= 64  ? select(Threads<64>(), scored)
                       : select(Threads<32>(), scored);
  if (e != cudaSuccess) return cuda_fail("select_pages launch", e);
  return MS_OK;
}

extern "C" int ms_attend_pages(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                               int32_t num_heads, int32_t num_kv_heads, const void* k_cache,
                               const void* v_cache, int32_t num_blocks, const int32_t* plan_dev,
                               const MsPlanInfo* plan, int32_t max_new, const int32_t* pages,
                               int32_t budget, float scale, void* stream) {
  const int rc = check_pool(k_cache, v_cache, num_blocks, num_kv_heads);
  if (rc) return rc;
  return attend_selected("ms_attend_pages", false, q, q_row_stride, out, out_row_stride, num_heads,
                         num_kv_heads, k_cache, num_blocks, plan_dev, plan, max_new, pages, budget, scale,
                         stream);
}

extern "C" int ms_attend_pages_kv8(const void* q, int64_t q_row_stride, void* out,
                                   int64_t out_row_stride, int32_t num_heads, int32_t num_kv_heads,
                                   const void* pool, int32_t num_blocks, const int32_t* plan_dev,
                                   const MsPlanInfo* plan, int32_t max_new, const int32_t* pages,
                                   int32_t budget, float scale, void* stream) {
  return attend_selected("ms_attend_pages_kv8", true, q, q_row_stride, out, out_row_stride, num_heads,
                         num_kv_heads, pool, num_blocks, plan_dev, plan, max_new, pages, budget, scale,
                         stream);
}

// ---- whole pages -----------------------------------------------------------------------------------

namespace {

// Bits of the blocks that a call's lists name; grows with the largest pool seen, and every call leaves
// it zero.
struct PageBits {
  std::vector<uint64_t> words;
  void room(int num_blocks) {
    const size_t need = (static_cast<size_t>(num_blocks) + 63) / 64;
    if (words.size() < need) words.resize(need, 0);
  }
  bool test(int b) const { return words[b >> 6] >> (b & 63) & 1u; }
  void set(int b) { words[b >> 6] |= uint64_t(1) << (b & 63); }
  void clear(const int32_t* list, int n) {
    for (int i = 0; i < n; ++i) words[list[i] >> 6] = 0;
  }
};

template <bool kCopy, int kMax>
cudaError_t launch_pages(const ms::PageArgs& a, int layers, const int32_t* src, const int32_t* dst,
                         cudaStream_t s) {
  ms::PageList<kMax> list;
  std::memcpy(list.dst, dst, sizeof(int32_t) * a.count);
  if (kCopy) std::memcpy(list.src, src, sizeof(int32_t) * a.count);
  return launch(ms::pages_kernel<kCopy, kMax>, dim3(a.count * a.pieces, layers), 256, 0, s, a, list);
}

template <bool kCopy>
int move_pages(const char* what, void* base, int64_t layer_stride, int64_t page_bytes, int layers,
               int num_blocks, const int32_t* src, const int32_t* dst, int count, void* stream) {
  if (base == nullptr || layers < 0 || num_blocks <= 0 || count < 0 || page_bytes <= 0 ||
      page_bytes % 16 || layer_stride % 16 || !aligned(base, 16) ||
      (layers > 1 && layer_stride / num_blocks < page_bytes) || layers > 65535 ||
      page_bytes > (int64_t(1) << 30)) {
    set_error(std::string(what) + ": null pointer, sizes, or pages that are not whole multiples of 16 "
              "bytes on 16-byte boundaries");
    return MS_ERR_ARG;
  }
  if (count > 0 && (dst == nullptr || (kCopy && src == nullptr))) {
    set_error(std::string(what) + ": null list");
    return MS_ERR_ARG;
  }
  if (count == 0 || layers == 0) return MS_OK;
  for (int i = 0; i < count; ++i)
    for (const int32_t b : {dst[i], kCopy ? src[i] : dst[i]})
      if (b < 0 || b >= num_blocks) {
        set_error(std::string(what) + ": block " + std::to_string(b) + " of a pool of " +
                  std::to_string(num_blocks));
        return MS_ERR_ARG;
      }
  if constexpr (kCopy) {  // a page that is written is neither written twice nor read
    static thread_local PageBits bits;
    try {
      bits.room(num_blocks);
    } catch (...) {
      set_error(std::string(what) + ": out of host memory");
      return MS_ERR_CAPACITY;
    }
    int bad = -1;
    for (int i = 0; i < count && bad < 0; ++i) {
      if (bits.test(dst[i])) bad = dst[i];
      bits.set(dst[i]);
    }
    for (int i = 0; i < count && bad < 0; ++i)
      if (bits.test(src[i])) bad = src[i];
    bits.clear(dst, count);
    if (bad >= 0) {
      set_error(std::string(what) + ": block " + std::to_string(bad) +
                " is written twice, or written and read, by one call");
      return MS_ERR_ARG;
    }
  }
  ms::PageArgs a;
  a.base = static_cast<uint8_t*>(base);
  a.layer_stride = layer_stride;
  a.page_bytes = page_bytes;
  a.pieces = static_cast<int>((page_bytes + ms::kPagePiece - 1) / ms::kPagePiece);
  a.piece_bytes = static_cast<int>((page_bytes / 16 + a.pieces - 1) / a.pieces * 16);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  constexpr int kFew = 32, kSome = 480, kMany = 4000;  // 256, 3840 and 32000 bytes of arguments
  const int per = static_cast<int>(std::min<int64_t>(kMany, 0x7fffffffLL / a.pieces));
  for (int at = 0; at < count; at += per) {
    a.count = std::min(per, count - at);
    const int32_t* from = kCopy ? src + at : nullptr;
    const cudaError_t e = a.count <= kFew    ? launch_pages<kCopy, kFew>(a, layers, from, dst + at, s)
                          : a.count <= kSome ? launch_pages<kCopy, kSome>(a, layers, from, dst + at, s)
                                             : launch_pages<kCopy, kMany>(a, layers, from, dst + at, s);
    if (e != cudaSuccess) return cuda_fail((std::string(what) + " launch").c_str(), e);
  }
  // Attention that starts early reads cached rows before the launch in front of it has ended, and the pages' launch
  // lets the next one start before its stores.
  return ms_kv_moved(stream);
}

}  // namespace

extern "C" int ms_copy_pages(void* base, int64_t layer_stride, int64_t page_bytes, int32_t num_layers,
                             int32_t num_blocks, const int32_t* src, const int32_t* dst, int32_t count,
                             void* stream) {
  return move_pages<true>("ms_copy_pages", base, layer_stride, page_bytes, num_layers, num_blocks, src, dst,
                          count, stream);
}

extern "C" int ms_clear_pages(void* base, int64_t layer_stride, int64_t page_bytes, int32_t num_layers,
                              int32_t num_blocks, const int32_t* blocks, int32_t count, void* stream) {
  return move_pages<false>("ms_clear_pages", base, layer_stride, page_bytes, num_layers, num_blocks,
                           nullptr, blocks, count, stream);
}
