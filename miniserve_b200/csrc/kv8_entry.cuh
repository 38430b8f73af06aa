// C-ABI entry points of the 8-bit pool, of reading rows back, and of attention over drafted token
// trees (declared in include/msattn.h).  Included at the end of msattn.cu, whose launch helpers and
// kernels they use.

namespace {

int check_pool8(const char* what, const void* pool, int num_blocks, int num_kv) {
  if (pool == nullptr || num_blocks <= 0 || num_kv <= 0) {
    set_error(std::string(what) + ": null pointer or empty pool");
    return MS_ERR_ARG;
  }
  if (!aligned(pool, 16)) {
    set_error(std::string(what) + ": the 8-bit layer must be 16-byte aligned");
    return MS_ERR_LAYOUT;
  }
  return MS_OK;
}

// Grid of the row-copy kernels (see row_group): a warp takes 4 tokens where that leaves every SM enough
// warps, else one, so that a decode step's few rows spread over more SMs.
constexpr int kCopyWarps = 8;
constexpr int64_t kMaxCopyWarps = int64_t(1) << 31;  // warp indices are 32-bit
template <typename Few, typename Many>
cudaError_t launch_rows(int64_t tokens, int num_kv, int sms, Few few, Many many) {
  const int64_t groups = (2 * static_cast<int64_t>(num_kv) + 3) / 4;
  const int64_t w4 = (tokens + 3) / 4 * groups, w1 = tokens * groups;
  if (w4 >= static_cast<int64_t>(16) * sms)
    return many(static_cast<unsigned>((w4 + kCopyWarps - 1) / kCopyWarps));
  return few(static_cast<unsigned>((w1 + kCopyWarps - 1) / kCopyWarps));
}

int check_attention(const char* what, const void* q, int64_t q_row_stride, const void* out,
                    int64_t out_row_stride, int num_heads, int num_kv, const int32_t* plan_dev,
                    const MsPlanInfo* plan, const void* workspace, int64_t workspace_bytes,
                    int64_t need, int64_t most_items, float scale) {
  if (plan == nullptr || num_kv <= 0 || num_heads != ms::kGroup * num_kv) {
    set_error(std::string(what) + ": need a plan and num_heads == 2 * num_kv_heads > 0");
    return MS_ERR_ARG;
  }
  if (!(scale > 0.f) || scale > 3e38f) {
    set_error(std::string(what) + ": scale must be positive and finite");
    return MS_ERR_ARG;
  }
  if (!q || !out || !plan_dev || q_row_stride < num_heads * ms::kHeadDim ||
      out_row_stride < num_heads * ms::kHeadDim || q_row_stride % 8 || out_row_stride % 8 ||
      !aligned(q, 16) || !aligned(out, 16) || !aligned(plan_dev, 16)) {
    set_error(std::string(what) + ": null pointer, or q/out rows not 16-byte aligned");
    return MS_ERR_ARG;
  }
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))) {
    set_error(std::string(what) + ": workspace of " + std::to_string(need) +
              " bytes (16-byte aligned) required");
    return MS_ERR_ARG;
  }
  if (most_items * num_kv > 0x7fffffffLL ||
      static_cast<int64_t>(plan->n_combine) * num_kv > 0x7fffffffLL) {
    set_error(std::string(what) + ": plan too large for one launch");
    return MS_ERR_ARG;
  }
  return MS_OK;
}

// A plan of ms_tree_plan_build.
int check_tree_plan(const char* what, const MsPlanInfo* plan) {
  if (plan != nullptr && plan->is_tree) return MS_OK;
  set_error(std::string(what) + ": need a plan of ms_tree_plan_build");
  return MS_ERR_ARG;
}

ms::AttnArgs attn_args(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                       int num_kv, int num_blocks, const int32_t* plan_dev, const MsPlanInfo* plan,
                       void* workspace, int64_t part_rows, float scale) {
  ms::AttnArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_row_stride = q_row_stride;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_row_stride = out_row_stride;
  a.seqs = plan_dev + plan->off_seqs;
  a.tables = plan_dev + plan->off_tables;
  a.items = nullptr;
  a.n_items = 0;
  a.num_kv = num_kv;
  a.num_blocks = num_blocks;
  float* ws = static_cast<float*>(workspace);
  a.ws_o = ws;
  a.ws_lse = ws != nullptr ? ws + part_rows * num_kv * ms::kHeadDim : nullptr;
  a.scale_log2 = scale * 1.4426950408889634f;
  return a;
}

// Where a packed plan holds kernel F's work.
struct RowsWork {
  int32_t n_narrow, off_narrow, n_wide, off_wide, off_combine;
  int64_t part_rows;  // of all partials in the workspace; the arrival counters lie behind them
};

// Kernel F over the narrow tiles and the wide ones.  behind: see RowsArgs; the wide tiles never depend on
// the narrow ones.
template <bool kKv8, bool kTree>
cudaError_t launch_rows_attention(const ms::AttnArgs& a, const void* pool, const CUtensorMap& map,
                                  const int32_t* plan_dev, const RowsWork& w, bool behind,
                                  cudaStream_t s) {
  ms::RowsArgs r;
  r.a = a;
  r.pool = static_cast<const uint8_t*>(pool);
  r.plan = plan_dev;
  r.combines = plan_dev + w.off_combine;
  r.arrived = a.ws_lse != nullptr ? reinterpret_cast<unsigned*>(a.ws_lse + w.part_rows * a.num_kv) : nullptr;
  r.behind = behind;
  cudaError_t e = cudaSuccess;
  if (w.n_narrow > 0) {
    using Cfg = ms::RowsCfg<kKv8, 1>;
    r.a.items = plan_dev + w.off_narrow;
    r.a.n_items = w.n_narrow;
    e = launch(ms::rows_attn_kernel<kKv8, kTree, 1>, static_cast<unsigned>(w.n_narrow * a.num_kv),
               Cfg::kThreads, Cfg::kSmemBytes, s, map, r);
    r.behind = 1;
  }
  if (e == cudaSuccess && w.n_wide > 0) {
    using Cfg = ms::RowsCfg<kKv8, 2>;
    r.a.items = plan_dev + w.off_wide;
    r.a.n_items = w.n_wide;
    e = launch(ms::rows_attn_kernel<kKv8, kTree, 2>, static_cast<unsigned>(w.n_wide * a.num_kv),
               Cfg::kThreads, Cfg::kSmemBytes, s, map, r);
  }
  return e;
}

}  // namespace

extern "C" int ms_kv_scatter_kv8(const void* k, int64_t k_row_stride, const void* v,
                                 int64_t v_row_stride, int32_t num_tokens, int32_t num_kv_heads,
                                 const int64_t* slot_mapping, void* pool, int32_t num_blocks,
                                 void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0) {
    set_error("ms_kv_scatter_kv8: bad sizes");
    return MS_ERR_ARG;
  }
  if (num_tokens == 0) return MS_OK;
  int rc = check_pool8("ms_kv_scatter_kv8", pool, num_blocks, num_kv_heads);
  if (rc) return rc;
  const int64_t width = static_cast<int64_t>(num_kv_heads) * ms::kHeadDim;
  if (!k || !v || !slot_mapping || k_row_stride < width || v_row_stride < width ||
      k_row_stride % 4 || v_row_stride % 4 || !aligned(k, 8) || !aligned(v, 8)) {
    set_error("ms_kv_scatter_kv8: null pointer, stride or alignment");
    return MS_ERR_ARG;
  }
  if (static_cast<int64_t>(num_tokens) * num_kv_heads > kMaxCopyWarps) {
    set_error("ms_kv_scatter_kv8: batch too large");
    return MS_ERR_ARG;
  }
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  ms::Scatter8Args a;
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.k_row_stride = k_row_stride;
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.v_row_stride = v_row_stride;
  a.slots = reinterpret_cast<const long long*>(slot_mapping);
  a.pool = static_cast<uint8_t*>(pool);
  a.num_slots = static_cast<long long>(num_blocks) * ms::kBlockTokens;
  a.num_tokens = num_tokens;
  a.num_kv = num_kv_heads;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool v16 = aligned(k, 16) && aligned(v, 16) && k_row_stride % 8 == 0 && v_row_stride % 8 == 0;
  auto go = [&](auto kernel) {
    return [=](unsigned grid) { return launch(kernel, grid, kCopyWarps * 32, 0, s, a, st); };
  };
  const cudaError_t e =
      v16 ? launch_rows(num_tokens, num_kv_heads, sms, go(ms::kv_scatter8_kernel<kCopyWarps, 1, true>),
                        go(ms::kv_scatter8_kernel<kCopyWarps, 4, true>))
          : launch_rows(num_tokens, num_kv_heads, sms, go(ms::kv_scatter8_kernel<kCopyWarps, 1, false>),
                        go(ms::kv_scatter8_kernel<kCopyWarps, 4, false>));
  if (e != cudaSuccess) return cuda_fail("kv_scatter_kv8 launch", e);
  return MS_OK;
}

extern "C" int ms_qk_norm_rope_scatter_kv8(
    const void* qkv, int64_t qkv_row_stride, int32_t num_tokens, int32_t num_heads,
    int32_t num_kv_heads, const void* q_weight, const void* k_weight, float eps, const float* cos,
    const float* sin, int64_t cs_row_stride, const int64_t* positions, int64_t max_positions,
    const int64_t* slot_mapping, void* q_out, int64_t q_out_row_stride, void* pool,
    int32_t num_blocks, void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_heads != ms::kGroup * num_kv_heads) {
    set_error("ms_qk_norm_rope_scatter_kv8: need num_heads == 2 * num_kv_heads > 0, "
              "num_tokens >= 0");
    return MS_ERR_ARG;
  }
  if (num_tokens == 0) return MS_OK;
  const int rc = check_pool8("ms_qk_norm_rope_scatter_kv8", pool, num_blocks, num_kv_heads);
  if (rc) return rc;
  return norm_rope_scatter<ms::Kv8Rows>(
      "ms_qk_norm_rope_scatter_kv8", qkv, qkv_row_stride, num_tokens, num_heads, num_kv_heads,
      q_weight, k_weight, eps, cos, sin, cs_row_stride, positions, max_positions, slot_mapping,
      q_out, q_out_row_stride, pool, num_blocks, stream);
}

namespace {

template <bool kKv8>
int gather(const char* what, const int64_t* slots, int32_t num_tokens, int32_t num_kv_heads,
           const void* pool, int32_t num_blocks, void* k_out, int64_t k_row_stride, void* v_out,
           int64_t v_row_stride, void* stream) {
  const int64_t width = static_cast<int64_t>(num_kv_heads) * ms::kHeadDim;
  if (!slots || !k_out || !v_out || k_row_stride < width || v_row_stride < width ||
      k_row_stride % 8 || v_row_stride % 8 || !aligned(k_out, 16) || !aligned(v_out, 16)) {
    set_error(std::string(what) + ": null pointer, or k/v rows not 16-byte aligned");
    return MS_ERR_ARG;
  }
  if (static_cast<int64_t>(num_tokens) * num_kv_heads > kMaxCopyWarps) {
    set_error(std::string(what) + ": batch too large");
    return MS_ERR_ARG;
  }
  int rc = MS_OK;
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  ms::GatherArgs a;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.pool = pool;
  a.head_stride = ms::kPageKVBytes / 2;
  a.block_stride = static_cast<long long>(num_kv_heads) * a.head_stride;
  a.num_slots = static_cast<long long>(num_blocks) * ms::kBlockTokens;
  a.k = static_cast<__nv_bfloat16*>(k_out);
  a.k_row_stride = k_row_stride;
  a.v = static_cast<__nv_bfloat16*>(v_out);
  a.v_row_stride = v_row_stride;
  a.num_tokens = num_tokens;
  a.num_kv = num_kv_heads;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) {
    return [=](unsigned grid) { return launch(kernel, grid, kCopyWarps * 32, 0, s, a, st); };
  };
  const cudaError_t e = launch_rows(num_tokens, num_kv_heads, sms, go(ms::kv_gather_kernel<kKv8, kCopyWarps, 1>),
                                    go(ms::kv_gather_kernel<kKv8, kCopyWarps, 4>));
  if (e != cudaSuccess) return cuda_fail((std::string(what) + " launch").c_str(), e);
  return MS_OK;
}

}  // namespace

extern "C" int ms_kv_gather(const int64_t* slots, int32_t num_tokens, int32_t num_kv_heads,
                            const void* k_cache, const void* v_cache, int32_t num_blocks,
                            void* k_out, int64_t k_row_stride, void* v_out, int64_t v_row_stride,
                            void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0) {
    set_error("ms_kv_gather: bad sizes");
    return MS_ERR_ARG;
  }
  if (num_tokens == 0) return MS_OK;
  const int rc = check_pool(k_cache, v_cache, num_blocks, num_kv_heads);
  if (rc) return rc;
  return gather<false>("ms_kv_gather", slots, num_tokens, num_kv_heads, k_cache, num_blocks, k_out,
                       k_row_stride, v_out, v_row_stride, stream);
}

extern "C" int ms_kv_gather_kv8(const int64_t* slots, int32_t num_tokens, int32_t num_kv_heads,
                                const void* pool, int32_t num_blocks, void* k_out,
                                int64_t k_row_stride, void* v_out, int64_t v_row_stride,
                                void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0) {
    set_error("ms_kv_gather_kv8: bad sizes");
    return MS_ERR_ARG;
  }
  if (num_tokens == 0) return MS_OK;
  const int rc = check_pool8("ms_kv_gather_kv8", pool, num_blocks, num_kv_heads);
  if (rc) return rc;
  return gather<true>("ms_kv_gather_kv8", slots, num_tokens, num_kv_heads, pool, num_blocks, k_out,
                      k_row_stride, v_out, v_row_stride, stream);
}

extern "C" int ms_paged_attention_kv8(const void* q, int64_t q_row_stride, void* out,
                                      int64_t out_row_stride, int32_t num_heads,
                                      int32_t num_kv_heads, const void* pool, int32_t num_blocks,
                                      const int32_t* plan_dev, const MsPlanInfo* plan,
                                      const MsKv8Info* info, void* workspace,
                                      int64_t workspace_bytes, float scale, void* stream) {
  const char* what = "ms_paged_attention_kv8";
  if (plan != nullptr && plan->is_tree) {
    set_error("ms_paged_attention_kv8: a plan of ms_tree_plan_build is for ms_tree_attention_kv8");
    return MS_ERR_ARG;
  }
  if (plan != nullptr &&
      static_cast<int64_t>(plan->n_decode_items) + plan->n_tile_items + plan->n_tc_items == 0)
    return MS_OK;
  if (plan != nullptr && (info == nullptr || info->total_ints < plan->total_ints ||
                          (plan->n_tc_items > 0 && info->n_pages <= 0))) {
    set_error("ms_paged_attention_kv8: the plan has no 8-bit part (ms_kv8_plan_build)");
    return MS_ERR_ARG;
  }
  const int64_t need = plan != nullptr ? ms_kv8_workspace_bytes(plan, info, num_kv_heads) : 0;
  int rc = check_attention(what, q, q_row_stride, out, out_row_stride, num_heads, num_kv_heads,
                           plan_dev, plan, workspace, workspace_bytes, need,
                           plan == nullptr ? 0 : std::max(std::max(info->n_narrow, info->n_wide),
                                                          plan->n_tc_items), scale);
  if (rc) return rc;
  rc = check_pool8(what, pool, num_blocks, num_kv_heads);
  if (rc) return rc;
  rc = ensure_smem_attrs();
  if (rc) return rc;
  unsigned* st = status_ptr(&rc);
  if (rc) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsWork work = {info->n_narrow,    info->off_narrow,  info->n_wide, info->off_wide,
                         info->off_combine, plan->part_rows + info->part_rows};
  ms::AttnArgs a = attn_args(q, q_row_stride, out, out_row_stride, num_kv_heads, num_blocks,
                             plan_dev, plan, workspace, work.part_rows, scale);

  // The pages of tensor-core items as a bf16 pool in the workspace, after the partials.
  void* pages = nullptr;
  CUtensorMap kmap, vmap;
  if (plan->n_tc_items > 0) {
    if (static_cast<int64_t>(info->n_pages) * num_kv_heads > 0x7fffffffLL) {
      set_error("ms_paged_attention_kv8: plan too large for one launch");
      return MS_ERR_ARG;
    }
    pages = static_cast<char*>(workspace) + need - static_cast<int64_t>(info->n_pages) * num_kv_heads *
                                                       ms::kPageKVBytes;
    rc = kv_tensor_map(pages, info->n_pages, num_kv_heads, 1, &kmap);
    if (rc) return rc;
    rc = kv_tensor_map(pages, info->n_pages, num_kv_heads, 2, &vmap);
    if (rc) return rc;
  }

  // As in ms_paged_attention: beside tensor-core work without cascade groups the bandwidth-bound
  // rows run on the side stream; with them they follow the kernel that writes the prefix partials.
  const int n_rows = work.n_narrow + work.n_wide;
  SideStream* side = nullptr;
  if (plan->n_tc_items > 0 && n_rows > 0 && plan->n_cascade == 0) side = side_stream();
  cudaStream_t ds = s;
  if (side != nullptr) {
    cudaError_t e = cudaEventRecord(side->fork, s);
    if (e == cudaSuccess) e = cudaStreamWaitEvent(side->stream, side->fork, 0);
    if (e != cudaSuccess) return cuda_fail("fork to the side stream", e);
    ds = side->stream;
  }
  auto join = [&]() -> cudaError_t {
    if (side == nullptr) return cudaSuccess;
    cudaError_t e = cudaEventRecord(side->join, ds);
    if (e == cudaSuccess) e = cudaStreamWaitEvent(s, side->join, 0);
    side = nullptr;
    return e;
  };
  if (plan->n_tc_items > 0) {
    cudaError_t e = launch(ms::kv8_expand_kernel, static_cast<unsigned>(info->n_pages * num_kv_heads),
                           256, 0, s, static_cast<const uint8_t*>(pool), plan_dev + info->off_map,
                           num_kv_heads, num_blocks, static_cast<__nv_bfloat16*>(pages), st);
    if (e == cudaSuccess) {
      ms::AttnArgs t = a;
      t.pages_fresh = 1;
      t.seqs = plan_dev + info->off_seqs;
      t.tables = plan_dev + info->off_tables;
      t.items = plan_dev + plan->off_tc;
      t.n_items = plan->n_tc_items;
      t.num_blocks = info->n_pages;
      e = launch(ms::prefill_tc_kernel, plan->n_tc_items * num_kv_heads, ms::TcCfg::kThreads,
                 ms::TcCfg::kSmemBytes, s, kmap, vmap, t);
    }
    if (e != cudaSuccess) {
      join();
      return cuda_fail("8-bit prefill launch", e);
    }
  }
  if (n_rows > 0) {
    CUtensorMap none;
    std::memset(&none, 0, sizeof(none));
    const cudaError_t e = launch_rows_attention<true, false>(a, pool, none, plan_dev, work, false, ds);
    if (e != cudaSuccess) {
      join();
      return cuda_fail("8-bit rows launch", e);
    }
  }
  {
    const cudaError_t e = join();
    if (e != cudaSuccess) return cuda_fail("join of the side stream", e);
  }
  // Kernel F merges its own splits; the tensor-core items' records are the last ones.
  MsPlanInfo tc = *plan;
  tc.off_combine += (plan->n_combine - plan->n_tc_combine) * 8;
  tc.n_combine = plan->n_tc_combine;
  return launch_combine(a, &tc, plan_dev, s);
}

extern "C" int ms_tree_attention(const void* q, int64_t q_row_stride, void* out,
                                 int64_t out_row_stride, int32_t num_heads, int32_t num_kv_heads,
                                 const void* k_cache, const void* v_cache, int32_t num_blocks,
                                 const int32_t* plan_dev, const MsPlanInfo* plan, void* workspace,
                                 int64_t workspace_bytes, float scale, void* stream) {
  const char* what = "ms_tree_attention";
  int rc = check_tree_plan(what, plan);
  if (rc) return rc;
  if (plan->n_decode_items + plan->n_tile_items == 0) return MS_OK;
  rc = check_attention(what, q, q_row_stride, out, out_row_stride, num_heads, num_kv_heads, plan_dev,
                       plan, workspace, workspace_bytes,
                       plan->workspace_bytes_per_kv_head * num_kv_heads,
                       std::max(std::max(plan->n_decode_items, plan->n_tile_items), plan->n_tc_items),
                       scale);
  if (rc) return rc;
  rc = check_pool(k_cache, v_cache, num_blocks, num_kv_heads);
  if (rc) return rc;
  rc = ensure_smem_attrs();
  if (rc) return rc;
  CUtensorMap map, kmap, vmap;
  rc = kv_tensor_map(k_cache, num_blocks, num_kv_heads, 0, &map);
  if (rc) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsWork work = {plan->n_decode_items, plan->off_decode,  plan->n_tile_items,
                         plan->off_tile,       plan->off_combine, plan->part_rows};
  const ms::AttnArgs a = attn_args(q, q_row_stride, out, out_row_stride, num_kv_heads, num_blocks,
                                   plan_dev, plan, workspace, work.part_rows, scale);
  // The cached blocks of larger trees first (see ms_tree_plan_build); kernel F merges their partials.
  cudaError_t e = cudaSuccess;
  if (plan->n_tc_items > 0) {
    rc = kv_tensor_map(k_cache, num_blocks, num_kv_heads, 1, &kmap);
    if (rc == MS_OK) rc = kv_tensor_map(k_cache, num_blocks, num_kv_heads, 2, &vmap);
    if (rc) return rc;
    ms::AttnArgs t = a;
    t.pages_fresh = 1;  // rows moved after a verify step lie below the cached length
    t.items = plan_dev + plan->off_tc;
    t.n_items = plan->n_tc_items;
    e = launch(ms::prefill_tc_kernel, plan->n_tc_items * num_kv_heads, ms::TcCfg::kThreads,
               ms::TcCfg::kSmemBytes, s, kmap, vmap, t);
  }
  if (e == cudaSuccess)
    e = launch_rows_attention<false, true>(a, nullptr, map, plan_dev, work, plan->n_tc_items > 0, s);
  if (e != cudaSuccess) return cuda_fail("tree attention launch", e);
  return MS_OK;
}

extern "C" int ms_tree_attention_kv8(const void* q, int64_t q_row_stride, void* out,
                                     int64_t out_row_stride, int32_t num_heads,
                                     int32_t num_kv_heads, const void* pool, int32_t num_blocks,
                                     const int32_t* plan_dev, const MsPlanInfo* plan,
                                     const MsKv8Info* info, void* workspace,
                                     int64_t workspace_bytes, float scale, void* stream) {
  const char* what = "ms_tree_attention_kv8";
  int rc = check_tree_plan(what, plan);
  if (rc) return rc;
  if (plan->n_decode_items + plan->n_tile_items == 0) return MS_OK;
  if (info == nullptr || info->total_ints < plan->total_ints ||
      info->n_narrow + info->n_wide == 0) {
    set_error("ms_tree_attention_kv8: the plan has no 8-bit part (ms_kv8_plan_build)");
    return MS_ERR_ARG;
  }
  rc = check_attention(what, q, q_row_stride, out, out_row_stride, num_heads, num_kv_heads, plan_dev,
                       plan, workspace, workspace_bytes,
                       ms_kv8_workspace_bytes(plan, info, num_kv_heads),
                       std::max(info->n_narrow, info->n_wide), scale);
  if (rc) return rc;
  rc = check_pool8(what, pool, num_blocks, num_kv_heads);
  if (rc) return rc;
  rc = ensure_smem_attrs();
  if (rc) return rc;
  CUtensorMap none;
  std::memset(&none, 0, sizeof(none));
  const RowsWork work = {info->n_narrow,    info->off_narrow,  info->n_wide, info->off_wide,
                         info->off_combine, plan->part_rows + info->part_rows};
  const ms::AttnArgs a = attn_args(q, q_row_stride, out, out_row_stride, num_kv_heads, num_blocks,
                                   plan_dev, plan, workspace, work.part_rows, scale);
  const cudaError_t e = launch_rows_attention<true, true>(a, pool, none, plan_dev, work,
                                                          false, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail("8-bit tree attention launch", e);
  return MS_OK;
}
