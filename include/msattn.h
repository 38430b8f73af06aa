/* C ABI of libmsattn.so: MiniServe's per-step attention path on B200 (sm_100a).
 *
 * Every entry point is extern "C", takes plain pointers and sizes, returns 0 on success or a
 * positive MS_ERR_* code (ms_last_error() then describes it), never allocates device memory and
 * never synchronises the stream it is given (except ms_device_status, whose job is to).
 * Device pointers are raw CUDA addresses; `stream` is a cudaStream_t passed as void*.
 *
 * Geometry: head_dim 128, 16-token KV blocks, two query heads per KV head (Qwen3-0.6B:
 * 16 query heads, 8 KV heads).  Activations are bf16; the cos/sin tables are fp32.
 *
 * KV pool layout (one layer): [num_blocks][num_kv_heads][2: K,V][2: d/64][16 tokens][64] bf16, so
 * K and V of one (block, head) are 8 KiB contiguous.  The layer's "k_cache" pointer is the start
 * of that region and "v_cache" must be k_cache + 4096 bytes; slot = block * 16 + token.
 *
 * 8-bit pool layout (one layer, the *_kv8 entry points): [num_blocks][num_kv_heads][4128 bytes]: K's
 * 16 rows of 128 e4m3 codes, V's 16 rows, K's 16 exponent bytes, V's 16.  Row t's 16-byte chunk i sits
 * at chunk i ^ (t % 2 + 2 (t / 4)).  A row with exponent byte b stands for its codes times 2^(b - 127); b - 127 is the
 * smallest integer in [-100, 120] that brings the row's largest magnitude to at most 448, and b = 255
 * marks a row that held a NaN or an infinity: it stands for NaN.  `pool` is the layer's first byte,
 * 16-byte aligned.
 */
#ifndef MSATTN_H_
#define MSATTN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MS_ABI_VERSION 1

#if defined(__GNUC__)
#define MS_API __attribute__((visibility("default")))
#else
#define MS_API
#endif

enum {
  MS_OK = 0,
  MS_ERR_ARG = 1,     /* a size, shape, stride or pointer argument is invalid */
  MS_ERR_LAYOUT = 2,  /* the KV pool views are not in the layout described above */
  MS_ERR_PLAN = 3,    /* the batch description cannot be planned (table too short, ...) */
  MS_ERR_CUDA = 4,    /* a CUDA runtime/driver call failed */
  MS_ERR_CAPACITY = 5 /* an output buffer given to the planner is too small */
};

/* Device status bits reported by ms_device_status. */
#define MS_DEV_BAD_SLOT 1u     /* slot_mapping entry outside the pool: that row was not written */
#define MS_DEV_BAD_BLOCK 2u    /* block table entry outside the pool: read as zeros */
#define MS_DEV_TIMEOUT 4u      /* a bounded pipeline wait gave up */
#define MS_DEV_BAD_POSITION 8u /* RoPE position outside the cos/sin table: row 0 used */

/* Library version (MS_ABI_VERSION * 100 + minor). */
MS_API int ms_version(void);

/* Description of the last error raised on the calling thread ("" if none). */
MS_API const char* ms_last_error(void);

/* Synchronises `stream`, then reads (and if `clear` != 0 resets) the current device's status
 * word into *flags.  Call it at points where the caller already synchronises. */
MS_API int ms_device_status(void* stream, uint32_t* flags, int clear);

/* ---- Per-step plan (host only) ---------------------------------------------------------------
 * Replaces build_attention_metadata (src/miniserve/attention/backends.py:80-142) and the int64
 * index/mask tensors it builds.  The batch is described the way SeqChunk does
 * (backends.py:36-47): for sequence i, its new tokens are rows flat_start[i] .. +num_new[i] of
 * the flat batch and num_cached[i] tokens are already in the pool; its block table is
 * tables[table_offsets[i] .. table_offsets[i+1]).  The plan is a packed int32 buffer, uploaded
 * once per step and read by every layer.
 */
typedef struct MsPlanInfo {
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t n_decode_items;  /* work items of <= 8 query tokens (decode / speculative verify) */
  int32_t n_tile_items;    /* work items of 9..64-token chunks (mma.sync tile kernel) */
  int32_t n_combine;       /* split tiles (and cascade rows) whose partials must be merged */
  int32_t off_seqs;        /* int32 offsets of each section inside the packed buffer */
  int32_t off_tables;
  int32_t off_decode;
  int32_t off_tile;
  int32_t off_combine;
  int32_t total_ints;      /* length of the packed buffer actually written */
  int32_t pages_per_split; /* split size chosen (pages of 16 tokens) */
  int64_t part_rows;       /* rows of fp32 partial output held in the workspace */
  int64_t workspace_bytes_per_kv_head; /* scratch per KV head the attention call needs:
                                          ms_paged_attention wants this x num_kv_heads bytes
                                          (0 when no tile is split) */
  int64_t total_pages;     /* sum over work tiles of KV pages read (per KV head) */
  int32_t n_tc_items;      /* work items of 64 query tokens of chunks longer than 64 tokens,
                              run on the tcgen05 tensor-core kernel */
  int32_t off_tc;
  int32_t n_cascade;       /* shared-prefix groups: runs of >= 16 consecutive decode / verify
                              rows whose tables share >= 16 cached blocks attend that prefix
                              once (tensor-core items over the group's tokens) and merge it with
                              their own pages; sequence records num_seqs .. num_seqs+n_cascade-1
                              describe the groups */
  int32_t decode_pages;    /* pages (per KV head) the decode / verify items read, in total */
  int32_t combine_tokens_max; /* most query tokens of one combine record (sizes its grid) */
  int32_t n_tc_combine;       /* combine records of tensor-core items: the last ones */
  int32_t is_tree;            /* 1: a plan of ms_tree_plan_build, for ms_tree_attention(_kv8) */
  int32_t reserved;
} MsPlanInfo;

/* Upper bound on the packed buffer length (int32 elements) for a batch of this size. */
MS_API int64_t ms_plan_capacity(int32_t num_seqs, int32_t num_tokens, int64_t total_table_entries);

/* Builds the plan.  block_size must be 16.  num_sms sizes the split-KV work; pages_per_split
 * forces a split size (0 = automatic).  Replaces backends.py:80-142 (grouping, padding, masks). */
MS_API int ms_plan_build(int32_t num_seqs, const int32_t* flat_start, const int32_t* num_new,
                  const int32_t* num_cached, const int64_t* table_offsets, const int32_t* tables,
                  int32_t num_tokens, int32_t block_size, int32_t num_sms,
                  int32_t pages_per_split, int32_t* out, int64_t out_capacity, MsPlanInfo* info);

/* Runner step preparation (host only).  Replaces the attention inputs of ModelRunner.prepare
 * (src/miniserve/runner/model_runner.py:162-205), which walks every scheduled token in Python:
 * sequence i schedules num_new[i] tokens after num_cached[i] computed ones, with block table
 * tables[table_offsets[i] .. table_offsets[i+1]).  Writes flat_start[i] (its first row in the
 * flat batch), and for its tokens, in flat-batch order, positions[t] = num_cached[i] + k and
 * slot_mapping[t] = table[p / block_size] * block_size + p % block_size (the reference's slot
 * formula, model_runner.py:188), and *num_tokens.  The outputs feed ms_plan_build and
 * ms_qk_norm_rope_scatter directly.  Errors: MS_ERR_ARG (bad sizes), MS_ERR_PLAN (a table
 * shorter than its context), MS_ERR_CAPACITY (more tokens than capacity_tokens). */
MS_API int ms_prepare_step(int32_t num_seqs, const int32_t* num_new, const int32_t* num_cached,
                    const int64_t* table_offsets, const int32_t* tables, int32_t block_size,
                    int32_t* flat_start, int64_t* positions, int64_t* slot_mapping,
                    int64_t capacity_tokens, int32_t* num_tokens);

/* ---- Kernel A: q/k RMSNorm + RoPE + K/V scatter ----------------------------------------------
 * Replaces, for one layer, qwen3.py:94-98 (split, q_norm, k_norm, apply_rope) and the K/V
 * index_copy_ at backends.py:159-160.  qkv is the fused projection output [T, (H+2*KVH)*128];
 * q_out receives the normalised, rotated queries [T, H, 128]; the normalised, rotated keys and
 * the raw values go to slot_mapping[t] of the pool.  cos/sin are either per-token rows [T, 128]
 * (positions == NULL, what Qwen3ForCausalLM.forward gathers at qwen3.py:149) or the whole
 * [max_positions, 128] table indexed by positions[t]. */
MS_API int ms_qk_norm_rope_scatter(const void* qkv, int64_t qkv_row_stride, int32_t num_tokens,
                            int32_t num_heads, int32_t num_kv_heads, const void* q_weight,
                            const void* k_weight, float eps, const float* cos, const float* sin,
                            int64_t cs_row_stride, const int64_t* positions,
                            int64_t max_positions, const int64_t* slot_mapping, void* q_out,
                            int64_t q_out_row_stride, void* k_cache, void* v_cache,
                            int32_t num_blocks, void* stream);

/* ---- Kernel E: qkv projection with kernel A as its epilogue -----------------------------------
 * Replaces, for one layer, `self.qkv_proj(x)` and the split/q_norm/k_norm/apply_rope after it
 * (qwen3.py:94-98, the projection built at qwen3.py:75-77 as nn.Linear(hidden, (H+2*KVH)*128,
 * bias=False)) plus the K/V index_copy_ at backends.py:159-160, in one tensor-core launch: the
 * projection output never reaches memory.  x is [T, hidden] bf16 (hidden a multiple of 64), w_qkv
 * the projection weight [(H+2*KVH)*128, hidden] bf16 as nn.Linear stores it; every other argument
 * means what it means for ms_qk_norm_rope_scatter, with x, w_qkv, q_out and the two norm weights
 * 16-byte aligned (row strides multiples of 8 elements).  The result equals
 * ms_qk_norm_rope_scatter applied to bf16(x @ w_qkv^T) except where the GEMM's fp32 accumulation
 * order moves a projection output by one bf16 ulp. */
MS_API int ms_qkv_proj_norm_rope_scatter(const void* x, int64_t x_row_stride, int32_t num_tokens,
                                  int32_t hidden, const void* w_qkv, int64_t w_row_stride,
                                  int32_t num_heads, int32_t num_kv_heads, const void* q_weight,
                                  const void* k_weight, float eps, const float* cos,
                                  const float* sin, int64_t cs_row_stride,
                                  const int64_t* positions, int64_t max_positions,
                                  const int64_t* slot_mapping, void* q_out,
                                  int64_t q_out_row_stride, void* k_cache, void* v_cache,
                                  int32_t num_blocks, void* stream);

/* Scatter only (backends.py:159-160): k, v [T, KVH, 128] with the given row strides.  The slots of one call
 * differ from each other.  ms_paged_attention may read rows below a sequence's cached length while the call
 * before it on the stream still runs: rows that are moved below it (accepted drafts) are followed by another
 * call of the step, such as the write of its own rows, or by ms_kv_moved. */
MS_API int ms_kv_scatter(const void* k, int64_t k_row_stride, const void* v, int64_t v_row_stride,
                  int32_t num_tokens, int32_t num_kv_heads, const int64_t* slot_mapping,
                  void* k_cache, void* v_cache, int32_t num_blocks, void* stream);

/* ---- Kernels B + C: attention through the pool ------------------------------------------------
 * Replaces backends.py:161-197 (gather, GQA fold, masked SDPA, output scatter).  q, out:
 * [T, H, 128] bf16 with the given row strides; plan_dev is the uploaded packed plan and `plan`
 * its host-side info; workspace holds plan->workspace_bytes_per_kv_head * num_kv_heads bytes of
 * scratch (may be NULL when that is 0).  Only rows covered by the plan's sequences are written. */
MS_API int ms_paged_attention(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                       int32_t num_heads, int32_t num_kv_heads, const void* k_cache,
                       const void* v_cache, int32_t num_blocks, const int32_t* plan_dev,
                       const MsPlanInfo* plan, void* workspace, int64_t workspace_bytes,
                       float scale, void* stream);

/* After rows were moved by the calls before: the next call on the stream starts when they have completed. */
MS_API int ms_kv_moved(void* stream);

/* ---- Rows of a pool by slot -------------------------------------------------------------------
 * No counterpart in the reference.  k_out, v_out [num_tokens, KVH, 128] bf16 (row strides in
 * elements, multiples of 8, 16-byte aligned) receive rows slots[t] of the pool: draft paths that are
 * moved after a verify step, sequences handed to another cache.  A slot outside the pool reads as
 * zeros and sets MS_DEV_BAD_SLOT.  From an 8-bit pool the values are exact (codes times a power of
 * two are bf16 values), and writing them back stores the same values again. */
MS_API int ms_kv_gather(const int64_t* slots, int32_t num_tokens, int32_t num_kv_heads,
                        const void* k_cache, const void* v_cache, int32_t num_blocks, void* k_out,
                        int64_t k_row_stride, void* v_out, int64_t v_row_stride, void* stream);
MS_API int ms_kv_gather_kv8(const int64_t* slots, int32_t num_tokens, int32_t num_kv_heads,
                            const void* pool, int32_t num_blocks, void* k_out,
                            int64_t k_row_stride, void* v_out, int64_t v_row_stride, void* stream);

/* ---- Writing an 8-bit pool ----------------------------------------------------------------------
 * ms_kv_scatter and kernel A with rows quantised as they are written.  The arguments are those of
 * ms_kv_scatter and ms_qk_norm_rope_scatter with `pool` in place of the two cache pointers; the
 * quantised values are exactly the bf16 rows those would store. */
MS_API int ms_kv_scatter_kv8(const void* k, int64_t k_row_stride, const void* v,
                             int64_t v_row_stride, int32_t num_tokens, int32_t num_kv_heads,
                             const int64_t* slot_mapping, void* pool, int32_t num_blocks,
                             void* stream);
MS_API int ms_qk_norm_rope_scatter_kv8(const void* qkv, int64_t qkv_row_stride, int32_t num_tokens,
                                       int32_t num_heads, int32_t num_kv_heads,
                                       const void* q_weight, const void* k_weight, float eps,
                                       const float* cos, const float* sin, int64_t cs_row_stride,
                                       const int64_t* positions, int64_t max_positions,
                                       const int64_t* slot_mapping, void* q_out,
                                       int64_t q_out_row_stride, void* pool, int32_t num_blocks,
                                       void* stream);

/* ---- Attention through an 8-bit pool --------------------------------------------------------------
 * Same work and plan as ms_paged_attention.  Rows of up to 64 new tokens read the 8-bit pages in
 * place; chunks of more than 64 tokens (and the shared prefix of cascade groups) run on the
 * tensor-core kernel over bf16 copies of their pages, expanded into the workspace first.  What that
 * needs beside the plan is described by MsKv8Info: ms_kv8_plan_build appends it (host only) to the
 * packed plan, at int offset plan->total_ints of the same buffer (so one upload brings both; the
 * buffer holds ms_kv8_plan_capacity ints beyond the plan), and the attention call gets
 * the uploaded whole.  workspace_bytes >= ms_kv8_workspace_bytes; the workspace is zero-filled before
 * its first use (it holds arrival counters of split tiles, which every call leaves at zero), and calls
 * that share one are ordered on the GPU. */
typedef struct MsKv8Info {
  int32_t n_pages;    /* pages (per KV head) expanded for the tensor-core kernel */
  int32_t off_seqs;   /* int offsets in the packed buffer: sequence records whose tables index */
  int32_t off_map;    /* the expanded pages; the expanded pages' block ids; 0, 1, 2, ... */
  int32_t off_tables;
  int32_t n_narrow;   /* work items of the rows with up to 64 new tokens: tiles of <= 16 tokens, */
  int32_t off_narrow; /* tiles of 17..32, and the combine records of split tiles */
  int32_t n_wide;
  int32_t off_wide;
  int32_t n_combine;
  int32_t off_combine;
  int32_t total_ints; /* length of the packed buffer with this part */
  int32_t reserved;
  int64_t part_rows;  /* partial rows beyond the plan's */
} MsKv8Info;

MS_API int64_t ms_kv8_plan_capacity(int32_t num_seqs, int64_t total_table_entries);
MS_API int ms_kv8_plan_build(int32_t* packed, int64_t capacity, const MsPlanInfo* plan,
                             int32_t num_sms, int32_t pages_per_split, MsKv8Info* info);
MS_API int64_t ms_kv8_workspace_bytes(const MsPlanInfo* plan, const MsKv8Info* info,
                                      int32_t num_kv_heads);
MS_API int ms_paged_attention_kv8(const void* q, int64_t q_row_stride, void* out,
                                  int64_t out_row_stride, int32_t num_heads, int32_t num_kv_heads,
                                  const void* pool, int32_t num_blocks, const int32_t* plan_dev,
                                  const MsPlanInfo* plan, const MsKv8Info* info, void* workspace,
                                  int64_t workspace_bytes, float scale, void* stream);

/* ---- Attention over trees of drafted tokens ---------------------------------------------------------
 * No counterpart in the reference (its drafts are chains).  Sequence i's new tokens are drafts: draft
 * k lies in the cache at position num_cached[i] + k (its slot), and sees the cached tokens, its
 * ancestors and itself.  parents (concatenated in sequence order, num_new[i] each) holds, for draft
 * k, an earlier draft of the sequence (0 <= parent < k), -1 for a child of the last cached token, or -2
 * for an unused position: that draft sees nothing, no draft sees it, and its output is zero whatever
 * its rows hold (it may not be a parent).  RoPE positions are the caller's: num_cached plus the draft's
 * depth.
 *
 * The plan is a packed int32 buffer described by MsPlanInfo, as ms_plan_build's (masks included);
 * ms_tree_attention launches it over a bf16 pool; its workspace of plan->workspace_bytes_per_kv_head *
 * num_kv_heads bytes is zero-filled before its first use, as ms_paged_attention_kv8's.  Over an 8-bit
 * pool ms_kv8_plan_build appends its part to the plan (the capacity below has room for it) and
 * ms_tree_attention_kv8 launches that, with a workspace of ms_kv8_workspace_bytes.  Sequences of at most
 * MS_MAX_TREE_TOKENS drafts. */
#define MS_MAX_TREE_TOKENS 1024
MS_API int64_t ms_tree_plan_capacity(int32_t num_seqs, const int32_t* num_new,
                                     int64_t total_table_entries);
MS_API int ms_tree_plan_build(int32_t num_seqs, const int32_t* flat_start, const int32_t* num_new,
                              const int32_t* num_cached, const int64_t* table_offsets,
                              const int32_t* tables, const int32_t* parents, int32_t num_tokens,
                              int32_t block_size, int32_t num_sms, int32_t pages_per_split,
                              int32_t* out, int64_t out_capacity, MsPlanInfo* info);
MS_API int ms_tree_attention(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                             int32_t num_heads, int32_t num_kv_heads, const void* k_cache,
                             const void* v_cache, int32_t num_blocks, const int32_t* plan_dev,
                             const MsPlanInfo* plan, void* workspace, int64_t workspace_bytes,
                             float scale, void* stream);
MS_API int ms_tree_attention_kv8(const void* q, int64_t q_row_stride, void* out,
                                 int64_t out_row_stride, int32_t num_heads, int32_t num_kv_heads,
                                 const void* pool, int32_t num_blocks, const int32_t* plan_dev,
                                 const MsPlanInfo* plan, const MsKv8Info* info, void* workspace,
                                 int64_t workspace_bytes, float scale, void* stream);

/* ---- Sparse attention over selected pages -------------------------------------------------------------
 * No counterpart in the reference.  A page is the 16 tokens of one block, of one KV head.  Its bounds, lo and
 * hi, are the smallest and the largest value of each channel over its tokens' keys; a layer's bounds are
 * [num_blocks][num_kv_heads][2: lo, hi][128] bf16, 16-byte aligned (8 KiB of K and V have 512 bytes of them).
 * No key of the page has a larger product with a query q than sum_d max(q_d lo_d, q_d hi_d).
 *
 * ms_key_bounds_step: the bounds of every page that the new tokens of a plan's sequences lie on (a plan of
 * ms_plan_build or ms_tree_plan_build), over the page's tokens up to the sequence's end, after the step's
 * rows are written.  A NaN key makes the channel's bounds NaN.
 * ms_key_bounds: of listed blocks (device int64), over the first rows[i] tokens of blocks[i]; an entry with
 * a negative block or no rows is skipped.  Moved rows (accepted drafts) need it, copied pages do not where
 * the bounds are copied with them.  A block outside the pool is skipped and sets MS_DEV_BAD_BLOCK. */
MS_API int ms_key_bounds_step(const void* k_cache, int32_t num_blocks, int32_t num_kv_heads,
                              const int32_t* plan_dev, const MsPlanInfo* plan, void* bounds,
                              void* stream);
MS_API int ms_key_bounds_step_kv8(const void* pool, int32_t num_blocks, int32_t num_kv_heads,
                                  const int32_t* plan_dev, const MsPlanInfo* plan, void* bounds,
                                  void* stream);
MS_API int ms_key_bounds(const void* k_cache, int32_t num_blocks, int32_t num_kv_heads,
                         const int64_t* blocks, const int64_t* rows, int32_t count, void* bounds,
                         void* stream);
MS_API int ms_key_bounds_kv8(const void* pool, int32_t num_blocks, int32_t num_kv_heads,
                             const int64_t* blocks, const int64_t* rows, int32_t count, void* bounds,
                             void* stream);

/* The pages that each query token of a plan's sequences of at most 8 new tokens keeps, for each KV head:
 * pages [num_tokens, num_kv_heads, budget] int32 (rows of other sequences are left as they are), indices into
 * the sequence's block table in ascending order, -1 behind.  A token at position p sees the pages 0 .. p / 16.
 * It keeps them all where they are at most budget; else the first `first`, the last `last` (>= 1: its own
 * page), and of those between the ones with the highest scores,
 *   score(page) = max over the KV head's two query heads of sum_d max(q_d lo_d, q_d hi_d),
 * equal scores by the lower page, one that is not finite as infinity, and so any score of a page with a bound
 * that is not finite.  Scores are compared as exactly as 64 bits give them.  max_new (1 .. 8) and max_pages (at
 * most 49152) bound the new tokens and the pages of those sequences; budget is at most 4096.  Bounds of the pages
 * between are read: they have to be up to date.  A block outside the pool is scored by the bounds of block 0 and
 * sets MS_DEV_BAD_BLOCK.
 * workspace: ms_select_workspace_bytes of scratch (num_seqs * max_new * num_kv_heads * max_pages * 4.25, max_pages
 * in steps of 64), 16-byte aligned; nothing is kept in it between calls. */
MS_API int64_t ms_select_workspace_bytes(int32_t num_seqs, int32_t max_new, int32_t max_pages,
                                         int32_t num_kv_heads);
MS_API int ms_select_pages(const void* q, int64_t q_row_stride, int32_t num_heads, int32_t num_kv_heads,
                           const void* bounds, int32_t num_blocks, const int32_t* plan_dev,
                           const MsPlanInfo* plan, int32_t max_new, int32_t max_pages, int32_t budget,
                           int32_t first, int32_t last, int32_t* pages, void* workspace,
                           int64_t workspace_bytes, void* stream);

/* Attention of those query tokens over the keys of their pages, up to the token's own position.  Entries of
 * `pages` that the token does not see (negative, or behind its own page) are skipped, in any place; a page
 * named twice counts twice; a row without pages gives zeros.  Other rows of out are left as they are.  A
 * block outside the pool is left out and sets MS_DEV_BAD_BLOCK.  Over an 8-bit pool a key adds nothing where
 * its weight times its value row's size is below 2^-36 of the largest such product of the query token, and a
 * query's channels below 2^-27 of its largest one lose bits. */
MS_API int ms_attend_pages(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                           int32_t num_heads, int32_t num_kv_heads, const void* k_cache,
                           const void* v_cache, int32_t num_blocks, const int32_t* plan_dev,
                           const MsPlanInfo* plan, int32_t max_new, const int32_t* pages, int32_t budget,
                           float scale, void* stream);
MS_API int ms_attend_pages_kv8(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                               int32_t num_heads, int32_t num_kv_heads, const void* pool,
                               int32_t num_blocks, const int32_t* plan_dev, const MsPlanInfo* plan,
                               int32_t max_new, const int32_t* pages, int32_t budget, float scale,
                               void* stream);

/* ---- Whole pages of a paged tensor ----------------------------------------------------------------------
 * No counterpart in the reference.  base: [num_layers][num_blocks][page_bytes] with layer_stride bytes from
 * layer to layer (a pool of either kind, key bounds); base, page_bytes and layer_stride are multiples of 16.
 * The lists are host memory, read before the call returns; a captured call keeps them.
 *
 * ms_copy_pages copies block src[i] to block dst[i] in every layer.  No block is written twice, or both
 * written and read, by one call (one block may go to several).
 * ms_clear_pages fills blocks with zeros.  Attention that follows either waits for it. */
MS_API int ms_copy_pages(void* base, int64_t layer_stride, int64_t page_bytes, int32_t num_layers,
                         int32_t num_blocks, const int32_t* src, const int32_t* dst, int32_t count,
                         void* stream);
MS_API int ms_clear_pages(void* base, int64_t layer_stride, int64_t page_bytes, int32_t num_layers,
                          int32_t num_blocks, const int32_t* blocks, int32_t count, void* stream);

/* ---- Attention for callers that cannot allocate device memory -------------------------------
 * No counterpart in the reference (MiniServe allocates everything through PyTorch).
 *
 * Same work and arguments as ms_paged_attention, minus the workspace: the split-KV partials go
 * to a fixed scratch array compiled into the library, MS_NOALLOC_SCRATCH_BYTES on every GPU that
 * loads it, held until the process exits.  It is meant for hosts that never let a plugin call
 * cudaMalloc (an engine that gives all GPU memory to its own arena, a custom-op interface with
 * no allocator hook, a loop that cannot take cudaMalloc's implicit synchronisation).  The call
 * itself allocates nothing.
 *
 *  - A plan needing more than MS_NOALLOC_SCRATCH_BYTES of partials
 *    (plan->workspace_bytes_per_kv_head * num_kv_heads) is rejected with MS_ERR_CAPACITY; plan
 *    with a larger pages_per_split or use ms_paged_attention.
 *  - Every call looks up the current context's address of the array (with that device current),
 *    so a context recreated after cudaDeviceReset gets the new address.  The first call in a
 *    process may load the library's device code; make that first call before any stream capture.
 *  - All calls share the array: calls that overlap on the GPU race on it; calls ordered on one
 *    stream are safe.  No state carries over between calls. */
#define MS_NOALLOC_SCRATCH_BYTES (16u * 1024u * 1024u)

MS_API int ms_paged_attention_noalloc(const void* q, int64_t q_row_stride, void* out,
                                      int64_t out_row_stride, int32_t num_heads,
                                      int32_t num_kv_heads, const void* k_cache,
                                      const void* v_cache, int32_t num_blocks,
                                      const int32_t* plan_dev, const MsPlanInfo* plan,
                                      float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSATTN_H_ */
