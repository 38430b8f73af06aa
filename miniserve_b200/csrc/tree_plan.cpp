// Host planners of the 8-bit pool and of drafted token trees (declared in include/msattn.h).
//
// Both cut the work of kernel F: tiles of at most 32 query tokens of one sequence, split over their
// pages where that fills the GPU.
//
// ms_kv8_plan_build adds to a packed plan those tiles for the sequences of up to 64 new tokens, and
// what its tensor-core items need over an 8-bit pool: the pages they read are expanded to bf16 in the
// workspace, numbered densely, so the part holds the expanded pages' block ids, the identity table
// the kernel walks instead of the block tables, and the sequence records with their tables' places
// in it.  To a plan of trees with tensor-core items it adds the tiles that kernel F reads whole in
// their place: expanding pages that one sequence reads once would write and read four times their
// bytes (48 trees of 32 drafts over 256-4096 tokens: 123 us with kernel F).
//
// ms_tree_plan_build cuts every sequence of drafts into tiles that read the cached context and the
// drafts up to the tile's last one (a parent precedes its children).  Masks are bit rows, one per
// draft, ceil(num_new / 32) words each, at the sequence record's field 6 (length in words in field 7).
#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstring>
#include <exception>
#include <functional>
#include <string>
#include <vector>

#include "../../include/msattn.h"

namespace ms_host {
void set_error(const std::string& msg);
}

namespace {

constexpr int kRec = 8;
constexpr int kTileTokens = 32;     // tokens of a wide tile (64 query rows) at most
constexpr int kNarrowTokens = 16;   // tiles of at most 32 query rows run three CTAs per SM, others two
// The planner does not see the head count, and only speed depends on it.  Narrow tiles are sized for two
// CTAs per SM at 8 KV heads: they are bound by memory, which fewer CTAs still keep busy at 4 heads, and
// more splits only cost merging (3 rows over 100k tokens: 51 us with 36 splits, 64 with 108; 64 trees
// of 16 drafts: 98 us, 107 in splits of 128 pages; the costs below instead of this rule: 36 trees of 12
// drafts at 8 heads 81 -> 107 us, 19 of 13 at 4 heads 55 -> 37).  Splits of less than 8 pages cost more than
// they fill (8 decode rows: 16 us in splits of 4 pages, 14 in 8).  The tiles of tensor-core items are sized
// for one CTA per SM at 4 heads.
constexpr int kNarrowHeads = 8, kTensorHeads = 4;
constexpr int kMinSplitPages = 8;
constexpr int kMaxSplitPages = 512;

// What wide tiles cost, in microseconds (measured with 1 and 2 CTAs per SM over 64 to 256 8-bit pages): a page
// for a CTA that has its SM to itself, a page of the SM's throughput, and a work item's fixed part (start,
// first pages, epilogue); an SM holds two.  A bf16 page takes as long, twice the bytes but no conversions: 37
// trees of 32 drafts over 32 and over 480 cached tokens take 20.2 and 33.6 us in 8 bits, 19.3 and 32.7 in
// bf16, 0.24 per page and SM in both.
constexpr double kWidePageAlone = 0.35, kWidePageSm = 0.26, kWideItem = 9;
constexpr int kWideCtas = 2;
// Tensor-core items, one per SM, and what follows them: kernel F's last pages and the merge.
constexpr double kTensorPage = 0.21, kTensorItem = 10, kTensorTail = 18;
constexpr int kHeads[2] = {8, 4};  // the head counts that times are weighed for
// The merge of n splits of `rows` rows: latencies of L2, see merge_splits.
double merge_cost(int n, int rows) {
  if (n <= 1) return 0;
  const int per_warp = (rows + 3) / 4;
  return 2 + 0.8 * (n <= 4 ? (per_warp + 3) / 4 : (per_warp + 1) / 2 * ((n + 7) / 8));
}

int64_t round4(int64_t x) { return (x + 3) & ~int64_t(3); }

// No C++ exception leaves an extern "C" function: the planners' vectors may fail to allocate.
template <typename F>
int guarded(const char* what, F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      ms_host::set_error(std::string(what) + ": " + e.what());
    } catch (...) {
    }
    return MS_ERR_CAPACITY;
  }
}

// A tile of at most 32 query tokens and the pages it reads, before splitting; then a work item.
struct RowsItem {
  int seq, tok0, n_q, pb, pe;
  int part_row = -1;
  // Fields 6 and 7: the combine record and 2 for a split, the shared-prefix partial row and 1 for a
  // cascade row, the combine record and 3 for the last pages of a tile whose cached blocks are read by
  // tensor-core items (which write the other partial rows of that record).
  int field6 = 0, field7 = 0;
};

// Cached whole 128-key blocks of the tiles of larger trees run on the tensor cores over a bf16 pool: tiles
// of more than 16 drafts are bound by mma.sync, and those blocks need no mask (16 trees of 63 drafts over
// 4000-8100 tokens: 117 us without this, 76 with it).  Fewer pages than kPrefixMinPages are not worth the
// second launch.
constexpr int kBlockPages = 8;
constexpr int kPrefixTileTokens = 64;  // 128 query rows
constexpr int kPrefixMinPages = 32, kPrefixMinSplitPages = 64;

// The items of kernel F: narrow and wide tiles (two launches), split over their pages, and the
// combine records of the split ones.
struct RowsPlan {
  // comb: pb = first partial row, pe = number of partials per row, part_row = rows between them,
  // field6 = how many of kernel F's CTAs arrive (per head).
  std::vector<RowsItem> narrow, wide, comb;
  int64_t part_rows = 0;                     // from `base` on
  int split_narrow = 0, split_wide = 0;
};

// The smallest multiple of 8 pages, at least `least`, whose items number at most `target`; when the
// tiles alone exceed it, tiles longer than the pages per slot are cut to about that size.
int fit_split(const std::vector<RowsItem>& tiles, int64_t target, int least) {
  int64_t all = 0;
  for (const RowsItem& t : tiles) all += t.pe - t.pb;
  auto items_at = [&](int64_t p) {
    int64_t items = 0;
    for (const RowsItem& t : tiles) items += (t.pe - t.pb + p - 1) / p;
    return items;
  };
  if (items_at(kMaxSplitPages) > target) {
    const int64_t per_slot = (all + target - 1) / target;
    return static_cast<int>(std::min<int64_t>(
        kMaxSplitPages, std::max<int64_t>(least, (per_slot + 7) / 8 * 8)));
  }
  int lo = least / 8, hi = kMaxSplitPages / 8;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (items_at(mid * 8) <= target) hi = mid; else lo = mid + 1;
  }
  return lo * 8;
}

// Time of pieces of `len` pages (longest first) of h heads each: every SM shares its throughput among the
// CTAs that it holds, so they are dealt to SMs, the least loaded one next.
double deal(const std::vector<int>& len, int h, double item, double page, int num_sms) {
  const size_t sms = std::max(1, num_sms / h);
  std::vector<double> load;  // a heap, the least loaded SM first
  load.reserve(sms);
  double end = 0;
  for (int p : len) {
    double t = item + p * page;
    if (load.size() == sms) {
      std::pop_heap(load.begin(), load.end(), std::greater<double>());
      t += load.back();
      load.pop_back();
    }
    load.push_back(t);
    std::push_heap(load.begin(), load.end(), std::greater<double>());
    end = std::max(end, t);
  }
  return end;
}
double wide_time(const std::vector<int>& len, int h, int num_sms) {
  const double item = kWideItem / kWideCtas;
  return std::max(len[0] * kWidePageAlone, deal(len, h, item, kWidePageSm, num_sms)) + kWideItem - item;
}

// Pages per split of wide tiles, which are bound by the SMs.  Many tiles (two waves of 8 heads and more) fill
// the GPU whole; only those longer than a CTA's share of the pages are cut to about that.  With fewer,
// the longest tile cut into 1, 2, 3 ... parts, and all others into parts as long, whichever the costs above
// put first: splits shorten the run, but the last CTA of a tile merges them alone (one tree of 24 drafts
// over 4000 tokens: 55 us in 3 splits, 35 as chosen here; 48 trees of 32 drafts: 143 us in
// splits of 80 pages, 133 in the 128 chosen).  4 and 8 heads are weighed, each against its own best.
// best: the times of that choice (0 where the tiles are many).
int wide_split(const std::vector<RowsItem>& tiles, int num_sms, double (&best)[2]) {
  best[0] = best[1] = 0;
  const int64_t slots = static_cast<int64_t>(num_sms) * kWideCtas;
  int64_t all = 0;
  int longest = 0;
  for (const RowsItem& t : tiles) {
    all += t.pe - t.pb;
    longest = std::max(longest, t.pe - t.pb);
  }
  if (static_cast<int64_t>(tiles.size()) * kHeads[0] >= 2 * slots) {
    const int64_t share = all * kHeads[1] / slots;
    return static_cast<int>(std::min<int64_t>(kMaxSplitPages, std::max<int64_t>(96, (share + 7) / 8 * 8)));
  }
  constexpr int kParts[] = {1,  2,  3,  4,  5,  6,  7,  8,  10, 12, 14, 16,
                            20, 24, 28, 32, 36, 40, 48, 56, 64, 96, 128};
  std::vector<int> split, len;
  std::vector<double> time[2];
  for (int parts : kParts) {
    const int p = std::max(kMinSplitPages, ((longest + parts - 1) / parts + 7) / 8 * 8);
    if (!split.empty() && p == split.back()) continue;
    len.clear();
    double merge = 0;
    for (const RowsItem& t : tiles) {
      const int pages = t.pe - t.pb, n = (pages + p - 1) / p;
      for (int k = 0; k < n; ++k) len.push_back(pages / n + (k < pages % n ? 1 : 0));
      merge = std::max(merge, merge_cost(n, 2 * t.n_q));
    }
    if (!split.empty() && static_cast<int64_t>(len.size()) * kHeads[1] > 2 * slots) break;
    std::sort(len.begin(), len.end(), std::greater<int>());
    split.push_back(p);
    for (int h = 0; h < 2; ++h) time[h].push_back(wide_time(len, kHeads[h], num_sms) + merge);
  }
  const double best0 = *std::min_element(time[0].begin(), time[0].end());
  const double best1 = *std::min_element(time[1].begin(), time[1].end());
  size_t at = 0;
  for (size_t i = 1; i < split.size(); ++i)
    if (time[0][i] / best0 + time[1][i] / best1 < time[0][at] / best0 + time[1][at] / best1) at = i;
  best[0] = time[0][at];
  best[1] = time[1][at];
  return split[at];
}

// Split size of kernel F's narrow or wide tiles.
int choose_split(const std::vector<RowsItem>& tiles, bool narrow, int num_sms) {
  std::vector<RowsItem> mine;
  for (const RowsItem& t : tiles)
    if ((t.n_q <= kNarrowTokens) == narrow && t.field7 == 0) mine.push_back(t);
  if (mine.empty()) return kMaxSplitPages;
  double unused[2];
  if (!narrow) return wide_split(mine, num_sms, unused);
  return fit_split(mine, std::max(1, num_sms * 2 / kNarrowHeads), kMinSplitPages);
}

// Whether kernel F alone is faster over trees that could have their cached blocks on the tensor cores: not for
// trees of more than 32 drafts, whose tiles read the pages twice, but for smaller ones unless they are
// many or long, since it cuts them into short pieces while the tensor-core kernel is followed by a second one
// (2 trees of 23 drafts over 1800 tokens: 29 us, 35 with tensor-core items; 51 of 17 over 900: 41 and 57;
// 61 of 17 over 4000: 86 with them).
bool wide_is_faster(const std::vector<RowsItem>& tiles, const std::vector<RowsItem>& prefix, int split,
                    int num_sms) {
  std::vector<RowsItem> wide;
  for (const RowsItem& t : tiles)
    if (t.n_q > kNarrowTokens) wide.push_back(t);
  std::vector<int> len;
  for (const RowsItem& t : prefix) {
    if (t.n_q > kTileTokens || t.tok0 > 0) return false;
    const int n = (t.pe + split - 1) / split;
    for (int k = 0; k < n; ++k) len.push_back(t.pe / n);
  }
  std::sort(len.begin(), len.end(), std::greater<int>());
  double best[2], ratio = 0;
  wide_split(wide, num_sms, best);
  if (best[0] == 0) return false;
  for (int h = 0; h < 2; ++h)
    ratio += best[h] / (deal(len, kHeads[h], kTensorItem, kTensorPage, num_sms) + kTensorTail);
  return ratio < 2;
}

// Splits the tiles (cascade rows and the tails of tensor-core prefixes, field7 != 0, stay whole).
// False: too many partial rows.
bool plan_rows(const std::vector<RowsItem>& tiles, int num_sms, int pages_per_split, int64_t base,
               RowsPlan* out) {
  out->split_narrow = pages_per_split > 0 ? pages_per_split : choose_split(tiles, true, num_sms);
  out->split_wide = pages_per_split > 0 ? pages_per_split : choose_split(tiles, false, num_sms);
  for (const RowsItem& t : tiles) {
    const bool narrow = t.n_q <= kNarrowTokens;
    const int split = narrow ? out->split_narrow : out->split_wide;
    std::vector<RowsItem>& items = narrow ? out->narrow : out->wide;
    const int pages = t.pe - t.pb;
    const int ns = (pages + split - 1) / split;
    if (ns <= 1 || t.field7 != 0) {
      items.push_back(t);
      continue;
    }
    const int rows = 2 * t.n_q;
    const int64_t first = base + out->part_rows;
    if (first + static_cast<int64_t>(ns) * rows >= INT32_MAX) return false;
    const int each = pages / ns, rem = pages % ns;
    int pb = t.pb;
    for (int s = 0; s < ns; ++s) {
      const int len = each + (s < rem ? 1 : 0);
      items.push_back({t.seq, t.tok0, t.n_q, pb, pb + len,
                       static_cast<int>(first + static_cast<int64_t>(s) * rows),
                       static_cast<int>(out->comb.size()), 2});
      pb += len;
    }
    out->comb.push_back({t.seq, t.tok0, t.n_q, static_cast<int>(first), ns, rows, ns, 0});
    out->part_rows += static_cast<int64_t>(ns) * rows;
  }
  auto longest_first = [](const RowsItem& x, const RowsItem& y) {
    return (x.pe - x.pb) > (y.pe - y.pb);
  };
  std::stable_sort(out->narrow.begin(), out->narrow.end(), longest_first);
  std::stable_sort(out->wide.begin(), out->wide.end(), longest_first);
  return true;
}

void put_items(int32_t* out, int64_t off, const std::vector<RowsItem>& v) {
  for (size_t k = 0; k < v.size(); ++k) {
    int32_t* r = out + off + static_cast<int64_t>(k) * kRec;
    r[0] = v[k].seq;
    r[1] = v[k].tok0;
    r[2] = v[k].n_q;
    r[3] = v[k].pb;
    r[4] = v[k].pe;
    r[5] = v[k].part_row;
    r[6] = v[k].field6;
    r[7] = v[k].field7;
  }
}

int64_t size4(const std::vector<RowsItem>& v) { return round4(static_cast<int64_t>(v.size()) * kRec); }

}  // namespace

extern "C" int64_t ms_kv8_plan_capacity(int32_t num_seqs, int64_t total_table_entries) {
  if (num_seqs < 0 || total_table_entries < 0) return 0;
  // At most two tiles of 32 tokens per sequence, each at most one item per page, as many combine
  // records; the records (one more per cascade group), map and tables of the tensor-core items.
  const int64_t tiles = 2 * static_cast<int64_t>(num_seqs);
  return 2 * round4((tiles + 2 * total_table_entries) * kRec) + round4(tiles * kRec) +
         round4(tiles * kRec) + 2 * round4(total_table_entries) + 16;
}

static int kv8_plan_build(int32_t* packed, int64_t capacity, const MsPlanInfo* plan,
                          int32_t num_sms, int32_t pages_per_split, MsKv8Info* info) {
  if (packed == nullptr || plan == nullptr || info == nullptr || num_sms <= 0 ||
      pages_per_split < 0) {
    ms_host::set_error("ms_kv8_plan_build: null argument or bad sizes");
    return MS_ERR_ARG;
  }
  std::memset(info, 0, sizeof(*info));
  if (plan->is_tree && plan->n_tc_items == 0) {  // kernel F's items serve either pool
    info->n_narrow = plan->n_decode_items;
    info->off_narrow = plan->off_decode;
    info->n_wide = plan->n_tile_items;
    info->off_wide = plan->off_tile;
    info->n_combine = plan->n_combine;
    info->off_combine = plan->off_combine;
    info->total_ints = plan->total_ints;
    return MS_OK;
  }
  const int32_t* seqs = packed + plan->off_seqs;

  // Kernel F's tiles: the sequences of up to 64 new tokens, in tiles of up to 32; the rows of
  // cascade groups read their own pages (their decode items say which) and merge the prefix partial.
  std::vector<const int32_t*> cascade(plan->num_seqs, nullptr);
  for (int i = 0; i < plan->n_decode_items; ++i) {
    const int32_t* it = packed + plan->off_decode + static_cast<int64_t>(i) * kRec;
    if (it[7] == 1) cascade[it[0]] = it;
  }
  std::vector<RowsItem> tiles;
  for (int i = 0; i < plan->num_seqs; ++i) {
    const int32_t* r = seqs + static_cast<int64_t>(i) * kRec;
    const int n = r[1], c = r[2];
    if (n > 2 * kTileTokens && !plan->is_tree) continue;
    if (cascade[i] != nullptr) {
      tiles.push_back({i, 0, n, cascade[i][3], cascade[i][4], -1, cascade[i][6], 1});
      continue;
    }
    for (int t0 = 0; t0 < n; t0 += kTileTokens) {
      const int nq = std::min(kTileTokens, n - t0);
      tiles.push_back({i, t0, nq, 0, (c + t0 + nq + 15) / 16});
    }
  }
  RowsPlan rows;
  if (!plan_rows(tiles, num_sms, pages_per_split, plan->part_rows, &rows)) {
    ms_host::set_error("ms_kv8_plan_build: too many partial rows");
    return MS_ERR_PLAN;
  }

  // Pages each record's tensor-core items read (the largest page end).
  const int n_rec = plan->num_seqs + plan->n_cascade;
  std::vector<int32_t> pages(n_rec, 0);
  int64_t n_pages = 0;
  for (int i = 0; i < plan->n_tc_items && !plan->is_tree; ++i) {
    const int32_t* it = packed + plan->off_tc + static_cast<int64_t>(i) * kRec;
    pages[it[0]] = std::max(pages[it[0]], it[4]);
  }
  for (int p : pages) n_pages += p;

  const int64_t off_narrow = round4(plan->total_ints);
  const int64_t off_wide = off_narrow + size4(rows.narrow);
  const int64_t off_combine = off_wide + size4(rows.wide);
  const int64_t off_seqs = off_combine + size4(rows.comb);
  const int64_t off_map =
      off_seqs + (n_pages > 0 ? round4(static_cast<int64_t>(n_rec) * kRec) : 0);
  const int64_t off_tables = off_map + round4(n_pages);
  const int64_t total = off_tables + round4(n_pages);
  if (total > capacity) {
    ms_host::set_error("ms_kv8_plan_build: the buffer holds " + std::to_string(capacity) +
                       " ints, the plan with its 8-bit part needs " + std::to_string(total));
    return MS_ERR_CAPACITY;
  }
  if (total >= INT32_MAX) {
    ms_host::set_error("ms_kv8_plan_build: plan larger than 2^31 ints");
    return MS_ERR_PLAN;
  }
  std::memset(packed + plan->total_ints, 0, sizeof(int32_t) * (total - plan->total_ints));
  put_items(packed, off_narrow, rows.narrow);
  put_items(packed, off_wide, rows.wide);
  put_items(packed, off_combine, rows.comb);
  int32_t at = 0;
  for (int i = 0; n_pages > 0 && i < n_rec; ++i) {
    int32_t* r = packed + off_seqs + static_cast<int64_t>(i) * kRec;
    std::memcpy(r, seqs + static_cast<int64_t>(i) * kRec, sizeof(int32_t) * kRec);
    if (pages[i] == 0) continue;
    const int32_t* table = packed + plan->off_tables + r[4];
    for (int p = 0; p < pages[i]; ++p) {
      packed[off_map + at + p] = table[p];
      packed[off_tables + at + p] = at + p;
    }
    r[4] = at;
    r[5] = pages[i];
    at += pages[i];
  }
  info->n_pages = static_cast<int32_t>(n_pages);
  info->off_seqs = static_cast<int32_t>(off_seqs);
  info->off_map = static_cast<int32_t>(off_map);
  info->off_tables = static_cast<int32_t>(off_tables);
  info->n_narrow = static_cast<int32_t>(rows.narrow.size());
  info->off_narrow = static_cast<int32_t>(off_narrow);
  info->n_wide = static_cast<int32_t>(rows.wide.size());
  info->off_wide = static_cast<int32_t>(off_wide);
  info->n_combine = static_cast<int32_t>(rows.comb.size());
  info->off_combine = static_cast<int32_t>(off_combine);
  info->part_rows = rows.part_rows;
  info->total_ints = static_cast<int32_t>(total);
  return MS_OK;
}

extern "C" int ms_kv8_plan_build(int32_t* packed, int64_t capacity, const MsPlanInfo* plan,
                                 int32_t num_sms, int32_t pages_per_split, MsKv8Info* info) {
  return guarded("ms_kv8_plan_build", [&] {
    return kv8_plan_build(packed, capacity, plan, num_sms, pages_per_split, info);
  });
}

extern "C" int64_t ms_kv8_workspace_bytes(const MsPlanInfo* plan, const MsKv8Info* info,
                                          int32_t num_kv_heads) {
  if (plan == nullptr || info == nullptr || num_kv_heads <= 0) return 0;
  // Partials (the plan's and the 8-bit part's), the arrival counters of kernel F's split tiles, then
  // the expanded pages (8 KiB per head) on a 1 KiB boundary.
  const int64_t part = ((plan->part_rows + info->part_rows) * (128 + 1) * 4 +
                        static_cast<int64_t>(info->n_combine) * 4) *
                       num_kv_heads;
  if (info->n_pages == 0) return part;
  return (part + 1023) / 1024 * 1024 + static_cast<int64_t>(info->n_pages) * num_kv_heads * 8192;
}

extern "C" int64_t ms_tree_plan_capacity(int32_t num_seqs, const int32_t* num_new,
                                         int64_t total_table_entries) {
  if (num_seqs < 0 || (num_seqs > 0 && num_new == nullptr)) return 0;
  int64_t tiles = 0, masks = 0, tiles_max = 1;
  for (int i = 0; i < num_seqs; ++i) {
    const int64_t n = std::max(num_new[i], 0);
    tiles += (n + kTileTokens - 1) / kTileTokens;
    tiles_max = std::max(tiles_max, (n + kTileTokens - 1) / kTileTokens);
    masks += n * ((n + 31) / 32);
  }
  // A tile has at most one item per page of its sequence; narrow, wide and tensor-core items, a
  // virtual record per sequence, and the 8-bit part's items and combine records.
  const int64_t items = tiles + tiles_max * total_table_entries;
  return round4(2 * static_cast<int64_t>(num_seqs) * kRec) + round4(total_table_entries) +
         5 * round4(items * kRec) + 2 * round4(tiles * kRec) + round4(masks) + 16;
}

static int tree_plan_build(int32_t num_seqs, const int32_t* flat_start, const int32_t* num_new,
                           const int32_t* num_cached, const int64_t* table_offsets,
                           const int32_t* tables, const int32_t* parents, int32_t num_tokens,
                           int32_t block_size, int32_t num_sms, int32_t pages_per_split,
                           int32_t* out, int64_t out_capacity, MsPlanInfo* info) {
  if (info == nullptr || out == nullptr) {
    ms_host::set_error("ms_tree_plan_build: null output");
    return MS_ERR_ARG;
  }
  std::memset(info, 0, sizeof(*info));
  if (num_seqs < 0 || num_tokens < 0 || block_size != 16 || num_sms <= 0 || pages_per_split < 0) {
    ms_host::set_error("ms_tree_plan_build: bad sizes (block_size must be 16, num_sms > 0)");
    return MS_ERR_ARG;
  }
  if (num_seqs > 0 && (flat_start == nullptr || num_new == nullptr || num_cached == nullptr ||
                       table_offsets == nullptr || parents == nullptr)) {
    ms_host::set_error("ms_tree_plan_build: null batch arrays");
    return MS_ERR_ARG;
  }
  const int64_t total_entries = num_seqs > 0 ? table_offsets[num_seqs] : 0;
  if (total_entries > 0 && tables == nullptr) {
    ms_host::set_error("ms_tree_plan_build: null block tables");
    return MS_ERR_ARG;
  }
  if (total_entries < 0 || total_entries >= (int64_t(1) << 31)) {
    ms_host::set_error("ms_tree_plan_build: block tables exceed 2^31 entries");
    return MS_ERR_ARG;
  }

  std::vector<RowsItem> tiles;
  int64_t mask_words = 0, total_pages = 0, parent_at = 0;
  std::vector<int64_t> mask_at(num_seqs, 0);
  std::vector<int64_t> parents_at(num_seqs, 0);
  for (int i = 0; i < num_seqs; ++i) {
    const std::string who = "ms_tree_plan_build: sequence " + std::to_string(i);
    const int64_t n = num_new[i], c = num_cached[i], f = flat_start[i];
    const int64_t tlen = table_offsets[i + 1] - table_offsets[i];
    if (n < 1 || c < 0 || f < 0 || f + n > num_tokens || tlen < 0) {
      ms_host::set_error(who + " has an invalid flat_start/num_new/num_cached");
      return MS_ERR_PLAN;
    }
    if (n > MS_MAX_TREE_TOKENS) {
      ms_host::set_error(who + " has " + std::to_string(n) + " drafts, more than " +
                         std::to_string(MS_MAX_TREE_TOKENS));
      return MS_ERR_PLAN;
    }
    if (c + n >= (int64_t(1) << 30)) {
      ms_host::set_error("ms_tree_plan_build: context too long");
      return MS_ERR_PLAN;
    }
    if (tlen * block_size < c + n) {
      ms_host::set_error(who + " needs " + std::to_string((c + n + block_size - 1) / block_size) +
                         " blocks but its table has " + std::to_string(tlen));
      return MS_ERR_PLAN;
    }
    const int32_t* par = parents + parent_at;
    for (int64_t k = 0; k < n; ++k) {
      const int32_t p = par[k];
      if (p < -2 || p >= k || (p >= 0 && par[p] == -2)) {
        ms_host::set_error(who + ": draft " + std::to_string(k) + " has parent " +
                           std::to_string(p) +
                           " (want an earlier draft in use, -1 for the last cached token, or -2 "
                           "for an unused position)");
        return MS_ERR_PLAN;
      }
    }
    parents_at[i] = parent_at;
    parent_at += n;
    mask_at[i] = mask_words;
    mask_words += n * ((n + 31) / 32);
    for (int64_t t0 = 0; t0 < n; t0 += kTileTokens) {
      const int nq = static_cast<int>(std::min<int64_t>(kTileTokens, n - t0));
      const int pages = static_cast<int>((c + t0 + nq + block_size - 1) / block_size);
      tiles.push_back({i, static_cast<int>(t0), nq, 0, pages});
      total_pages += pages;
    }
  }

  // The cached blocks of larger trees: tensor-core items over virtual sequences (records after the
  // real ones) whose cached context is those blocks, one tile of up to 64 drafts each, split over the
  // pages; the drafts' tiles keep the pages after them.
  RowsPlan rows;
  std::vector<RowsItem> prefix, tc;
  std::vector<int> vseq_of(num_seqs, -1);
  int n_vseq = 0;
  for (int i = 0; i < num_seqs; ++i) {
    const int pages = num_cached[i] / (kBlockPages * 16) * kBlockPages;
    if (num_new[i] <= kNarrowTokens || pages < kPrefixMinPages) continue;
    vseq_of[i] = n_vseq++;
    for (int t0 = 0; t0 < num_new[i]; t0 += kPrefixTileTokens)
      prefix.push_back({i, t0, std::min(kPrefixTileTokens, num_new[i] - t0), 0, pages});
  }
  const int split =
      prefix.empty() ? 0
      : pages_per_split > 0
          ? (pages_per_split + kBlockPages - 1) / kBlockPages * kBlockPages
          : fit_split(prefix, std::max(1, num_sms / kTensorHeads), kPrefixMinSplitPages);
  if (!prefix.empty() && pages_per_split == 0 && wide_is_faster(tiles, prefix, split, num_sms)) {
    prefix.clear();
    vseq_of.assign(num_seqs, -1);
    n_vseq = 0;
  }
  if (!prefix.empty()) {
    std::vector<RowsItem> rest;
    for (const RowsItem& t : tiles)
      if (vseq_of[t.seq] < 0) rest.push_back(t);
    for (const RowsItem& p : prefix) {
      const int blocks = p.pe / kBlockPages, ns = (p.pe + split - 1) / split, stride = 2 * p.n_q;
      const int64_t first = rows.part_rows;
      rows.part_rows += static_cast<int64_t>(ns + 1) * stride;
      if (rows.part_rows >= INT32_MAX) {
        ms_host::set_error("ms_tree_plan_build: too many partial rows");
        return MS_ERR_PLAN;
      }
      int pb = 0;
      for (int s = 0; s < ns; ++s) {
        const int len = (blocks / ns + (s < blocks % ns ? 1 : 0)) * kBlockPages;
        tc.push_back({num_seqs + vseq_of[p.seq], p.tok0, p.n_q, pb, pb + len,
                      static_cast<int>(first + static_cast<int64_t>(s) * stride)});
        pb += len;
      }
      for (int t0 = p.tok0; t0 < p.tok0 + p.n_q; t0 += kTileTokens) {
        const int nq = std::min(kTileTokens, p.tok0 + p.n_q - t0);
        const int row0 = static_cast<int>(first) + 2 * (t0 - p.tok0);
        rest.push_back({p.seq, t0, nq, p.pe, (num_cached[p.seq] + t0 + nq + 15) / 16,
                        row0 + ns * stride, static_cast<int>(rows.comb.size()), 3});
        rows.comb.push_back({p.seq, t0, nq, row0, ns + 1, stride, 1, 0});
      }
    }
    tiles.swap(rest);
    std::stable_sort(tc.begin(), tc.end(), [](const RowsItem& x, const RowsItem& y) {
      return (x.pe - x.pb) > (y.pe - y.pb);
    });
  }
  if (!plan_rows(tiles, num_sms, pages_per_split, 0, &rows)) {
    ms_host::set_error("ms_tree_plan_build: too many partial rows");
    return MS_ERR_PLAN;
  }

  const int64_t off_tables = round4((static_cast<int64_t>(num_seqs) + n_vseq) * kRec);
  const int64_t off_narrow = off_tables + round4(total_entries);
  const int64_t off_tile = off_narrow + size4(rows.narrow);
  const int64_t off_tc = off_tile + size4(rows.wide);
  const int64_t off_combine = off_tc + size4(tc);
  const int64_t off_masks = off_combine + size4(rows.comb);
  const int64_t total = off_masks + round4(mask_words);
  if (total > out_capacity) {
    ms_host::set_error("ms_tree_plan_build: output buffer holds " + std::to_string(out_capacity) +
                       " ints, plan needs " + std::to_string(total));
    return MS_ERR_CAPACITY;
  }
  if (total >= (int64_t(1) << 31)) {
    ms_host::set_error("ms_tree_plan_build: plan larger than 2^31 ints");
    return MS_ERR_PLAN;
  }
  std::memset(out, 0, sizeof(int32_t) * total);
  for (int i = 0; i < num_seqs; ++i) {
    const int n = num_new[i], words = (n + 31) / 32;
    int32_t* r = out + static_cast<int64_t>(i) * kRec;
    r[0] = flat_start[i];
    r[1] = n;
    r[2] = num_cached[i];
    r[3] = num_cached[i] + n;
    r[4] = static_cast<int32_t>(table_offsets[i]);
    r[5] = static_cast<int32_t>(table_offsets[i + 1] - table_offsets[i]);
    r[6] = static_cast<int32_t>(off_masks + mask_at[i]);
    r[7] = words;
    if (vseq_of[i] >= 0) {
      const int pages = num_cached[i] / (kBlockPages * 16) * kBlockPages;
      int32_t* v = out + (static_cast<int64_t>(num_seqs) + vseq_of[i]) * kRec;
      v[0] = flat_start[i];
      v[1] = n;
      v[2] = pages * 16;
      v[3] = pages * 16 + n;
      v[4] = r[4];
      v[5] = pages;
    }
    const int32_t* par = parents + parents_at[i];
    uint32_t* mask = reinterpret_cast<uint32_t*>(out + off_masks + mask_at[i]);
    for (int k = 0; k < n; ++k) {
      if (par[k] == -2) continue;
      uint32_t* row = mask + static_cast<int64_t>(k) * words;
      if (par[k] >= 0)
        std::memcpy(row, mask + static_cast<int64_t>(par[k]) * words, sizeof(uint32_t) * words);
      row[k >> 5] |= 1u << (k & 31);
    }
  }
  if (total_entries > 0) std::memcpy(out + off_tables, tables, sizeof(int32_t) * total_entries);
  put_items(out, off_narrow, rows.narrow);
  put_items(out, off_tile, rows.wide);
  put_items(out, off_tc, tc);
  put_items(out, off_combine, rows.comb);

  info->is_tree = 1;
  info->num_seqs = num_seqs;
  info->num_tokens = num_tokens;
  info->n_decode_items = static_cast<int32_t>(rows.narrow.size());
  info->n_tile_items = static_cast<int32_t>(rows.wide.size());
  info->n_combine = static_cast<int32_t>(rows.comb.size());
  info->off_tables = static_cast<int32_t>(off_tables);
  info->off_decode = static_cast<int32_t>(off_narrow);
  info->off_tile = static_cast<int32_t>(off_tile);
  info->n_tc_items = static_cast<int32_t>(tc.size());
  info->off_tc = static_cast<int32_t>(off_tc);
  info->off_combine = static_cast<int32_t>(off_combine);
  info->total_ints = static_cast<int32_t>(total);
  info->pages_per_split = rows.narrow.empty() ? rows.split_wide : rows.split_narrow;
  info->part_rows = rows.part_rows;
  info->total_pages = total_pages;
  for (const RowsItem& c : rows.comb)
    info->combine_tokens_max = std::max<int32_t>(info->combine_tokens_max, c.n_q);
  // Partials and the arrival counters of split tiles.
  info->workspace_bytes_per_kv_head =
      rows.part_rows * (128 + 1) * 4 + static_cast<int64_t>(rows.comb.size()) * 4;
  return MS_OK;
}

extern "C" int ms_tree_plan_build(int32_t num_seqs, const int32_t* flat_start,
                                  const int32_t* num_new, const int32_t* num_cached,
                                  const int64_t* table_offsets, const int32_t* tables,
                                  const int32_t* parents, int32_t num_tokens, int32_t block_size,
                                  int32_t num_sms, int32_t pages_per_split, int32_t* out,
                                  int64_t out_capacity, MsPlanInfo* info) {
  return guarded("ms_tree_plan_build", [&] {
    return tree_plan_build(num_seqs, flat_start, num_new, num_cached, table_offsets, tables, parents,
                           num_tokens, block_size, num_sms, pages_per_split, out, out_capacity, info);
  });
}
