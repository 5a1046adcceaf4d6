// C ABI of the drafted-tree calls: argument checks, planning, dispatch.
// Declared in include/mvr_draft.h.
#include "mvr_draft.h"

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <exception>
#include <memory>
#include <new>
#include <vector>

#include "api_common.hpp"
#include "draft_attention.hpp"
#include "draft_cache.hpp"
#include "paged_attention_kernels.hpp" // kChunkTokens
#include "paged_prefill.hpp" // page_divider

namespace {

using namespace mvr::api;

// ---------------------------------------------------------------------------
// Tree attention
// ---------------------------------------------------------------------------

int check_tree(const mvr_paged_attention_args* a, const mvr_draft_trees* t) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  if (!t) return fail(MVR_E_INVALID_ARGUMENT, "trees is null");
  mvr_paged_attention_args b = *a;
  b.total_q = 0; // empty requests make its lower bound 0
  const int rc = mvr::api::check_attention_scalars(&b);
  if (rc != MVR_OK) return rc;
  if (a->total_q < 0 || a->total_q > (int64_t)a->num_seqs * a->max_q_len)
    return fail(MVR_E_INVALID_ARGUMENT, "total_q %d is outside [0, num_seqs * max_q_len]", a->total_q);
  if (a->num_seqs == 1 && !a->cu_q_lens && a->total_q > 0 && a->total_q < a->max_q_len)
    return fail(MVR_E_INVALID_ARGUMENT, "total_q %d is smaller than max_q_len %d, the q_len of a call without cu_q_lens",
                a->total_q, a->max_q_len);
  if (a->max_seq_len > INT32_MAX - 1024) // (positions of whole key tiles are counted in 32 bits)
    return fail(MVR_E_UNSUPPORTED, "max_seq_len %d is too close to 2^31", a->max_seq_len);
  if (!t->masks) return fail(MVR_E_INVALID_ARGUMENT, "masks is null");
  if ((uintptr_t)t->masks % sizeof(uint32_t)) return fail(MVR_E_INVALID_ARGUMENT, "masks must be 4-byte aligned");
  if (t->mask_words < (a->max_q_len - 1) / 32 + 1)
    return fail(MVR_E_INVALID_ARGUMENT, "mask rows of %d words cannot hold max_q_len %d drafts", t->mask_words,
                a->max_q_len);
  if (a->page_size % mvr::kChunkTokens != 0 && (int64_t)a->page_size * a->head_dim * es_of(a->dtype) > INT32_MAX)
    return fail(MVR_E_UNSUPPORTED, "pages of 2 GiB per KV head whose size is not a multiple of %d tokens",
                mvr::kChunkTokens);
  // The kernels count a page's rows, a head's rows and work items in 32 bits.
  if (a->num_pages > INT32_MAX || (int64_t)a->num_kv_heads * a->page_size > INT32_MAX)
    return fail(MVR_E_UNSUPPORTED, "pools of over 2^31 pages, or pages of over 2^31 rows");
  const int64_t group = a->num_q_heads / a->num_kv_heads;
  const int64_t pairs = (int64_t)a->num_seqs * a->num_kv_heads + mvr::kDraftXcds - 1;
  const int64_t tiles = pairs * ((group * a->max_q_len + 15) / 16);
  if (group * a->max_q_len > INT32_MAX || tiles > kMaxThreads / 256)
    return fail(MVR_E_UNSUPPORTED, "%d requests of %d drafts are more than one call takes", a->num_seqs, a->max_q_len);
  return MVR_OK;
}

int64_t units_of(int64_t tokens) { return (tokens + mvr::kDraftUnitTokens - 1) / mvr::kDraftUnitTokens; }

constexpr int kTileSizes = 4;
constexpr int kTileRowsLog2[kTileSizes] = {4, 5, 6, 7};

// The requests as the planner sees them: the host tables where they are given and
// within the call's bounds, else every request at those bounds.  Two passes over the
// tables, whatever is planned on them afterwards: they leave, for each tile size, the
// row tiles of requests of each length, from whose sums over the longer lengths a
// split's parts are counted in a few look-ups (64 at most, a request's most parts).
class Requests {
 public:
  explicit Requests(const mvr_paged_attention_args* a) : hkv_(a->num_kv_heads) {
    const int64_t group = a->num_q_heads / a->num_kv_heads;
    tables_ = read_bounds(a);
    if (!tables_) {
      // sum_seq_lens alone tells the average context: requests of other lengths round
      // up to a unit and a part more each.
      const int64_t tokens = a->sum_seq_lens > 0 ? (a->sum_seq_lens + a->num_seqs - 1) / a->num_seqs : a->max_seq_len;
      const int64_t rows = group * a->max_q_len;
      longest = shortest = units_of(tokens);
      more_ = tokens < a->max_seq_len;
      all_units = a->num_seqs * longest;
      for (int t = 0; t < kTileSizes; t++) {
        tiles[t] = a->num_seqs * hkv_ * tiles_of(rows, t);
        work[t] = tiles[t] * longest;
      }
      return;
    }
    while (longest >> scale_ >= kBuckets) scale_++;
    const int top = bucket(longest);
    std::fill(longest_in_, longest_in_ + top + 1, 0);
    for (int t = 0; t < kTileSizes; t++) std::fill(from_[t], from_[t] + top + 2, 0);
    for (int s = 0; s < a->num_seqs; s++) {
      const int64_t rows = group * (a->cu_q_lens_host[s + 1] - a->cu_q_lens_host[s]);
      if (rows == 0) continue;
      const int64_t units = units_of(a->seq_lens_host[s]);
      const int b = bucket(units);
      all_units += units;
      longest_in_[b] = b;
      for (int t = 0; t < kTileSizes; t++) {
        const int64_t n = tiles_of(rows, t);
        from_[t][b] += (int32_t)n;
        tiles[t] += n;
        work[t] += n * units;
      }
    }
    for (int b = 1; b <= top; b++) longest_in_[b] = std::max(longest_in_[b], longest_in_[b - 1]);
    for (int t = 0; t < kTileSizes; t++) {
      for (int b = top - 1; b >= 1; b--) from_[t][b] += from_[t][b + 1];
      tiles[t] *= hkv_;
      work[t] *= hkv_;
    }
  }

  // Items of the tile size where every request is split in parts of at most `part`
  // units (kDraftMaxParts parts at most).  (Lengths of kBuckets units or more count as
  // rounded up by 1 / 512 at most.)
  int64_t items(int t, int64_t part) const {
    if (!tables_) return tiles[t] * uniform_parts(part);
    const int64_t end = longest_counted();
    int64_t n = 0, at = 0; // a request has a k-th part where it is longer than k parts
    for (int k = 0; k < mvr::kDraftMaxParts && at < end; k++, at += part) n += from_[t][(at >> scale_) + 1];
    return n * hkv_;
  }

  // Units of the longest part then.
  int64_t longest_part(int64_t part) const {
    if (!tables_) return (longest + uniform_parts(part) - 1) / uniform_parts(part);
    const int64_t end = longest_counted();
    const int64_t most = std::min<int64_t>((end + part - 1) / part, mvr::kDraftMaxParts);
    int64_t best = (end + most - 1) / most;
    for (int64_t k = 1; k < most && best < part; k++) { // the longest request of k parts
      const int64_t units = (int64_t)longest_in_[(k * part) >> scale_] << scale_;
      if (units > (k - 1) * part) best = std::max(best, (units + k - 1) / k);
    }
    return best;
  }

  bool from_tables() const { return tables_; }

  int64_t longest = 0, shortest = 0;           // units; 0: no request has drafts
  int64_t all_units = 0;                       // of all requests
  int64_t tiles[kTileSizes] = {};              // row tiles, over the KV heads
  int64_t work[kTileSizes] = {};               // tiles x units

 private:
  static constexpr int kBuckets = 1024; // of units, 2^scale_ each

  static int64_t tiles_of(int64_t rows, int t) { return (rows + (1 << kTileRowsLog2[t]) - 1) >> kTileRowsLog2[t]; }
  int bucket(int64_t units) const { return (int)((units + ((int64_t)1 << scale_) - 1) >> scale_); }
  int64_t longest_counted() const { return (int64_t)bucket(longest) << scale_; }
  int64_t uniform_parts(int64_t part) const {
    return std::min<int64_t>((longest + more_ + part - 1) / part + more_, mvr::kDraftMaxParts);
  }

  // Longest and shortest of the requests with drafts; false where the tables are not
  // given or leave the call's bounds.
  bool read_bounds(const mvr_paged_attention_args* a) {
    const int32_t* cu = a->cu_q_lens_host;
    const int32_t* sl = a->seq_lens_host;
    if (!cu || !sl) return false;
    int32_t most = 0, least = INT32_MAX;
    for (int s = 0; s < a->num_seqs; s++) {
      const int64_t q = (int64_t)cu[s + 1] - cu[s];
      if (q < 0 || q > a->max_q_len || sl[s] < q || sl[s] > a->max_seq_len) return false;
      if (q == 0) continue;
      most = std::max(most, sl[s]);
      least = std::min(least, sl[s]);
    }
    if (most > 0) {
      longest = units_of(most);
      shortest = units_of(least);
    }
    return true;
  }

  int64_t hkv_;
  bool tables_;
  int64_t more_ = 0; // units and parts that a request may have beyond the average
  int scale_ = 0;
  int32_t from_[kTileSizes][kBuckets + 2]; // [t][b]: row tiles (of a KV head) of the requests of bucket b or longer
  int32_t longest_in_[kBuckets + 2];       // [b]: the longest bucket up to b that holds a request, or 0
};

// What a block of one tile size costs, in us, for head_dim 128: `fixed` beside
// its keys, `unit` per 64 keys with one to four blocks on its CU.  Fitted to 965
// timed plans (tile sizes and splits of 53 calls: 1 to 64 requests on 100 to 16,000
// tokens, 1 to 840 rows per KV head, head_dim 64 and 128, both types).  Timed again
// since, the plan that these costs make fastest takes 0.9% longer than the fastest of
// 989 plans of those calls on average, 12% at most (4 drafts on 4,000 keys); on 20
// calls of other head dimensions and page sizes 6%, and 28 to 44% on F16 calls of many
// rows on 5-token pages and of head_dim 32: neither has costs of its own.  F32 products
// take 7 times as long as F16 ones.
struct TileCost {
  int rows;
  double fixed, unit[4];
};

constexpr TileCost kF16Costs[] = {{16, 6.3, {0.57, 1.17, 1.81, 2.48}}, {32, 6.3, {0.75, 1.55, 2.33, 2.33}},
                                  {64, 6.6, {1.02, 1.30, 1.30, 1.30}}, {128, 8.0, {1.32, 1.62, 1.62, 1.62}}};
constexpr TileCost kF32Costs[] = {{16, 2.5, {1.97, 4.05, 6.23, 8.55}}, {32, 5.8, {3.06, 5.80, 7.43, 7.43}},
                                  {64, 5.7, {4.73, 9.50, 9.50, 9.50}}, {128, 6.6, {7.61, 14.8, 14.8, 14.8}}};

// The tile size and the split of its keys that these costs make fastest: every
// tile whole, or in parts that give each CU one block, two, up to as many as it
// holds, or two, three or four times that.  A call takes its blocks' time (all of
// them in one round; in more rounds the average load and most of a last block, the
// shortest where the longest start first), joined with the time that its keys take
// from HBM (as a 3-norm: 128 blocks of 126 units and a bound of 89 us ran in 119,
// 256 of 63 in 98).  A split call scans the lengths and merges: 4.5 us, and its
// partial results written and read at 4.3 TB/s.
mvr::DraftAttentionPlan plan_tree(const mvr_paged_attention_args* a, size_t limit) {
  const bool f16 = a->dtype == MVR_DTYPE_F16;
  const Requests requests(a);
  const int64_t longest = requests.longest, shortest = requests.shortest;
  const double unit_scale = a->head_dim / 128.0;
  const int64_t cus = mvr::api::compute_units(), hkv = a->num_kv_heads;
  const int64_t longest_rows = (int64_t)(a->num_q_heads / a->num_kv_heads) * a->max_q_len;
  const double hbm = requests.all_units * (2.0 * mvr::kDraftUnitTokens * hkv * a->head_dim * es_of(a->dtype) / 5.9e6);
  // Overrides, for tests and tuning: a tile size that the head dimension has, and
  // its parts.
  static const int set_rows = mvr::api::env_int("MVR_DRAFT_TILE_ROWS", 0);
  static const int set_units = mvr::api::env_int("MVR_DRAFT_PART_UNITS", 0);
  bool rows_set = false;
  for (const TileCost& tile : kF16Costs)
    rows_set |= tile.rows == set_rows && mvr::draft_tile_supported(set_rows, a->head_dim);
  mvr::DraftAttentionPlan best{};
  double best_cost = INFINITY;
  for (int t = 0; t < kTileSizes; t++) {
    const TileCost& tile = f16 ? kF16Costs[t] : kF32Costs[t];
    if (!mvr::draft_tile_supported(tile.rows, a->head_dim)) continue;
    // (A tile that no request fills half costs what the smaller one does, or more.)
    if (rows_set ? tile.rows != set_rows : longest_rows <= tile.rows / 2 && best_cost < INFINITY) continue;
    const int held = mvr::draft_blocks_per_cu(tile.rows, f16, a->head_dim);
    const int64_t tiles = requests.tiles[t], work = requests.work[t];
    auto cost_of = [&](int64_t blocks, int64_t part, int64_t last) { // of `part` units at most, the last one of `last`
      double body;
      if (blocks <= held * cus)
        body = part * tile.unit[std::max<int64_t>(0, (blocks + cus - 1) / cus - 1)];
      else
        body = std::max(work * tile.unit[held - 1] / (held * cus) + 0.87 * last * tile.unit[0], part * tile.unit[0]) + 6.1;
      body *= unit_scale;
      return tile.fixed + cbrt(body * body * body + hbm * hbm * hbm);
    };
    auto take = [&](double cost, int64_t part, int64_t items, size_t bytes) {
      if (!(cost < best_cost)) return;
      best_cost = cost;
      best.tile_rows = tile.rows;
      best.row_tiles = (int)((longest_rows + tile.rows - 1) / tile.rows);
      best.part_units = (int)part;
      best.max_items = (int)items;
      // Not split: the pairs of request and KV head by eights.
      const int64_t pairs = (a->num_seqs * hkv + mvr::kDraftXcds - 1) / mvr::kDraftXcds * mvr::kDraftXcds;
      best.blocks = (int)(part ? items : pairs * best.row_tiles);
      // (Finding a length's rank takes 0.3 us: not where all are alike, or start at once.)
      best.by_length = part == 0 && best.blocks > cus && (!requests.from_tables() || shortest < longest);
      best.partial_bytes = bytes;
    };
    auto bytes_of = [&](int64_t items) {
      return align_up((size_t)items * tile.rows * a->head_dim * sizeof(float), 256) +
             align_up((size_t)items * tile.rows * 2 * sizeof(float), 256);
    };
    auto take_split = [&](int64_t part) {
      const int64_t items = requests.items(t, part), part_longest = requests.longest_part(part);
      const size_t bytes = bytes_of(items);
      take(cost_of(items, part_longest, part_longest) + 4.5 + 2 * bytes / 4.3e6, part, items, bytes);
    };
    // (The blocks of a split call and of its merge have to fit a launch each.)
    const bool may_split = limit > 0 && longest > 1 &&
                           a->num_seqs * hkv * ((longest_rows + 15) / 16) <= kMaxThreads / 256 / 64;
    if (may_split && set_units && set_units < longest && bytes_of(requests.items(t, set_units)) <= limit) {
      take_split(set_units);
      continue;
    }
    take(cost_of(tiles, longest, shortest), 0, 0, 0);
    if (!may_split || set_units) continue;
    int64_t last = 0;
    for (int64_t target = cus; target <= 4 * held * cus; target += target < held * cus ? cus : held * cus) {
      if (tiles >= target) continue;
      // The shortest parts whose blocks are no more than `target`, in steps of 1/16: from
      // an estimate (a request's last part is half full on average) upwards.  Longer
      // parts are fewer: bisected, from the length whose parts are few enough even where
      // every request's last one holds a single unit.
      auto fits = [&](int64_t part) {
        const int64_t items = requests.items(t, part);
        return items <= target && bytes_of(items) <= limit;
      };
      int64_t part = std::max<int64_t>(1, work / (target - tiles / 2));
      if (part >= longest) continue;
      if (!fits(part)) {
        int64_t below = part, above = std::min(longest - 1, std::max(part + 1, work / (target - tiles) + 1));
        if (!fits(above)) {
          below = above;
          above = longest - 1;
          if (below >= above || !fits(above)) continue;
        }
        while (above - below > 1) {
          const int64_t middle = below + (above - below) / 2;
          (fits(middle) ? above : below) = middle;
        }
        while (part < above) part += 1 + part / 16;
      }
      if (part < longest && part != last) take_split(part);
      last = part;
    }
  }
  return best;
}

} // namespace

extern "C" {

size_t mvr_paged_attention_tree_workspace_size(const mvr_paged_attention_args* a, const mvr_draft_trees* t) {
  if (check_tree(a, t) != MVR_OK) return 0;
  return plan_tree(a, SIZE_MAX).partial_bytes;
}

int mvr_paged_attention_tree_validate(const mvr_paged_attention_args* a, const mvr_draft_trees* t,
                                      const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                      const int32_t* cu_q_lens_host, const uint32_t* masks_host) {
  mvr::api::clear_error();
  const int rc = check_tree(a, t);
  if (rc != MVR_OK) return rc;
  if (cu_q_lens_host && check_cu_q_lens(cu_q_lens_host, a->num_seqs, a->total_q, a->max_q_len) != MVR_OK)
    return MVR_E_INVALID_ARGUMENT;
  for (int s = 0; s < a->num_seqs; s++) {
    int64_t q_len = a->num_seqs == 1 ? a->max_q_len : -1, at = 0;
    if (cu_q_lens_host) {
      at = cu_q_lens_host[s];
      q_len = (int64_t)cu_q_lens_host[s + 1] - at;
    }
    const int64_t seq_len = seq_lens_host ? seq_lens_host[s] : a->num_seqs == 1 ? a->max_seq_len : -1;
    if (seq_lens_host) {
      if (seq_len < 0 || seq_len > a->max_seq_len)
        return fail(MVR_E_INVALID_ARGUMENT, "request %d has seq_len %lld outside [0, max_seq_len %d]", s,
                    (long long)seq_len, a->max_seq_len);
      if (q_len >= 0 && seq_len < q_len)
        return fail(MVR_E_LENGTH_MISMATCH, "paged KV cache reports sequence length %lld, expected at least %lld",
                    (long long)seq_len, (long long)q_len);
    }
    if (block_tables_host && seq_len >= 0 && q_len != 0)
      for (int64_t pi = 0; pi < (seq_len + a->page_size - 1) / a->page_size; pi++) {
        const int32_t id = block_tables_host[(int64_t)s * a->max_pages_per_seq + pi];
        if (id < 0 || id >= a->num_pages)
          return fail(MVR_E_PAGE_ID, "request %d page %lld has id %d outside a pool of %lld pages", s, (long long)pi, id,
                      (long long)a->num_pages);
      }
    if (masks_host && q_len > 0)
      for (int64_t i = 0; i < q_len; i++)
        if (!(masks_host[(at + i) * t->mask_words + i / 32] >> (i % 32) & 1))
          return fail(MVR_E_INVALID_ARGUMENT, "request %d: draft %lld does not see itself", s, (long long)i);
  }
  return MVR_OK;
}

int mvr_paged_attention_tree(const mvr_paged_attention_args* a, const mvr_draft_trees* t) {
  mvr::api::Range range("attn"); // trace.rs:64
  mvr::api::clear_error();
  int rc = check_tree(a, t);
  if (rc != MVR_OK) return rc;
  if (mvr::api::checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> bt, sl, cu;
      if (!mvr::api::copy_to_host(a->block_tables, (size_t)a->num_seqs * a->max_pages_per_seq, a->stream, bt) ||
          !mvr::api::copy_to_host(a->seq_lens, a->num_seqs, a->stream, sl) ||
          !mvr::api::copy_to_host(a->cu_q_lens, (size_t)a->num_seqs + 1, a->stream, cu))
        return copy_failed();
      return mvr_paged_attention_tree_validate(a, t, data_or_null(bt), data_or_null(sl), data_or_null(cu), nullptr);
    });
    if (rc != MVR_OK) return rc;
  }
  if (a->workspace && ((uintptr_t)a->workspace & 255u))
    return fail(MVR_E_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  const mvr::DraftAttentionPlan plan = plan_tree(a, a->workspace ? a->workspace_bytes : 0);
  mvr::DraftAttentionParams p{};
  p.q = a->q;
  p.q_stride_head = a->q_stride_head;
  p.q_stride_token = a->q_stride_token;
  p.key_pool = a->key_pool;
  p.value_pool = a->value_pool;
  p.block_tables = a->block_tables;
  p.block_table_stride = a->max_pages_per_seq;
  p.seq_lens = a->seq_lens;
  p.cu_q_lens = a->cu_q_lens;
  p.max_seq_len = a->max_seq_len;
  p.max_q_len = a->max_q_len;
  p.out = a->out;
  p.out_stride_head = a->out_stride_head;
  p.out_stride_token = a->out_stride_token;
  p.masks = t->masks;
  p.mask_words = t->mask_words;
  p.num_seqs = a->num_seqs;
  p.num_kv_heads = a->num_kv_heads;
  p.group_size = a->num_q_heads / a->num_kv_heads;
  p.page_size = a->page_size;
  p.last_page = (uint32_t)(a->num_pages - 1);
  mvr::page_divider(a->page_size, p.page_magic, p.page_magic_shift);
  p.row_tiles = plan.row_tiles;
  p.part_units = plan.part_units;
  p.max_items = plan.max_items;
  p.by_length = plan.by_length;
  if (plan.max_items) {
    p.partial_o = static_cast<float*>(a->workspace);
    p.partial_ml = reinterpret_cast<float*>(
        static_cast<char*>(a->workspace) +
        align_up((size_t)plan.max_items * plan.tile_rows * a->head_dim * sizeof(float), 256));
  }
  const float scale = a->scale > 0.f ? a->scale : (float)(1.0 / sqrt((double)a->head_dim));
  p.scale_log2 = scale * 1.4426950408889634f;
  mvr::api::Range launch("attn-paged-fused");
  return launch_status(
      mvr::launch_draft_attention(plan, p, a->dtype, a->head_dim, static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// Norm, rotation and append
// ---------------------------------------------------------------------------

static int check_norm_rope_append(const mvr_rope_append_args* a, const mvr_head_norms* n) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  if (!n) return fail(MVR_E_INVALID_ARGUMENT, "norms is null");
  if (a->dtype != MVR_DTYPE_F32 && a->dtype != MVR_DTYPE_F16)
    return fail(MVR_E_UNSUPPORTED, "dtype %d is not F32 (0) or F16 (1)", a->dtype);
  if (a->rope_type != MVR_ROPE_NEOX && a->rope_type != MVR_ROPE_INTERLEAVED)
    return fail(MVR_E_UNSUPPORTED, "rope_type %d is not Neox (0) or Interleaved (1)", a->rope_type);
  if (a->num_seqs < 1) return fail(MVR_E_INVALID_ARGUMENT, "forward requires at least one request");
  if (a->num_kv_heads < 1 || a->num_q_heads < 1 || a->num_q_heads % a->num_kv_heads != 0)
    return fail(MVR_E_INVALID_ARGUMENT, "num_q_heads %d is not a multiple of num_kv_heads %d", a->num_q_heads,
                a->num_kv_heads);
  if (a->head_dim < 8 || a->head_dim > 512 || a->head_dim % 8 != 0)
    return fail(MVR_E_UNSUPPORTED, "head_dim %d is not a multiple of 8 in [8, 512]", a->head_dim);
  if (a->page_size < 1) return fail(MVR_E_INVALID_ARGUMENT, "page_size must be positive");
  if (a->num_pages < 1) return fail(MVR_E_INVALID_ARGUMENT, "num_pages must be positive");
  if (a->total_q < 1) return fail(MVR_E_INVALID_ARGUMENT, "cannot append an empty KV-cache tensor"); // kv_cache/utils.rs:33-36
  if (a->max_seq_len < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_seq_len must be positive");
  if (a->rope_len < 1) return fail(MVR_E_INVALID_ARGUMENT, "rope_len must be positive");
  if (!n->positions && a->rope_len < a->max_seq_len)
    return fail(MVR_E_INVALID_ARGUMENT, "rotary tables hold %d positions, max_seq_len is %d", a->rope_len,
                a->max_seq_len);
  const int64_t pages_needed = (a->max_seq_len + (int64_t)a->page_size - 1) / a->page_size;
  if (a->max_pages_per_seq < pages_needed)
    return fail(MVR_E_PAGES_UNCOVERED, "block table rows of %d pages cannot hold %d tokens of %d-token pages",
                a->max_pages_per_seq, a->max_seq_len, a->page_size);
  if (a->num_seqs > 1 && (!a->seq_lens || !a->cu_q_lens))
    return fail(MVR_E_INVALID_ARGUMENT, "seq_lens and cu_q_lens are required when num_seqs > 1");
  if (!a->q || !a->k || !a->v || !a->cos_table || !a->sin_table || !a->block_tables || !a->q_out || !a->key_pool ||
      !a->value_pool)
    return fail(MVR_E_INVALID_ARGUMENT, "null tensor, table or pool pointer");
  if (a->num_q_heads > INT32_MAX / 4 / 64 || // (rows of a token and their lanes, in 32 bits)
      a->total_q > kMaxThreads / 64 / mvr::append_token_waves(a->num_q_heads + 2 * a->num_kv_heads, a->head_dim))
    return fail(MVR_E_UNSUPPORTED, "%d tokens of %d and 2 x %d heads are more than one call takes", a->total_q,
                a->num_q_heads, a->num_kv_heads);
  if (!(n->eps >= 0.f) || !isfinite(n->eps)) return fail(MVR_E_INVALID_ARGUMENT, "eps must be finite and >= 0");
  const size_t align = a->dtype == MVR_DTYPE_F16 ? 8 : 16; // every access moves 4 elements
  const void* ptrs[] = {a->q,        a->k,          a->v,       a->cos_table, a->sin_table, a->q_out,
                        a->key_pool, a->value_pool, n->q_weight, n->k_weight};
  for (const void* ptr : ptrs)
    if ((uintptr_t)ptr % align)
      return fail(MVR_E_INVALID_ARGUMENT, "tensors, tables, weights and pools must be %zu-byte aligned", align);
  const int64_t strides[] = {a->q_stride_head, a->q_stride_token, a->k_stride_head,     a->k_stride_token,
                             a->v_stride_head, a->v_stride_token, a->q_out_stride_head, a->q_out_stride_token};
  for (int64_t st : strides)
    if (st % 4) return fail(MVR_E_INVALID_ARGUMENT, "strides must be multiples of 4 elements");
  return MVR_OK;
}

int mvr_norm_rope_append_validate(const mvr_rope_append_args* a, const mvr_head_norms* n,
                                  const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                  const int32_t* cu_q_lens_host, const int32_t* positions_host,
                                  const uint8_t* page_writable_host) {
  mvr::api::clear_error();
  const int rc = check_norm_rope_append(a, n);
  if (rc != MVR_OK) return rc;
  if (cu_q_lens_host && check_cu_q_lens(cu_q_lens_host, a->num_seqs, a->total_q) != MVR_OK)
    return MVR_E_INVALID_ARGUMENT;
  // Pages that an earlier request of this call writes (two writers would race).
  std::unique_ptr<uint8_t[]> written;
  if (block_tables_host) {
    written.reset(new (std::nothrow) uint8_t[(size_t)a->num_pages]());
    if (!written) return fail(MVR_E_INVALID_ARGUMENT, "out of host memory");
  }
  for (int s = 0; s < a->num_seqs; s++) {
    if (!cu_q_lens_host && a->num_seqs > 1) break;
    const int64_t at = cu_q_lens_host ? cu_q_lens_host[s] : 0;
    const int64_t q_len = cu_q_lens_host ? (int64_t)cu_q_lens_host[s + 1] - at : a->total_q;
    if (positions_host && n->positions)
      for (int64_t i = at; i < at + q_len; i++)
        if (positions_host[i] < 0 || positions_host[i] >= a->rope_len)
          return fail(MVR_E_INVALID_ARGUMENT, "token %lld has position %d outside the rotary tables of %d positions",
                      (long long)i, positions_host[i], a->rope_len);
    if (!seq_lens_host && a->num_seqs > 1) continue;
    const int64_t seq_len = seq_lens_host ? seq_lens_host[s] : a->max_seq_len;
    if (q_len == 0) continue;
    if (seq_len > a->max_seq_len)
      return fail(MVR_E_INVALID_ARGUMENT, "request %d has seq_len %lld > max_seq_len %d", s, (long long)seq_len,
                  a->max_seq_len);
    if (seq_len < q_len)
      return fail(MVR_E_LENGTH_MISMATCH, "KV-cache contains %lld tokens after appending %lld", (long long)seq_len,
                  (long long)q_len);
    if (!block_tables_host) continue;
    for (int64_t pi = (seq_len - q_len) / a->page_size; pi <= (seq_len - 1) / a->page_size; pi++) {
      const int32_t id = block_tables_host[(int64_t)s * a->max_pages_per_seq + pi];
      if (id < 0 || id >= a->num_pages)
        return fail(MVR_E_PAGE_ID, "request %d page %lld has id %d outside a pool of %lld pages", s, (long long)pi, id,
                    (long long)a->num_pages);
      if (page_writable_host && !page_writable_host[id])
        return fail(MVR_E_READ_ONLY_PAGE, "cannot mutate written physical page %d", id); // physical_page_pool.rs:197-201
      if (written[id]) return fail(MVR_E_INVALID_ARGUMENT, "page %d is written by more than one request", id);
      written[id] = 1;
    }
  }
  return MVR_OK;
}

int mvr_norm_rope_append(const mvr_rope_append_args* a, const mvr_head_norms* n) {
  mvr::api::Range range("attn-rope tensor=query,key"); // trace.rs:77-79
  mvr::api::clear_error();
  int rc = check_norm_rope_append(a, n);
  if (rc != MVR_OK) return rc;
  if (mvr::api::checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> bt, sl, cu, pos;
      if (!mvr::api::copy_to_host(a->block_tables, (size_t)a->num_seqs * a->max_pages_per_seq, a->stream, bt) ||
          !mvr::api::copy_to_host(a->seq_lens, a->num_seqs, a->stream, sl) ||
          !mvr::api::copy_to_host(a->cu_q_lens, (size_t)a->num_seqs + 1, a->stream, cu) ||
          !mvr::api::copy_to_host(n->positions, a->total_q, a->stream, pos))
        return copy_failed();
      return mvr_norm_rope_append_validate(a, n, data_or_null(bt), data_or_null(sl), data_or_null(cu), data_or_null(pos),
                                           nullptr);
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::NormRopeAppendParams p{};
  p.q = a->q;
  p.q_stride_head = a->q_stride_head;
  p.q_stride_token = a->q_stride_token;
  p.k = a->k;
  p.k_stride_head = a->k_stride_head;
  p.k_stride_token = a->k_stride_token;
  p.v = a->v;
  p.v_stride_head = a->v_stride_head;
  p.v_stride_token = a->v_stride_token;
  p.q_weight = n->q_weight;
  p.k_weight = n->k_weight;
  p.eps = n->eps;
  p.cos_table = a->cos_table;
  p.sin_table = a->sin_table;
  p.positions = n->positions;
  p.rope_len = a->rope_len;
  p.block_tables = a->block_tables;
  p.block_table_stride = a->max_pages_per_seq;
  p.seq_lens = a->seq_lens;
  p.cu_q_lens = a->cu_q_lens;
  p.max_seq_len = a->max_seq_len;
  p.q_out = a->q_out;
  p.q_out_stride_head = a->q_out_stride_head;
  p.q_out_stride_token = a->q_out_stride_token;
  p.key_pool = a->key_pool;
  p.value_pool = a->value_pool;
  p.num_pages = a->num_pages;
  p.num_seqs = a->num_seqs;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.head_dim = a->head_dim;
  p.page_size = a->page_size;
  p.total_q = a->total_q;
  mvr::api::Range append("attn-cache operation=append"); // trace.rs:81-83
  return launch_status(
      mvr::launch_norm_rope_append(p, a->dtype, a->rope_type, static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// Compaction
// ---------------------------------------------------------------------------

static int check_compact(const mvr_compact_drafts_args* a) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  const int rc =
      check_pool(a->dtype, a->num_kv_heads, a->head_dim, a->page_size, a->num_pages, a->key_pool, a->value_pool);
  if (rc != MVR_OK) return rc;
  if (a->num_layers < 1) return fail(MVR_E_INVALID_ARGUMENT, "num_layers must be positive");
  if (a->num_seqs < 1) return fail(MVR_E_INVALID_ARGUMENT, "forward requires at least one request");
  if (a->max_seq_len < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_seq_len must be positive");
  if (a->max_accepted < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_accepted must be positive");
  const int64_t pages_needed = (a->max_seq_len + (int64_t)a->page_size - 1) / a->page_size;
  if (a->max_pages_per_seq < pages_needed)
    return fail(MVR_E_PAGES_UNCOVERED, "block table rows of %d pages cannot hold %d tokens of %d-token pages",
                a->max_pages_per_seq, a->max_seq_len, a->page_size);
  if (!a->block_tables || !a->seq_lens || !a->cu_q_lens || !a->accepted || !a->accepted_lens)
    return fail(MVR_E_INVALID_ARGUMENT, "null table pointer");
  if ((int64_t)a->num_layers * a->num_seqs > kMaxThreads / 64 / a->num_kv_heads)
    return fail(MVR_E_UNSUPPORTED, "more layers, requests and KV heads than one call takes");
  // Every head and layer reads the tables, one writes the new lengths.
  auto overlaps = [a](const int32_t* table, int64_t entries) {
    return a->new_seq_lens && (uintptr_t)a->new_seq_lens < (uintptr_t)(table + entries) &&
           (uintptr_t)table < (uintptr_t)(a->new_seq_lens + a->num_seqs);
  };
  if (overlaps(a->seq_lens, a->num_seqs)) return fail(MVR_E_INVALID_ARGUMENT, "new_seq_lens must not overlap seq_lens");
  if (overlaps(a->cu_q_lens, (int64_t)a->num_seqs + 1) || overlaps(a->accepted_lens, a->num_seqs) ||
      overlaps(a->accepted, (int64_t)a->num_seqs * a->max_accepted) ||
      overlaps(a->block_tables, (int64_t)a->num_layers * a->num_seqs * a->max_pages_per_seq))
    return fail(MVR_E_INVALID_ARGUMENT, "new_seq_lens must not overlap another table");
  return MVR_OK;
}

int mvr_compact_drafts_validate(const mvr_compact_drafts_args* a, const int32_t* block_tables_host,
                                const int32_t* seq_lens_host, const int32_t* cu_q_lens_host,
                                const int32_t* accepted_host, const int32_t* accepted_lens_host) {
  mvr::api::clear_error();
  const int rc = check_compact(a);
  if (rc != MVR_OK) return rc;
  if (cu_q_lens_host && check_cu_q_lens(cu_q_lens_host, a->num_seqs, 0) != MVR_OK) return MVR_E_INVALID_ARGUMENT;
  std::unique_ptr<uint8_t[]> written;
  if (block_tables_host) {
    written.reset(new (std::nothrow) uint8_t[(size_t)a->num_pages]());
    if (!written) return fail(MVR_E_INVALID_ARGUMENT, "out of host memory");
  }
  for (int s = 0; s < a->num_seqs; s++) {
    const int64_t q_len = cu_q_lens_host ? (int64_t)cu_q_lens_host[s + 1] - cu_q_lens_host[s] : -1;
    if (seq_lens_host) {
      if (seq_lens_host[s] < 0 || seq_lens_host[s] > a->max_seq_len)
        return fail(MVR_E_INVALID_ARGUMENT, "request %d has seq_len %d outside [0, max_seq_len %d]", s, seq_lens_host[s],
                    a->max_seq_len);
      if (seq_lens_host[s] < q_len)
        return fail(MVR_E_LENGTH_MISMATCH, "paged KV cache reports sequence length %d, expected at least %lld",
                    seq_lens_host[s], (long long)q_len);
    }
    if (!accepted_lens_host) continue;
    const int count = accepted_lens_host[s];
    if (count < 0 || count > a->max_accepted || (q_len >= 0 && count > q_len))
      return fail(MVR_E_INVALID_ARGUMENT, "request %d accepts %d of its drafts, more than it has (or max_accepted)", s,
                  count);
    if (!accepted_host) continue;
    const int32_t* list = accepted_host + (int64_t)s * a->max_accepted;
    for (int j = 0; j < count; j++) {
      if (list[j] < 0 || (q_len >= 0 && list[j] >= q_len))
        return fail(MVR_E_INVALID_ARGUMENT, "request %d accepts draft %d, outside its drafts", s, list[j]);
      if (j > 0 && list[j] <= list[j - 1])
        return fail(MVR_E_INVALID_ARGUMENT, "request %d: accepted drafts must ascend (%d after %d)", s, list[j],
                    list[j - 1]);
    }
    if (!block_tables_host || !seq_lens_host || q_len < 0 || count == 0) continue;
    // Pages that hold the accepted rows: read or written up to the last one.
    const int64_t first = seq_lens_host[s] - q_len, last = first + list[count - 1];
    for (int layer = 0; layer < a->num_layers; layer++)
      for (int64_t pi = first / a->page_size; pi <= last / a->page_size; pi++) {
        const int32_t id =
            block_tables_host[((int64_t)layer * a->num_seqs + s) * a->max_pages_per_seq + pi];
        if (id < 0 || id >= a->num_pages)
          return fail(MVR_E_PAGE_ID, "layer %d request %d page %lld has id %d outside a pool of %lld pages", layer, s,
                      (long long)pi, id, (long long)a->num_pages);
        if (written[id])
          return fail(MVR_E_INVALID_ARGUMENT, "page %d holds the drafts of more than one request or layer", id);
        written[id] = 1;
      }
  }
  return MVR_OK;
}

int mvr_compact_drafts(const mvr_compact_drafts_args* a) {
  mvr::api::Range range("attn-cache operation=compact");
  mvr::api::clear_error();
  int rc = check_compact(a);
  if (rc != MVR_OK) return rc;
  if (mvr::api::checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> bt, sl, cu, acc, lens;
      if (!mvr::api::copy_to_host(a->block_tables, (size_t)a->num_layers * a->num_seqs * a->max_pages_per_seq,
                                  a->stream, bt) ||
          !mvr::api::copy_to_host(a->seq_lens, a->num_seqs, a->stream, sl) ||
          !mvr::api::copy_to_host(a->cu_q_lens, (size_t)a->num_seqs + 1, a->stream, cu) ||
          !mvr::api::copy_to_host(a->accepted, (size_t)a->num_seqs * a->max_accepted, a->stream, acc) ||
          !mvr::api::copy_to_host(a->accepted_lens, a->num_seqs, a->stream, lens))
        return copy_failed();
      return mvr_compact_drafts_validate(a, bt.data(), sl.data(), cu.data(), acc.data(), lens.data());
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::CompactDraftsParams p{};
  p.key_pool = a->key_pool;
  p.value_pool = a->value_pool;
  p.block_tables = a->block_tables;
  p.block_table_stride = a->max_pages_per_seq;
  p.seq_lens = a->seq_lens;
  p.cu_q_lens = a->cu_q_lens;
  p.accepted = a->accepted;
  p.accepted_lens = a->accepted_lens;
  p.new_seq_lens = a->new_seq_lens;
  p.num_pages = a->num_pages;
  p.num_layers = a->num_layers;
  p.num_seqs = a->num_seqs;
  p.num_kv_heads = a->num_kv_heads;
  p.page_size = a->page_size;
  p.max_seq_len = a->max_seq_len;
  p.max_accepted = a->max_accepted;
  return launch_status(
      mvr::launch_compact_drafts(p, (int64_t)a->head_dim * es_of(a->dtype), static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// Copies of pages
// ---------------------------------------------------------------------------

static int check_copy(const mvr_copy_pages_args* a) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  const int rc =
      check_pool(a->dtype, a->num_kv_heads, a->head_dim, a->page_size, a->num_pages, a->key_pool, a->value_pool);
  if (rc != MVR_OK) return rc;
  if (a->num_copies < 0) return fail(MVR_E_INVALID_ARGUMENT, "num_copies must not be negative");
  if (a->num_copies > 0 && (!a->src_pages || !a->dst_pages))
    return fail(MVR_E_INVALID_ARGUMENT, "null page list pointer");
  if (mvr::copy_pages_pieces(a->num_kv_heads * a->page_size, (int64_t)a->head_dim * es_of(a->dtype), a->key_pool,
                             a->value_pool) * 2 * a->num_copies > kMaxThreads / 256)
    return fail(MVR_E_UNSUPPORTED, "%d copies of pages of this size are more than one call takes", a->num_copies);
  return MVR_OK;
}

int mvr_copy_pages_validate(const mvr_copy_pages_args* a, const int32_t* src_pages_host, const int32_t* dst_pages_host,
                            const int32_t* tokens_host) {
  mvr::api::clear_error();
  const int rc = check_copy(a);
  if (rc != MVR_OK) return rc;
  std::unique_ptr<uint8_t[]> use(new (std::nothrow) uint8_t[(size_t)a->num_pages]()); // 1: source, 2: destination
  if (!use) return fail(MVR_E_INVALID_ARGUMENT, "out of host memory");
  for (int pass = 0; pass < 2; pass++) {
    const int32_t* list = pass ? dst_pages_host : src_pages_host;
    for (int i = 0; list && i < a->num_copies; i++) {
      if (list[i] < 0 || list[i] >= a->num_pages)
        return fail(MVR_E_PAGE_ID, "copy %d has %s page %d outside a pool of %lld pages", i,
                    pass ? "destination" : "source", list[i], (long long)a->num_pages);
      if (pass && use[list[i]])
        return fail(MVR_E_INVALID_ARGUMENT, "destination page %d is %s of this call", list[i],
                    use[list[i]] == 1 ? "a source" : "twice a destination");
      use[list[i]] = (uint8_t)(pass + 1);
    }
  }
  for (int i = 0; tokens_host && i < a->num_copies; i++)
    if (tokens_host[i] < 0 || tokens_host[i] > a->page_size)
      return fail(MVR_E_INVALID_ARGUMENT, "copy %d has %d tokens, outside a page of %d", i, tokens_host[i], a->page_size);
  return MVR_OK;
}

int mvr_copy_pages(const mvr_copy_pages_args* a) {
  mvr::api::Range range("attn-cache operation=copy");
  mvr::api::clear_error();
  int rc = check_copy(a);
  if (rc != MVR_OK) return rc;
  if (a->num_copies == 0) return MVR_OK;
  if (mvr::api::checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> src, dst, tokens;
      if (!mvr::api::copy_to_host(a->src_pages, a->num_copies, a->stream, src) ||
          !mvr::api::copy_to_host(a->dst_pages, a->num_copies, a->stream, dst) ||
          !mvr::api::copy_to_host(a->tokens, a->num_copies, a->stream, tokens))
        return copy_failed();
      return mvr_copy_pages_validate(a, src.data(), dst.data(), data_or_null(tokens));
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::CopyPagesParams p{};
  p.key_pool = a->key_pool;
  p.value_pool = a->value_pool;
  p.src_pages = a->src_pages;
  p.dst_pages = a->dst_pages;
  p.tokens = a->tokens;
  p.num_pages = a->num_pages;
  p.num_copies = a->num_copies;
  p.num_kv_heads = a->num_kv_heads;
  p.page_size = a->page_size;
  return launch_status(
      mvr::launch_copy_pages(p, (int64_t)a->head_dim * es_of(a->dtype), static_cast<hipStream_t>(a->stream)));
}

} // extern "C"
