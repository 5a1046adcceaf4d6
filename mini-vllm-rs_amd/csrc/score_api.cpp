// C ABI of the calls on scores: argument checks, planning, dispatch.
// Declared in include/mvr_score.h.
#include "mvr_score.h"

#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <memory>
#include <new>
#include <vector>

#include "api_common.hpp"
#include "paged_attention_kernels.hpp" // kChunkTokens
#include "paged_prefill.hpp"           // page_divider
#include "score_attention.hpp"

namespace {

using namespace mvr::api;

constexpr double kLog2e = 1.4426950408889634;

float scale_of(const mvr_paged_attention_args* a) {
  return a->scale > 0.f ? a->scale : (float)(1.0 / sqrt((double)a->head_dim));
}

// ---------------------------------------------------------------------------
// Attention with bent and masked scores
// ---------------------------------------------------------------------------

int check_rules(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  if (!r) return fail(MVR_E_INVALID_ARGUMENT, "rules is null");
  if (!(r->cap >= 0.f) || !isfinite(r->cap)) return fail(MVR_E_INVALID_ARGUMENT, "cap must be finite and >= 0");
  if (r->cap > 0.f && (r->cap > 1e30f || !(scale_of(a) / r->cap < 1e30f)))
    return fail(MVR_E_UNSUPPORTED, "cap %g is out of range for scores in 32 bits", r->cap);
  if (r->window < 0) return fail(MVR_E_INVALID_ARGUMENT, "window must not be negative");
  if (((uintptr_t)r->slopes | (uintptr_t)r->first_keys | (uintptr_t)r->prefix_lens | (uintptr_t)r->lse) % 4)
    return fail(MVR_E_INVALID_ARGUMENT, "slopes, first_keys, prefix_lens and lse must be 4-byte aligned");
  if (r->lse && r->lse_stride_head < a->total_q)
    return fail(MVR_E_INVALID_ARGUMENT, "lse_stride_head %lld is smaller than total_q %d", (long long)r->lse_stride_head,
                a->total_q);
  return MVR_OK;
}

// The checks that attention and weights share.
int check_scored(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  mvr_paged_attention_args b = *a;
  b.total_q = 0; // empty requests make its lower bound 0
  int rc = check_attention_scalars(&b);
  if (rc != MVR_OK) return rc;
  if (a->total_q < 0 || a->total_q > (int64_t)a->num_seqs * a->max_q_len)
    return fail(MVR_E_INVALID_ARGUMENT, "total_q %d is outside [0, num_seqs * max_q_len]", a->total_q);
  if (a->num_seqs == 1 && !a->cu_q_lens && a->total_q > 0 && a->total_q < a->max_q_len)
    return fail(MVR_E_INVALID_ARGUMENT, "total_q %d is smaller than max_q_len %d, the q_len of a call without cu_q_lens",
                a->total_q, a->max_q_len);
  rc = check_rules(a, r);
  if (rc != MVR_OK) return rc;
  if (a->max_seq_len > INT32_MAX - 1024) // (positions of whole key tiles are counted in 32 bits)
    return fail(MVR_E_UNSUPPORTED, "max_seq_len %d is too close to 2^31", a->max_seq_len);
  if (a->page_size % mvr::kChunkTokens != 0 && (int64_t)a->page_size * a->head_dim * es_of(a->dtype) > INT32_MAX)
    return fail(MVR_E_UNSUPPORTED, "pages of 2 GiB per KV head whose size is not a multiple of %d tokens",
                mvr::kChunkTokens);
  // The kernels count a page's rows, a head's rows and work items in 32 bits.
  if (a->num_pages > INT32_MAX || (int64_t)a->num_kv_heads * a->page_size > INT32_MAX)
    return fail(MVR_E_UNSUPPORTED, "pools of over 2^31 pages, or pages of over 2^31 rows");
  if ((int64_t)(a->num_q_heads / a->num_kv_heads) * a->max_q_len > INT32_MAX - 1024)
    return fail(MVR_E_UNSUPPORTED, "requests of %d tokens are more than one call takes", a->max_q_len);
  return MVR_OK;
}

// Places for row tiles: those of the longest request for every request; packed, as many as
// the packed tokens have and one more of each request, whose owner a block finds by a
// search of cu_q_lens: where that leaves half of the places out, or a launch could not
// hold them.  (63 single tokens and 2,000 new ones on 2,000 keys each, F16: 112 us packed
// and 151 padded for 28/4 heads, 43 and 125 for 7/1; ten batches whose lengths vary less,
// 0.82 to 1.07 times.)
struct Places {
  int64_t groups, row_tiles, padded; // (padded: row tiles of the longest request)
  bool packed;
};

bool one_launch(int64_t groups, int64_t inner, int waves) {
  const int64_t blocks = kMaxThreads / (64 * waves);
  return inner <= blocks / groups && mvr::score_grid(groups, inner) <= blocks;
}

Places places_of(const mvr_paged_attention_args* a, int tile_rows, int waves) {
  const int64_t group = a->num_q_heads / a->num_kv_heads;
  const int64_t padded = (group * a->max_q_len + tile_rows - 1) / tile_rows, all = mvr::score_groups(false, a->num_seqs, a->num_kv_heads);
  const int64_t tokens = a->total_q > 0 ? a->total_q : (int64_t)a->num_seqs * a->max_q_len;
  const int64_t in_all = group * tokens / tile_rows + a->num_seqs;
  if (a->cu_q_lens && (2 * in_all <= padded * a->num_seqs || !one_launch(all, padded, waves)))
    return {mvr::score_groups(true, a->num_seqs, a->num_kv_heads), in_all, padded, true};
  return {all, padded, padded, false};
}

// The checks of the attention call.
int check_attention(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  const int rc = check_scored(a, r);
  if (rc != MVR_OK) return rc;
  const Places x = places_of(a, 16, 4);
  if (!one_launch(x.groups, x.row_tiles, 4))
    return fail(MVR_E_UNSUPPORTED, "%d requests of up to %d tokens (%d in all; 0: not given) are more than one call takes",
                a->num_seqs, a->max_q_len, a->total_q);
  return MVR_OK;
}

mvr::ScoreTables tables_of(const mvr_paged_attention_args* a) {
  mvr::ScoreTables t{};
  t.q = a->q;
  t.q_stride_head = a->q_stride_head;
  t.q_stride_token = a->q_stride_token;
  t.key_pool = a->key_pool;
  t.block_tables = a->block_tables;
  t.block_table_stride = a->max_pages_per_seq;
  t.seq_lens = a->seq_lens;
  t.cu_q_lens = a->cu_q_lens;
  t.max_seq_len = a->max_seq_len;
  t.max_q_len = a->max_q_len;
  t.num_seqs = a->num_seqs;
  t.num_kv_heads = a->num_kv_heads;
  t.group_size = a->num_q_heads / a->num_kv_heads;
  t.page_size = a->page_size;
  t.last_page = (uint32_t)(a->num_pages - 1);
  mvr::page_divider(a->page_size, t.page_magic, t.page_magic_shift);
  return t;
}

mvr::ScoreRules rules_of(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  mvr::ScoreRules k{};
  const float scale = scale_of(a);
  k.scale_log2 = (float)(scale * kLog2e);
  if (r->cap > 0.f) {
    k.cap_log2 = (float)(r->cap * kLog2e);
    const double y = (double)scale / r->cap; // of a dot product of 1
    k.cap_exp_scale = (float)(2 * kLog2e * y);
    // Where y is so small that a coefficient leaves the normal numbers, it and those after
    // it are left out, and the range ends where they would be 2^-25 of the result.  Where
    // it is so large that one overflows, there is no range.
    double limit = mvr::kTanhPolynomial;
    for (int i = 0; i < 6; i++) {
      const double c = mvr::kTanhCoefficients[i], folded = c * scale * kLog2e * pow(y, 2 * i);
      if (fabs(folded) < 1e-37 && i > 0) {
        limit = std::min(limit, pow(0x1p-25 / fabs(c), 1.0 / (2 * i)));
        break;
      }
      if (!(fabs(folded) < 1e37)) {
        limit = -1;
        break;
      }
      k.cap_poly[i] = (float)folded;
    }
    k.cap_poly_limit = (float)std::min(limit / y, 1e18); // (its square is a number)
  }
  k.window = r->window;
  k.slopes = r->slopes;
  k.first_keys = r->first_keys;
  k.prefix_lens = r->prefix_lens;
  k.lse = r->lse;
  k.lse_stride_head = r->lse_stride_head;
  return k;
}

int64_t units_of(int64_t tokens) { return (tokens + mvr::kScoreUnitTokens - 1) / mvr::kScoreUnitTokens; }

// Row tiles of one size, as the planner sees them: by the host tables, or as if all
// requests were alike.  One pass over the tables; requests of like lengths count as one
// afterwards, so that a split's parts are estimated in a few steps.
class TileWork {
 public:
  TileWork(const mvr_paged_attention_args* a, const mvr_score_rules* r, int tile_rows) {
    const int64_t group = a->num_q_heads / a->num_kv_heads;
    int64_t bound = units_of(a->max_seq_len); // units that a window leaves a row tile
    if (r->window > 0 && !r->prefix_lens)
      bound = std::min(bound, units_of((int64_t)r->window + (tile_rows + group - 1) / group) + 1);
    const double per_unit = kGroups / (double)(bound + 1);
    auto add = [&](int64_t q, int64_t keys, int64_t requests) {
      const int64_t n = requests * ((group * q + tile_rows - 1) / tile_rows);
      // (A causal mask leaves the request's first token its past alone.)
      const int64_t least = std::min(bound, units_of(std::max<int64_t>(keys - q + 1, 1)));
      const int64_t most = std::min(bound, units_of(std::max<int64_t>(keys, 1)));
      if (n == 0) return;
      Group& g = groups_[(int)(most * per_unit)];
      g.tiles += n;
      g.least += (double)n * least;
      g.most += (double)n * most;
      longest = std::max(longest, most);
    };
    const int32_t *cu = a->cu_q_lens_host, *sl = a->seq_lens_host;
    if (cu && sl) {
      for (int s = 0; s < a->num_seqs; s++)
        add(std::min<int64_t>(std::max<int64_t>(0, (int64_t)cu[s + 1] - cu[s]), a->max_q_len),
            std::min(std::max(sl[s], 0), a->max_seq_len), 1);
    } else {
      add(a->max_q_len, a->sum_seq_lens > 0 ? (a->sum_seq_lens + a->num_seqs - 1) / a->num_seqs : a->max_seq_len,
          a->num_seqs);
    }
    double sum = 0;
    for (Group& g : groups_) {
      g.tiles *= a->num_kv_heads;
      if (g.tiles == 0) continue;
      sum += (g.least + g.most) / 2;
      g.least *= a->num_kv_heads / g.tiles;
      g.most *= a->num_kv_heads / g.tiles;
      tiles += (int64_t)g.tiles;
    }
    units = (int64_t)(sum * a->num_kv_heads);
  }

  // Blocks of a call that is split into parts of `part` units.
  int64_t blocks(int64_t part) const {
    // Parts of tiles of 1, 2, ... x units, together.
    auto upto = [part](double x) {
      const double k = floor(x / part);
      return part * k * (k + 1) / 2 + (x - k * part) * (k + 1);
    };
    double count = 0;
    for (const Group& g : groups_)
      if (g.tiles > 0) count += g.tiles * (upto(g.most) - upto(g.least - 1)) / (g.most - g.least + 1);
    return (int64_t)ceil(count);
  }

  int64_t tiles = 0, units = 0; // row tiles; units of 64 keys over all of them
  int64_t longest = 0;          // units of one

 private:
  static constexpr int kGroups = 16;
  struct Group { // of requests: row tiles, units that the first one's keys take, and the last one's
    double tiles = 0, least = 0, most = 0;
  };
  Group groups_[kGroups];
};

// What a block of one tile size costs, in us, for head_dim 128: `fixed` beside its keys,
// `unit` per 64 keys with one to four blocks on its CU, of which the share `own` does not
// go by the head dimension; `capped` times that under a cap.  Fitted to 185 timed plans
// (tile sizes and splits of 13 calls: 1 to 32 requests on 100 to 16,000 tokens, 1 to 2,000
// new ones, head_dim 64 and 128), which they meet within 13 to 25% (root mean square).
struct TileCost {
  int rows, waves;
  double fixed, unit[4], own, capped;
};

constexpr TileCost kF16Costs[] = {{16, 4, 3.0, {0.70, 1.45, 2.20, 3.00}, 0.85, 1.1},
                                  {64, 4, 7.2, {0.97, 1.57, 1.57, 1.57}, 0.7, 1.3},
                                  {128, 4, 6.5, {1.50, 1.53, 1.53, 1.53}, 0.5, 1.4},
                                  {128, 8, 7.0, {0.97, 0.97, 0.97, 0.97}, 0.5, 1.45}};
constexpr TileCost kF32Costs[] = {{16, 4, 3.3, {2.00, 4.20, 5.80, 6.90}, 0.0, 1.0},
                                  {64, 4, 10.0, {5.50, 8.50, 8.50, 8.50}, 0.0, 1.0},
                                  {128, 4, 12.0, {7.20, 14.3, 14.3, 14.3}, 0.0, 1.0},
                                  {128, 8, 12.0, {7.50, 7.50, 7.50, 7.50}, 0.0, 1.0}};

// Bytes of partial results that a split may take, at most; they hold a slot for every part
// of every place, also where few tiles have so many.  (11 calls of F32 prompts and long
// contexts whose fastest plans by cost take 37 to 238 MiB: none is over 5% slower within
// 96 MiB, four are faster; within 48, 36%, 41% and 20% slower are three.)
constexpr size_t kSplitBudget = (size_t)96 << 20;

// The tile size and the split of its keys that these costs make fastest: every tile
// whole, or in parts that give each CU one block, two, up to as many as it holds, or
// two, three or four times that, or in fewer parts where tiles are few.  A call takes its blocks' time (all of them in one
// round; in more rounds the average load and most of a last block), joined with the time
// that its keys take from HBM (as a 3-norm).  A split call merges: a launch, a chain of
// loads over a row's parts, and its partial results written and read at 4.3 TB/s.
mvr::ScoreAttentionPlan plan_scored(const mvr_paged_attention_args* a, const mvr_score_rules* r, size_t limit) {
  limit = std::min(limit, kSplitBudget);
  const bool f16 = a->dtype == MVR_DTYPE_F16;
  const int64_t group = a->num_q_heads / a->num_kv_heads, longest_rows = group * a->max_q_len;
  const int64_t cus = compute_units();
  // Overrides, for tests and tuning: a tile size that the head dimension has, and its parts.
  static const int set_rows = env_int("MVR_SCORE_TILE_ROWS", 0);
  static const int set_waves = env_int("MVR_SCORE_TILE_WAVES", 4);
  static const int set_units = env_int("MVR_SCORE_PART_UNITS", 0);
  bool rows_set = false;
  auto runs = [&](const TileCost& tile, const Places& x) {
    return mvr::score_tile_supported(tile.rows, tile.waves, a->head_dim) && one_launch(x.groups, x.row_tiles, tile.waves);
  };
  for (const TileCost& tile : kF16Costs)
    rows_set |= tile.rows == set_rows && tile.waves == set_waves && runs(tile, places_of(a, tile.rows, tile.waves));
  mvr::ScoreAttentionPlan best{};
  double best_cost = INFINITY;
  for (const TileCost& tile : f16 ? kF16Costs : kF32Costs) {
    const Places x = places_of(a, tile.rows, tile.waves);
    if (!runs(tile, x)) continue; // (16 rows do: check_attention)
    // (A tile that no request fills half costs what the smaller one does, or more.)
    if (rows_set ? tile.rows != set_rows || tile.waves != set_waves : longest_rows <= tile.rows / 2 && best_cost < INFINITY) continue;
    const int held = mvr::score_blocks_per_cu(tile.rows, tile.waves, f16, a->head_dim);
    const TileWork w(a, r, tile.rows);
    const int64_t groups = x.groups, row_tiles = x.row_tiles, all_tiles = groups * row_tiles;
    const double unit_scale = (tile.own + (1 - tile.own) * a->head_dim / 128.0) * (r->cap > 0.f ? tile.capped : 1.0);
    // (Row tiles of one KV head read the same keys, which the caches keep.)
    const double hbm = (double)w.units / std::max<int64_t>(1, x.padded) *
                       (2.0 * mvr::kScoreUnitTokens * a->head_dim * es_of(a->dtype) / 5.9e6);
    auto cost_of = [&](int64_t blocks, double longest) { // of `longest` units at most
      double body;
      if (blocks <= held * cus)
        body = longest * tile.unit[std::max<int64_t>(0, (blocks + cus - 1) / cus - 1)];
      else
        body = std::max(w.units * tile.unit[held - 1] / (held * cus) + 0.5 * longest * tile.unit[0], longest * tile.unit[0]);
      body *= unit_scale;
      return tile.fixed + cbrt(body * body * body + hbm * hbm * hbm);
    };
    auto take = [&](double cost, int64_t parts, int64_t part_units, size_t bytes) {
      if (!(cost < best_cost)) return;
      best_cost = cost;
      best.tile_rows = tile.rows;
      best.waves = tile.waves;
      best.row_tiles = (int)row_tiles;
      best.packed = x.packed;
      best.parts = (int)parts;
      best.part_units = (int)std::min<int64_t>(part_units, INT32_MAX / 2); // (units are added to it)
      best.partial_bytes = bytes;
    };
    bool too_large = false;
    auto take_split = [&](int64_t part) { // parts of `part` units
      const int64_t parts = std::min<int64_t>((w.longest + part - 1) / part, mvr::kScoreMaxParts);
      if (parts < 2 || !one_launch(groups, row_tiles * parts, tile.waves)) return;
      if (all_tiles > kMaxThreads / (tile.rows * a->head_dim / 4 + 256)) return; // (the merge's)
      const int64_t rows = all_tiles * parts * tile.rows;
      const size_t bytes = align_up((size_t)rows * a->head_dim * sizeof(float), 256) +
                           align_up((size_t)rows * 2 * sizeof(float), 256) +
                           align_up((size_t)all_tiles * sizeof(int32_t), 256);
      if (bytes > limit) {
        too_large = true;
        return;
      }
      part = std::max(part, (w.longest + parts - 1) / parts);
      const int64_t blocks = w.blocks(part);
      // (The partials that are written: the others' slots are left alone.)
      const double moved = 2.0 * blocks * tile.rows * (a->head_dim + 2) * sizeof(float) / 4.3e6;
      take(cost_of(blocks, part) + 3.5 + 0.17 * parts + moved, parts, part, bytes);
    };
    take(cost_of(w.tiles, w.longest), 1, INT32_MAX, 0);
    if (w.tiles == 0 || w.longest < 2 || limit == 0) continue;
    if (set_units) {
      if (set_units < w.longest) best_cost = rows_set ? INFINITY : best_cost, take_split(set_units);
      continue;
    }
    int64_t last = 0;
    for (int64_t target = cus; target <= 4 * held * cus; target += target < held * cus ? cus : held * cus) {
      if (w.tiles >= target) continue;
      // (A tile's last part is half full on average.)
      const int64_t part = std::max<int64_t>(1, (w.units + target - w.tiles / 2 - 1) / (target - w.tiles / 2));
      if (part < w.longest && part != last) take_split(part);
      last = part;
    }
    // And where tiles of 16 rows are few, fewer parts than that, which are merged sooner.
    // (One token on 3,000, 14/2 heads of 64 F16: 9.7 us in 12 parts, 15.7 in 47.)
    for (int64_t parts = 2; tile.rows == 16 && parts * w.tiles < cus && parts < std::min<int64_t>(w.longest, mvr::kScoreMaxParts);
         parts += (parts + 1) / 2)
      take_split((w.longest + parts - 1) / parts);
    // Where a workspace is too small for these, the fewest parts that fit.
    if (too_large && best.parts <= 1)
      for (int64_t parts = 2; parts <= 8; parts++) take_split((w.longest + parts - 1) / parts);
  }
  return best;
}

int copy_floats(const float* dev, size_t count, void* stream, std::vector<float>& host) {
  if (!dev) return MVR_OK;
  std::vector<int32_t> bits;
  if (!copy_to_host(reinterpret_cast<const int32_t*>(dev), count, stream, bits)) return copy_failed();
  host.resize(count);
  for (size_t i = 0; i < count; i++) host[i] = __builtin_bit_cast(float, bits[i]);
  return MVR_OK;
}

const float* floats_or_null(const std::vector<float>& v) { return v.empty() ? nullptr : v.data(); }

// Host copies of the tables that attention and weights read.
struct HostTables {
  std::vector<int32_t> bt, sl, cu, first, prefix;
  std::vector<float> slopes;

  int read(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
    if (!copy_to_host(a->block_tables, (size_t)a->num_seqs * a->max_pages_per_seq, a->stream, bt) ||
        !copy_to_host(a->seq_lens, a->num_seqs, a->stream, sl) ||
        !copy_to_host(a->cu_q_lens, (size_t)a->num_seqs + 1, a->stream, cu) ||
        !copy_to_host(r->prefix_lens, a->num_seqs, a->stream, prefix))
      return copy_failed();
    // (Packed tokens: as many as the starts say, once those are known to be sound.)
    if (!cu.empty() && check_cu_q_lens(cu.data(), a->num_seqs, a->total_q, a->max_q_len) != MVR_OK)
      return MVR_E_INVALID_ARGUMENT;
    const int64_t tokens = cu.empty() ? a->max_q_len : cu[a->num_seqs];
    if (!copy_to_host(r->first_keys, (size_t)tokens, a->stream, first)) return copy_failed();
    return copy_floats(r->slopes, a->num_q_heads, a->stream, slopes);
  }
};

int validate_scored(const mvr_paged_attention_args* a, const int32_t* block_tables_host, const int32_t* seq_lens_host,
                    const int32_t* cu_q_lens_host, const int32_t* first_keys_host, const int32_t* prefix_lens_host,
                    const float* slopes_host) {
  if (cu_q_lens_host && check_cu_q_lens(cu_q_lens_host, a->num_seqs, a->total_q, a->max_q_len) != MVR_OK)
    return MVR_E_INVALID_ARGUMENT;
  for (int h = 0; slopes_host && h < a->num_q_heads; h++)
    if (!isfinite(slopes_host[h])) return fail(MVR_E_INVALID_ARGUMENT, "slope of head %d is not finite", h);
  for (int s = 0; s < a->num_seqs; s++) {
    int64_t q_len = a->cu_q_lens ? -1 : a->max_q_len, at = 0; // (-1: not known here)
    if (cu_q_lens_host) {
      at = cu_q_lens_host[s];
      q_len = (int64_t)cu_q_lens_host[s + 1] - at;
    }
    const int64_t seq_len = seq_lens_host ? seq_lens_host[s] : a->seq_lens ? -1 : a->max_seq_len;
    if (seq_lens_host) {
      if (seq_len < 0 || seq_len > a->max_seq_len)
        return fail(MVR_E_INVALID_ARGUMENT, "request %d has seq_len %lld outside [0, max_seq_len %d]", s,
                    (long long)seq_len, a->max_seq_len);
      if (q_len >= 0 && seq_len < q_len)
        return fail(MVR_E_LENGTH_MISMATCH, "paged KV cache reports sequence length %lld, expected at least %lld",
                    (long long)seq_len, (long long)q_len);
    }
    if (prefix_lens_host && prefix_lens_host[s] < 0)
      return fail(MVR_E_INVALID_ARGUMENT, "request %d has a prefix of %d tokens", s, prefix_lens_host[s]);
    if (block_tables_host && seq_len >= 0 && q_len != 0)
      for (int64_t pi = 0; pi < (seq_len + a->page_size - 1) / a->page_size; pi++) {
        const int32_t id = block_tables_host[(int64_t)s * a->max_pages_per_seq + pi];
        if (id < 0 || id >= a->num_pages)
          return fail(MVR_E_PAGE_ID, "request %d page %lld has id %d outside a pool of %lld pages", s, (long long)pi, id,
                      (long long)a->num_pages);
      }
    if (first_keys_host && q_len > 0)
      for (int64_t n = at; n < at + q_len; n++)
        if (first_keys_host[n] < 0)
          return fail(MVR_E_INVALID_ARGUMENT, "token %lld has first key %d", (long long)n, first_keys_host[n]);
  }
  return MVR_OK;
}

} // namespace

extern "C" {

size_t mvr_paged_attention_scored_workspace_size(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  if (check_attention(a, r) != MVR_OK) return 0;
  return plan_scored(a, r, SIZE_MAX).partial_bytes;
}

int mvr_paged_attention_scored_validate(const mvr_paged_attention_args* a, const mvr_score_rules* r,
                                        const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                        const int32_t* cu_q_lens_host, const int32_t* first_keys_host,
                                        const int32_t* prefix_lens_host, const float* slopes_host) {
  clear_error();
  const int rc = check_attention(a, r);
  if (rc != MVR_OK) return rc;
  return validate_scored(a, block_tables_host, seq_lens_host, cu_q_lens_host, first_keys_host, prefix_lens_host,
                         slopes_host);
}

int mvr_paged_attention_scored(const mvr_paged_attention_args* a, const mvr_score_rules* r) {
  Range range("attn"); // trace.rs:64
  clear_error();
  int rc = check_attention(a, r);
  if (rc != MVR_OK) return rc;
  if (checked()) {
    rc = run_checked([&] {
      HostTables h;
      const int read = h.read(a, r);
      if (read != MVR_OK) return read;
      return validate_scored(a, data_or_null(h.bt), data_or_null(h.sl), data_or_null(h.cu), data_or_null(h.first),
                             data_or_null(h.prefix), floats_or_null(h.slopes));
    });
    if (rc != MVR_OK) return rc;
  }
  if (a->workspace && ((uintptr_t)a->workspace & 255u))
    return fail(MVR_E_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  const mvr::ScoreAttentionPlan plan = plan_scored(a, r, a->workspace ? a->workspace_bytes : 0);
  mvr::ScoreAttentionParams p{};
  p.t = tables_of(a);
  p.r = rules_of(a, r);
  p.value_pool = a->value_pool;
  p.out = a->out;
  p.out_stride_head = a->out_stride_head;
  p.out_stride_token = a->out_stride_token;
  p.row_tiles = plan.row_tiles;
  p.packed = plan.packed;
  p.parts = plan.parts;
  p.part_units = plan.part_units;
  const int64_t groups = mvr::score_groups(plan.packed, a->num_seqs, a->num_kv_heads);
  p.run = (int)mvr::score_run(groups, (int64_t)plan.row_tiles * plan.parts);
  if (plan.parts > 1) {
    const size_t rows = (size_t)groups * plan.row_tiles * plan.parts * plan.tile_rows;
    char* at = static_cast<char*>(a->workspace);
    p.partial_o = reinterpret_cast<float*>(at);
    at += align_up(rows * a->head_dim * sizeof(float), 256);
    p.partial_ml = reinterpret_cast<float*>(at);
    at += align_up(rows * 2 * sizeof(float), 256);
    p.tile_parts = reinterpret_cast<int32_t*>(at);
  }
  Range launch("attn-paged-fused");
  return launch_status(
      mvr::launch_score_attention(plan, p, a->dtype, a->head_dim, static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// The weight that keys get
// ---------------------------------------------------------------------------

static int check_weights(const mvr_paged_attention_args* a, const mvr_score_rules* r, const mvr_key_weights* w) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  mvr_paged_attention_args b = *a; // (what this call does not use need not be there)
  b.value_pool = a->key_pool;
  b.out = const_cast<void*>(a->q);
  b.out_stride_head = a->q_stride_head;
  b.out_stride_token = a->q_stride_token;
  const int rc = check_scored(&b, r);
  if (rc != MVR_OK) return rc;
  if (!r->lse) return fail(MVR_E_INVALID_ARGUMENT, "weights need the rows' log-sum-exps");
  if (!w) return fail(MVR_E_INVALID_ARGUMENT, "weights is null");
  if (!w->weights) return fail(MVR_E_INVALID_ARGUMENT, "null weights pool pointer");
  if (((uintptr_t)w->weights | (uintptr_t)w->fresh_from) % 4)
    return fail(MVR_E_INVALID_ARGUMENT, "the weights pool and fresh_from must be 4-byte aligned");
  if (!(w->decay >= 0.f) || !isfinite(w->decay)) return fail(MVR_E_INVALID_ARGUMENT, "decay must be finite and >= 0");
  const int64_t unit = mvr::weights_unit_tokens(es_of(a->dtype), a->head_dim);
  const int64_t blocks = (a->max_seq_len + unit - 1) / unit;
  if ((int64_t)a->num_seqs * a->num_kv_heads > kMaxThreads / 256 / blocks)
    return fail(MVR_E_UNSUPPORTED, "%d requests of %d tokens are more than one call takes", a->num_seqs, a->max_seq_len);
  return MVR_OK;
}

// Marks a page as written; an error where it was before.
static int mark_page(uint8_t* written, int32_t id, const char* what) {
  if (written[id]) return fail(MVR_E_INVALID_ARGUMENT, "page %d %s more than one request or layer", id, what);
  written[id] = 1;
  return MVR_OK;
}

static int validate_weights(const mvr_paged_attention_args* a, const int32_t* block_tables_host,
                            const int32_t* seq_lens_host, const int32_t* cu_q_lens_host, const int32_t* first_keys_host,
                            const int32_t* prefix_lens_host, const float* slopes_host, const int32_t* fresh_from_host) {
  int rc = validate_scored(a, block_tables_host, seq_lens_host, cu_q_lens_host, first_keys_host, prefix_lens_host,
                           slopes_host);
  if (rc != MVR_OK) return rc;
  for (int s = 0; fresh_from_host && s < a->num_seqs; s++)
    if (fresh_from_host[s] < 0) return fail(MVR_E_INVALID_ARGUMENT, "request %d has fresh_from %d", s, fresh_from_host[s]);
  if (!block_tables_host || (a->seq_lens && !seq_lens_host) || (a->cu_q_lens && !cu_q_lens_host)) return MVR_OK;
  std::unique_ptr<uint8_t[]> written(new (std::nothrow) uint8_t[(size_t)a->num_pages]());
  if (!written) return fail(MVR_E_INVALID_ARGUMENT, "out of host memory");
  for (int s = 0; s < a->num_seqs; s++) {
    if (cu_q_lens_host && cu_q_lens_host[s + 1] == cu_q_lens_host[s]) continue;
    const int64_t seq_len = seq_lens_host ? seq_lens_host[s] : a->max_seq_len;
    for (int64_t pi = 0; pi < (seq_len + a->page_size - 1) / a->page_size && rc == MVR_OK; pi++)
      rc = mark_page(written.get(), block_tables_host[(int64_t)s * a->max_pages_per_seq + pi],
                     "holds the weights of");
    if (rc != MVR_OK) return rc;
  }
  return MVR_OK;
}

int mvr_attention_weights_validate(const mvr_paged_attention_args* a, const mvr_score_rules* r, const mvr_key_weights* w,
                                   const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                   const int32_t* cu_q_lens_host, const int32_t* first_keys_host,
                                   const int32_t* prefix_lens_host, const float* slopes_host,
                                   const int32_t* fresh_from_host) {
  clear_error();
  const int rc = check_weights(a, r, w);
  if (rc != MVR_OK) return rc;
  return validate_weights(a, block_tables_host, seq_lens_host, cu_q_lens_host, first_keys_host, prefix_lens_host,
                          slopes_host, fresh_from_host);
}

int mvr_attention_weights(const mvr_paged_attention_args* a, const mvr_score_rules* r, const mvr_key_weights* w) {
  Range range("attn-cache operation=weigh");
  clear_error();
  int rc = check_weights(a, r, w);
  if (rc != MVR_OK) return rc;
  if (checked()) {
    rc = run_checked([&] {
      HostTables h;
      std::vector<int32_t> fresh;
      const int read = h.read(a, r);
      if (read != MVR_OK) return read;
      if (!copy_to_host(w->fresh_from, a->num_seqs, a->stream, fresh)) return copy_failed();
      return validate_weights(a, data_or_null(h.bt), data_or_null(h.sl), data_or_null(h.cu), data_or_null(h.first),
                              data_or_null(h.prefix), floats_or_null(h.slopes), data_or_null(fresh));
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::ScoreWeightsParams p{};
  p.t = tables_of(a);
  p.r = rules_of(a, r);
  p.weights = w->weights;
  p.decay = w->decay;
  p.fresh_from = w->fresh_from;
  // Where the keys give the SIMDs less than a wavefront each, a block's wavefronts share
  // its keys and split the rows (28/4 heads of 128 F16: 32 new tokens on 1,500, 7.9 us
  // split and 16.6 not; where there are more, 4 times 32 on 6,000, 29.8 and 24.5).
  const int64_t unit = mvr::weights_unit_tokens(es_of(a->dtype), a->head_dim);
  const int64_t units = (int64_t)a->num_seqs * a->num_kv_heads * ((a->max_seq_len + unit - 1) / unit);
  const int64_t rows = (int64_t)(a->num_q_heads / a->num_kv_heads) * a->max_q_len;
  const bool split = rows > 32 && units < 4 * (int64_t)compute_units();
  return launch_status(mvr::launch_score_weights(p, a->dtype, a->head_dim, split, static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// Which tokens stay
// ---------------------------------------------------------------------------

constexpr int64_t kMaxSlots = (int64_t)1 << 40;

// Geometry of a call over the tables of several layers.
static int check_layers(int32_t num_layers, int32_t num_seqs, int32_t num_kv_heads, int32_t page_size, int64_t num_pages,
                        int64_t threads_per_row, int32_t max_moves) {
  if (num_layers < 1) return fail(MVR_E_INVALID_ARGUMENT, "num_layers must be positive");
  if (num_seqs < 1) return fail(MVR_E_INVALID_ARGUMENT, "forward requires at least one request");
  if (max_moves < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_moves must be positive");
  if (num_pages > INT32_MAX || num_pages > kMaxSlots / num_kv_heads / page_size)
    return fail(MVR_E_UNSUPPORTED, "pools of over 2^31 pages, or 2^40 tokens and heads");
  if ((int64_t)num_kv_heads * page_size > INT32_MAX) return fail(MVR_E_UNSUPPORTED, "pages of over 2^31 rows");
  if ((int64_t)num_layers * num_seqs + 7 > kMaxThreads / threads_per_row / num_kv_heads)
    return fail(MVR_E_UNSUPPORTED, "more layers, requests and KV heads than one call takes");
  return MVR_OK;
}

struct Extent {
  const void* at;
  int64_t bytes;
  bool overlaps(const Extent& o) const {
    return at && o.at && (uintptr_t)at < (uintptr_t)o.at + o.bytes && (uintptr_t)o.at < (uintptr_t)at + bytes;
  }
};

static int check_select(const mvr_select_tokens_args* a) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  int rc = check_pool(MVR_DTYPE_F32, a->num_kv_heads, 1, a->page_size, a->num_pages, a->weights, a->positions);
  if (rc != MVR_OK) return rc;
  rc = check_layers(a->num_layers, a->num_seqs, a->num_kv_heads, a->page_size, a->num_pages, 1024, a->max_moves);
  if (rc != MVR_OK) return rc;
  if (a->max_seq_len < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_seq_len must be positive");
  if (a->max_seq_len > INT32_MAX - mvr::kSelectStep)
    return fail(MVR_E_UNSUPPORTED, "max_seq_len %d is too close to 2^31", a->max_seq_len);
  if (a->recent < 0 || a->first < 0) return fail(MVR_E_INVALID_ARGUMENT, "recent and first must not be negative");
  const int64_t pages_needed = (a->max_seq_len + (int64_t)a->page_size - 1) / a->page_size;
  if (a->max_pages_per_seq < pages_needed)
    return fail(MVR_E_PAGES_UNCOVERED, "block table rows of %d pages cannot hold %d tokens of %d-token pages",
                a->max_pages_per_seq, a->max_seq_len, a->page_size);
  if (!a->block_tables || !a->seq_lens || !a->keep_lens || !a->moves || !a->num_moves)
    return fail(MVR_E_INVALID_ARGUMENT, "null table pointer");
  if ((uintptr_t)a->moves % 8) return fail(MVR_E_INVALID_ARGUMENT, "moves must be 8-byte aligned");
  // Every block reads the tables while others write.
  const int64_t rows = (int64_t)a->num_layers * a->num_seqs * a->num_kv_heads;
  const int64_t slots = a->num_pages * a->num_kv_heads * a->page_size;
  const Extent written[] = {{a->positions, slots * 4}, {a->moves, rows * a->max_moves * 8}, {a->num_moves, rows * 4},
                            {a->new_seq_lens, (int64_t)a->num_seqs * 4}};
  const Extent read[] = {{a->weights, slots * 4},
                         {a->block_tables, (int64_t)a->num_layers * a->num_seqs * a->max_pages_per_seq * 4},
                         {a->seq_lens, (int64_t)a->num_seqs * 4},
                         {a->next_positions, (int64_t)a->num_seqs * 4},
                         {a->kept_lens, (int64_t)a->num_seqs * 4},
                         {a->keep_lens, (int64_t)a->num_seqs * 4}};
  for (const Extent& w : written) {
    for (const Extent& x : read)
      if (w.overlaps(x)) return fail(MVR_E_INVALID_ARGUMENT, "a written array overlaps a table or the weights");
    for (const Extent& x : written)
      if (&x != &w && w.overlaps(x)) return fail(MVR_E_INVALID_ARGUMENT, "written arrays overlap each other");
  }
  return MVR_OK;
}

int mvr_select_tokens_validate(const mvr_select_tokens_args* a, const int32_t* block_tables_host,
                               const int32_t* seq_lens_host, const int32_t* next_positions_host,
                               const int32_t* kept_lens_host, const int32_t* keep_lens_host) {
  clear_error();
  int rc = check_select(a);
  if (rc != MVR_OK) return rc;
  std::unique_ptr<uint8_t[]> written;
  if (block_tables_host && seq_lens_host) {
    written.reset(new (std::nothrow) uint8_t[(size_t)a->num_pages]());
    if (!written) return fail(MVR_E_INVALID_ARGUMENT, "out of host memory");
  }
  for (int s = 0; s < a->num_seqs; s++) {
    const int64_t n = seq_lens_host ? seq_lens_host[s] : -1;
    if (seq_lens_host && (n < 0 || n > a->max_seq_len))
      return fail(MVR_E_INVALID_ARGUMENT, "request %d has seq_len %lld outside [0, max_seq_len %d]", s, (long long)n,
                  a->max_seq_len);
    if (n >= 0 && next_positions_host && next_positions_host[s] < n)
      return fail(MVR_E_LENGTH_MISMATCH, "request %d has next position %d before its %lld tokens", s,
                  next_positions_host[s], (long long)n);
    if (kept_lens_host && (kept_lens_host[s] < 0 || (n >= 0 && kept_lens_host[s] > n)))
      return fail(MVR_E_LENGTH_MISMATCH, "request %d has kept_len %d outside its tokens", s, kept_lens_host[s]);
    if (keep_lens_host) {
      const int64_t keep = keep_lens_host[s];
      if (keep < 0) return fail(MVR_E_INVALID_ARGUMENT, "request %d has keep_len %lld", s, (long long)keep);
      if (n > keep) {
        if ((int64_t)a->first + a->recent > keep)
          return fail(MVR_E_INVALID_ARGUMENT, "request %d keeps %lld tokens, fewer than the first %d and the last %d", s,
                      (long long)keep, a->first, a->recent);
        if (std::min(keep, n - keep) > a->max_moves)
          return fail(MVR_E_INVALID_ARGUMENT, "request %d may need %lld moves, more than max_moves %d", s,
                      (long long)std::min(keep, n - keep), a->max_moves);
      }
    }
    for (int layer = 0; written && layer < a->num_layers; layer++)
      for (int64_t pi = 0; pi < (n + a->page_size - 1) / a->page_size; pi++) {
        const int32_t id = block_tables_host[((int64_t)layer * a->num_seqs + s) * a->max_pages_per_seq + pi];
        if (id < 0 || id >= a->num_pages)
          return fail(MVR_E_PAGE_ID, "layer %d request %d page %lld has id %d outside a pool of %lld pages", layer, s,
                      (long long)pi, id, (long long)a->num_pages);
        rc = mark_page(written.get(), id, "holds the tokens of");
        if (rc != MVR_OK) return rc;
      }
  }
  return MVR_OK;
}

int mvr_select_tokens(const mvr_select_tokens_args* a) {
  Range range("attn-cache operation=select");
  clear_error();
  int rc = check_select(a);
  if (rc != MVR_OK) return rc;
  if (checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> bt, sl, next, kept, keep;
      if (!copy_to_host(a->block_tables, (size_t)a->num_layers * a->num_seqs * a->max_pages_per_seq, a->stream, bt) ||
          !copy_to_host(a->seq_lens, a->num_seqs, a->stream, sl) ||
          !copy_to_host(a->next_positions, a->num_seqs, a->stream, next) ||
          !copy_to_host(a->kept_lens, a->num_seqs, a->stream, kept) ||
          !copy_to_host(a->keep_lens, a->num_seqs, a->stream, keep))
        return copy_failed();
      return mvr_select_tokens_validate(a, bt.data(), sl.data(), data_or_null(next), data_or_null(kept), keep.data());
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::SelectTokensParams p{};
  p.weights = a->weights;
  p.positions = a->positions;
  p.block_tables = a->block_tables;
  p.block_table_stride = a->max_pages_per_seq;
  p.seq_lens = a->seq_lens;
  p.next_positions = a->next_positions;
  p.kept_lens = a->kept_lens;
  p.keep_lens = a->keep_lens;
  p.moves = a->moves;
  p.num_moves = a->num_moves;
  p.new_seq_lens = a->new_seq_lens;
  p.num_pages = a->num_pages;
  p.num_layers = a->num_layers;
  p.num_seqs = a->num_seqs;
  p.num_kv_heads = a->num_kv_heads;
  p.page_size = a->page_size;
  p.max_seq_len = a->max_seq_len;
  p.max_moves = a->max_moves;
  p.recent = a->recent;
  p.first = a->first;
  mvr::page_divider(a->page_size, p.page_magic, p.page_magic_shift);
  return launch_status(mvr::launch_select_tokens(p, compute_units(), static_cast<hipStream_t>(a->stream)));
}

// ---------------------------------------------------------------------------
// Moves of tokens
// ---------------------------------------------------------------------------

static int check_move(const mvr_move_tokens_args* a) {
  if (!a) return fail(MVR_E_INVALID_ARGUMENT, "args is null");
  int rc = check_pool(a->dtype, a->num_kv_heads, a->head_dim, a->page_size, a->num_pages, a->key_pool, a->value_pool);
  if (rc != MVR_OK) return rc;
  rc = check_layers(a->num_layers, a->num_seqs, a->num_kv_heads, a->page_size, a->num_pages, 256, a->max_moves);
  if (rc != MVR_OK) return rc;
  if (a->max_moves > INT32_MAX - mvr::kMoveStep)
    return fail(MVR_E_UNSUPPORTED, "max_moves %d is too close to 2^31", a->max_moves);
  if (a->max_pages_per_seq < 1) return fail(MVR_E_INVALID_ARGUMENT, "max_pages_per_seq must be positive");
  if (!a->block_tables || !a->moves || !a->num_moves) return fail(MVR_E_INVALID_ARGUMENT, "null table pointer");
  if ((uintptr_t)a->moves % 8) return fail(MVR_E_INVALID_ARGUMENT, "moves must be 8-byte aligned");
  if (((uintptr_t)a->weights | (uintptr_t)a->positions) % 4)
    return fail(MVR_E_INVALID_ARGUMENT, "weights and positions must be 4-byte aligned");
  return MVR_OK;
}

int mvr_move_tokens_validate(const mvr_move_tokens_args* a, const int32_t* block_tables_host, const int32_t* moves_host,
                             const int32_t* num_moves_host) {
  clear_error();
  const int rc = check_move(a);
  if (rc != MVR_OK) return rc;
  if (!moves_host || !num_moves_host) return MVR_OK;
  const int64_t slots = (int64_t)a->max_pages_per_seq * a->page_size;
  return run_checked([&]() -> int {
    std::vector<int32_t> used; // slots of one row of moves: targets, then sources among them
    for (int64_t row = 0; row < (int64_t)a->num_layers * a->num_seqs * a->num_kv_heads; row++) {
      const int32_t count = num_moves_host[row], *moves = moves_host + row * a->max_moves * 2;
      if (count < 0 || count > a->max_moves)
        return fail(MVR_E_INVALID_ARGUMENT, "row %lld has %d moves, outside [0, max_moves %d]", (long long)row, count,
                    a->max_moves);
      used.clear();
      for (int64_t j = 0; j < 2 * (int64_t)count; j++) {
        const int32_t slot = moves[j];
        if (slot < 0 || slot >= slots)
          return fail(MVR_E_INVALID_ARGUMENT, "row %lld moves slot %d, outside its pages", (long long)row, slot);
        if (block_tables_host) {
          const int32_t id = block_tables_host[row / a->num_kv_heads * a->max_pages_per_seq + slot / a->page_size];
          if (id < 0 || id >= a->num_pages)
            return fail(MVR_E_PAGE_ID, "row %lld page %d has id %d outside a pool of %lld pages", (long long)row,
                        slot / a->page_size, id, (long long)a->num_pages);
        }
        if (j % 2) used.push_back(slot);
      }
      std::sort(used.begin(), used.end());
      for (size_t i = 1; i < used.size(); i++)
        if (used[i] == used[i - 1])
          return fail(MVR_E_INVALID_ARGUMENT, "row %lld moves to slot %d twice", (long long)row, used[i]);
      for (int32_t j = 0; j < count; j++)
        if (std::binary_search(used.begin(), used.end(), moves[2 * (int64_t)j]))
          return fail(MVR_E_INVALID_ARGUMENT, "row %lld moves both to and from slot %d", (long long)row,
                      moves[2 * (int64_t)j]);
    }
    return MVR_OK;
  });
}

int mvr_move_tokens(const mvr_move_tokens_args* a) {
  Range range("attn-cache operation=move");
  clear_error();
  int rc = check_move(a);
  if (rc != MVR_OK) return rc;
  if (checked()) {
    rc = run_checked([&] {
      std::vector<int32_t> bt, moves, counts;
      const size_t rows = (size_t)a->num_layers * a->num_seqs * a->num_kv_heads;
      if (!copy_to_host(a->block_tables, (size_t)a->num_layers * a->num_seqs * a->max_pages_per_seq, a->stream, bt) ||
          !copy_to_host(a->moves, rows * a->max_moves * 2, a->stream, moves) ||
          !copy_to_host(a->num_moves, rows, a->stream, counts))
        return copy_failed();
      return mvr_move_tokens_validate(a, bt.data(), moves.data(), counts.data());
    });
    if (rc != MVR_OK) return rc;
  }
  mvr::MoveTokensParams p{};
  p.key_pool = a->key_pool;
  p.value_pool = a->value_pool;
  p.weights = a->weights;
  p.positions = a->positions;
  p.block_tables = a->block_tables;
  p.block_table_stride = a->max_pages_per_seq;
  p.moves = a->moves;
  p.num_moves = a->num_moves;
  p.num_pages = a->num_pages;
  p.num_layers = a->num_layers;
  p.num_seqs = a->num_seqs;
  p.num_kv_heads = a->num_kv_heads;
  p.page_size = a->page_size;
  p.max_moves = a->max_moves;
  mvr::page_divider(a->page_size, p.page_magic, p.page_magic_shift);
  return launch_status(
      mvr::launch_move_tokens(p, (int64_t)a->head_dim * es_of(a->dtype), static_cast<hipStream_t>(a->stream)));
}

} // extern "C"
