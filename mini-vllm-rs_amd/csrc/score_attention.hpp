// Internal launch interface of the kernels of mvr_score.h (score_attention.hip,
// score_weights.hip, score_evict.hip).  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace mvr {

// Keys are split between parts in units of 64 tokens.
constexpr int kScoreUnitTokens = 64;
// Parts of one row tile, at most.
constexpr int kScoreMaxParts = 64;
constexpr int kScoreXcds = 8;

// Where queries, keys and lengths are.
struct ScoreTables {
  const void* q;
  int64_t q_stride_head, q_stride_token;
  const void* key_pool;
  const int32_t* block_tables;
  int32_t block_table_stride;
  const int32_t* seq_lens;  // may be null: max_seq_len
  const int32_t* cu_q_lens; // may be null: max_q_len
  int32_t max_seq_len, max_q_len;
  int32_t num_seqs, num_kv_heads, group_size, page_size;
  uint32_t last_page;  // num_pages - 1
  uint64_t page_magic; // page of token t = t * page_magic >> page_magic_shift (page_divider)
  int32_t page_magic_shift;
};

// tanh(y) = y * sum_k c_k y^2k for |y| <= kTanhPolynomial but for 4.4e-9 of it (least
// squares, reweighted towards the largest error); in 32 bits it is within 1.0e-7.
constexpr float kTanhPolynomial = 0.625f;
constexpr float kTanhCoefficients[6] = {1.0f,
                                        -0.3333328068256378f,
                                        0.13331441581249237f,
                                        -0.05373971164226532f,
                                        0.020639080554246902f,
                                        -0.005704979412257671f};

struct ScoreRules {
  float scale_log2; // scale * log2(e)
  float cap_log2;   // cap * log2(e); 0: none
  // Of a dot product s up to cap_poly_limit in size, the capped score in log2 units is
  // s * sum_k cap_poly[k] s^2k; of any, cap_log2 * (1 - 2 / (2^(cap_exp_scale * s) + 1)).
  float cap_poly_limit, cap_poly[6];
  float cap_exp_scale; // 2 * log2(e) * scale / cap
  int32_t window;   // 0: none
  const float* slopes;
  const int32_t* first_keys;
  const int32_t* prefix_lens;
  float* lse;
  int64_t lse_stride_head;
};

// Attention.  A row tile holds tile_rows rows rho = i * group_size + r of one
// (request, KV head): i the query token, r the query head within its group.  Its
// keys, from the first that any of its rows sees to the last, are split into parts of
// at least part_units units, `parts` at most.
struct ScoreAttentionParams {
  ScoreTables t;
  ScoreRules r;
  const void* value_pool;
  void* out;
  int64_t out_stride_head, out_stride_token;
  // Places for row tiles.  Padded: `row_tiles` of each (request, KV head), as many as the
  // longest request has.  Packed: `row_tiles` of each KV head, request b's from
  // cu_q_lens[b] * group_size / tile_rows + b on (rounded down: a request's tiles fit
  // before the next one's).
  int32_t row_tiles;
  bool packed;
  int32_t parts, part_units;
  int32_t run; // items that follow each other on one XCD
  float* partial_o;    // [place][part][tile_rows][head_dim]
  float* partial_ml;   // [place][part][tile_rows][2]: maximum (log2 units), sum
  int32_t* tile_parts; // [place]: parts that its tile was split into
};

struct ScoreAttentionPlan {
  int tile_rows; // 16 (key streaming), 64 or 128 (key tiles in LDS)
  int waves;     // of a block: 4, or 8 (128 rows)
  int row_tiles;
  bool packed;
  int parts, part_units;
  size_t partial_bytes; // 0: not split
};

// Row tiles: 16 and 128 rows for every head dimension, 64, and 128 in 8 wavefronts, up to
// 128.
constexpr bool score_tile_supported(int tile_rows, int waves, int head_dim) {
  return tile_rows == 16 || (tile_rows == 128 && waves == 4) || head_dim <= 128;
}

// Blocks that a CU holds at once, by registers (16 rows, whose wavefronts keep K and V
// chunks in them) and LDS (64 and 128 rows).
constexpr int score_stream_blocks_per_cu(bool f16, int head_dim) {
  return head_dim <= 64 ? 4 : head_dim <= (f16 ? 128 : 96) ? 3 : head_dim <= 160 ? 2 : 1;
}
constexpr int score_tile_blocks_per_cu(int tile_rows, int waves, bool f16, int head_dim) {
  if (waves == 8) return 1;
  if (tile_rows == 64) return f16 || head_dim <= 64 ? 2 : 1;
  return head_dim <= 128 ? 2 : 1;
}
constexpr int score_tile_waves_per_simd(int tile_rows, int waves, bool f16, int head_dim) {
  return waves / 4 * score_tile_blocks_per_cu(tile_rows, waves, f16, head_dim);
}

constexpr int score_blocks_per_cu(int tile_rows, int waves, bool f16, int head_dim) {
  return tile_rows == 16 ? score_stream_blocks_per_cu(f16, head_dim)
                         : score_tile_blocks_per_cu(tile_rows, waves, f16, head_dim);
}

// Row tiles' places: so many times row_tiles.
inline int64_t score_groups(bool packed, int64_t num_seqs, int64_t num_kv_heads) {
  return packed ? num_kv_heads : num_seqs * num_kv_heads;
}

// Items that follow each other on one XCD: a group's `inner` ones, where the groups share
// out evenly; else fewer, for some eight runs on each.
inline int64_t score_run(int64_t groups, int64_t inner) {
  return groups % kScoreXcds == 0 ? inner : std::max<int64_t>(1, std::min(inner, groups * inner / (8 * kScoreXcds)));
}

// Blocks of one launch: whole rounds of runs.
inline int64_t score_grid(int64_t groups, int64_t inner) {
  const int64_t round = kScoreXcds * score_run(groups, inner);
  return (groups * inner + round - 1) / round * round;
}

inline unsigned score_blocks(const ScoreAttentionParams& p) {
  return (unsigned)score_grid(score_groups(p.packed, p.t.num_seqs, p.t.num_kv_heads), (int64_t)p.row_tiles * p.parts);
}

// score_tiles.hip: the attention itself, of row tiles of 64 (head_dim up to 128) and 128
// rows.
hipError_t launch_score_tiles(const ScoreAttentionPlan& plan, const ScoreAttentionParams& params, int dtype, int head_dim,
                              hipStream_t stream);

// The attention, then the merge of what was split.
hipError_t launch_score_attention(const ScoreAttentionPlan& plan, const ScoreAttentionParams& params, int dtype,
                                  int head_dim, hipStream_t stream);

// Weights of keys.
struct ScoreWeightsParams {
  ScoreTables t;
  ScoreRules r;
  float* weights;
  float decay;
  const int32_t* fresh_from; // may be null: seq_len - q_len
};

// Keys of one wavefront: as many as 64 registers hold the rows of (64 at most).
constexpr int weights_unit_tokens(int elem_bytes, int head_dim) {
  return head_dim * elem_bytes <= 256 ? 64 : head_dim * elem_bytes <= 512 ? 32 : 16;
}

// split: the rows are shared out among a block's wavefronts, not the keys.
hipError_t launch_score_weights(const ScoreWeightsParams& params, int dtype, int head_dim, bool split, hipStream_t stream);

// Which tokens stay.  Slots that a block steps over at a time, at most: the kernel's slot
// numbers pass a request's length by less than that.
constexpr int kSelectStep = 4096;

struct SelectTokensParams {
  const float* weights;
  int32_t* positions;
  const int32_t* block_tables; // [num_layers][num_seqs][block_table_stride]
  int32_t block_table_stride;
  const int32_t* seq_lens;
  const int32_t* next_positions; // may be null: seq_lens
  const int32_t* kept_lens;      // may be null: 0
  const int32_t* keep_lens;
  int32_t* moves;
  int32_t* num_moves;
  int32_t* new_seq_lens; // may be null
  int64_t num_pages;
  int32_t num_layers, num_seqs, num_kv_heads, page_size, max_seq_len, max_moves, recent, first;
  uint64_t page_magic;
  int32_t page_magic_shift;
};

hipError_t launch_select_tokens(const SelectTokensParams& params, int compute_units, hipStream_t stream);

// Moves.  Those of one row that its blocks step over at a time, at most: the kernel's
// numbers of moves pass max_moves by less than that.
constexpr int kMoveStep = 1 << 23;

struct MoveTokensParams {
  void* key_pool;
  void* value_pool;
  float* weights;     // may be null
  int32_t* positions; // may be null
  const int32_t* block_tables;
  int32_t block_table_stride;
  const int32_t* moves;
  const int32_t* num_moves;
  int64_t num_pages;
  int32_t num_layers, num_seqs, num_kv_heads, page_size, max_moves;
  uint64_t page_magic;
  int32_t page_magic_shift;
};

hipError_t launch_move_tokens(const MoveTokensParams& params, int64_t row_bytes, hipStream_t stream);

} // namespace mvr
