// Internal launch interface of the drafted-tree attention kernels
// (draft_attention.hip).  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace mvr {

// Keys are split between parts in units of 64 tokens.
constexpr int kDraftUnitTokens = 64;
// Parts of one row tile, at most.
constexpr int kDraftMaxParts = 64;
constexpr int kDraftXcds = 8;

// Row tiles: 16 rows for every head dimension, 128 too, 32 and 64 up to 128.
constexpr bool draft_tile_supported(int tile_rows, int head_dim) {
  return tile_rows == 16 || tile_rows == 128 || ((tile_rows == 32 || tile_rows == 64) && head_dim <= 128);
}

// Blocks that a CU holds at once, by registers (16- and 32-row tiles, whose
// wavefronts keep K and V chunks in them) and LDS (64 and 128 rows).
constexpr int draft_blocks_per_cu(int tile_rows, bool f16, int head_dim) {
  if (tile_rows == 16) return head_dim <= 64 ? 4 : head_dim <= (f16 ? 128 : 96) ? 3 : head_dim <= 160 ? 2 : 1;
  if (tile_rows == 32) return head_dim <= 64 ? 3 : f16 || head_dim <= 96 ? 2 : 1;
  if (tile_rows == 64) return f16 || head_dim <= 64 ? 2 : 1;
  return head_dim <= 128 ? 2 : 1;
}

// One launch.  A row tile holds tile_rows grouped query rows rho = r * q_len +
// i of one (request, KV head): r the query head within its group, i the draft.
// An item is one part of one row tile's keys.
struct DraftAttentionParams {
  const void* q;
  int64_t q_stride_head, q_stride_token;
  const void* key_pool;
  const void* value_pool;
  const int32_t* block_tables;
  int32_t block_table_stride;
  const int32_t* seq_lens;  // may be null: max_seq_len
  const int32_t* cu_q_lens; // may be null: max_q_len
  int32_t max_seq_len, max_q_len;
  void* out;
  int64_t out_stride_head, out_stride_token;
  const uint32_t* masks; // [token][mask_words]
  int32_t mask_words;
  int32_t num_seqs, num_kv_heads, group_size, page_size;
  uint32_t last_page; // num_pages - 1
  uint64_t page_magic; // page of token t = t * page_magic >> page_magic_shift (page_divider)
  int32_t page_magic_shift;
  int32_t row_tiles; // of the longest request, per (request, KV head)
  // 0: every row tile is one item, found from the block index (of by_length: the
  // longest requests first).  Otherwise parts
  // of at most part_units key units (longer ones where that makes more than
  // kDraftMaxParts), found by a scan of the length tables, whose items' partial
  // results lie in the slot of the item's number; max_items of them.  Where the
  // device tables hold more items than that, tiles are not split.
  int32_t part_units, max_items, by_length;
  float* partial_o;  // [max_items][tile_rows][head_dim]
  float* partial_ml; // [max_items][tile_rows][2]: maximum (log2 units), sum
  float scale_log2;
};

struct DraftAttentionPlan {
  int tile_rows; // 16 or 32 (key streaming), 64 or 128 (key tiles in LDS)
  int row_tiles;
  int part_units; // 0: not split
  int blocks;
  int by_length;
  int max_items; // 0: no partials
  size_t partial_bytes;
};

// draft_tiles.hip: the attention itself, of row tiles of 64 (head_dim up to 128)
// and 128 rows.
hipError_t launch_draft_tiles(const DraftAttentionPlan& plan, const DraftAttentionParams& params, int dtype,
                              int head_dim, hipStream_t stream);

// The attention, then the merge of what was split.
hipError_t launch_draft_attention(const DraftAttentionPlan& plan, const DraftAttentionParams& params, int dtype,
                                  int head_dim, hipStream_t stream);

} // namespace mvr
