// Internal launch interface of the cache kernels beside drafted-tree attention
// (draft_cache.hip).  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mvr {

struct NormRopeAppendParams {
  const void* q;
  int64_t q_stride_head, q_stride_token;
  const void* k;
  int64_t k_stride_head, k_stride_token;
  const void* v;
  int64_t v_stride_head, v_stride_token;
  const void* q_weight; // [head_dim] or null
  const void* k_weight;
  float eps;
  const void* cos_table; // [rope_len, head_dim / 2]
  const void* sin_table;
  const int32_t* positions; // [total_q] or null: the cache slot
  int32_t rope_len;
  const int32_t* block_tables;
  int32_t block_table_stride;
  const int32_t* seq_lens;  // may be null: max_seq_len
  const int32_t* cu_q_lens; // may be null: one request of total_q tokens
  int32_t max_seq_len;
  void* q_out;
  int64_t q_out_stride_head, q_out_stride_token;
  void* key_pool;
  void* value_pool;
  int64_t num_pages;
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, total_q;
};

// Lanes of a row, a power of two (8 elements each), and wavefronts of a token.
inline int append_row_lanes_log2(int head_dim) {
  int lanes_log2 = 0;
  while ((8 << lanes_log2) < head_dim) lanes_log2++;
  return lanes_log2;
}
inline int append_token_waves(int rows, int head_dim) { return ((rows << append_row_lanes_log2(head_dim)) + 63) / 64; }

// dtype: 0 = F32, 1 = F16; rope_type: 0 = Neox, 1 = Interleaved.
hipError_t launch_norm_rope_append(const NormRopeAppendParams& params, int dtype, int rope_type, hipStream_t stream);

struct CompactDraftsParams {
  void* key_pool;
  void* value_pool;
  const int32_t* block_tables; // [num_layers][num_seqs][block_table_stride]
  int32_t block_table_stride;
  const int32_t* seq_lens;
  const int32_t* cu_q_lens;
  const int32_t* accepted; // [num_seqs][max_accepted]
  const int32_t* accepted_lens;
  int32_t* new_seq_lens; // or null
  int64_t num_pages;
  int32_t num_layers, num_seqs, num_kv_heads, page_size, max_seq_len, max_accepted;
};

hipError_t launch_compact_drafts(const CompactDraftsParams& params, int64_t row_bytes, hipStream_t stream);

struct CopyPagesParams {
  void* key_pool;
  void* value_pool;
  const int32_t* src_pages;
  const int32_t* dst_pages;
  const int32_t* tokens; // or null: whole pages
  int64_t num_pages;
  int32_t num_copies, num_kv_heads, page_size;
};

// Bytes that one access moves: the widest that rows and pools allow.
inline int cache_vector_bytes(int64_t row_bytes, const void* a, const void* b) {
  const uintptr_t align = (uintptr_t)a | (uintptr_t)b | (uintptr_t)row_bytes;
  return align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : 2;
}

constexpr int kCopyPieceVecs = 4 * 256; // that a block copies

// Blocks of one page's copy in one pool.
inline int64_t copy_pages_pieces(int64_t rows, int64_t row_bytes, const void* a, const void* b) {
  const int64_t vecs = rows * (row_bytes / cache_vector_bytes(row_bytes, a, b));
  return (vecs + kCopyPieceVecs - 1) / kCopyPieceVecs;
}

hipError_t launch_copy_pages(const CopyPagesParams& params, int64_t row_bytes, hipStream_t stream);

} // namespace mvr
