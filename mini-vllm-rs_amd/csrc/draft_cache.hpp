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

hipError_t launch_copy_pages(const CopyPagesParams& params, int64_t row_bytes, hipStream_t stream);

} // namespace mvr
