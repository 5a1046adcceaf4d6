// Rust binding of the drafted-tree calls of libmvr_attn.so (C ABI: include/mvr_draft.h).
//
// Drop-in module for lun0522/mini-vllm-rs beside mvr_attn.rs
// (src/models/backends/mvr_draft.rs).  Its callers are the target's
// verification forward (generation/text_generation.rs:1015-1066), once drafts
// form trees, and, in the place of truncate_cache after a rejection
// (text_generation.rs:531-537), the compaction of the accepted path.
//
// tests/test_draft_api.py parses this file and the header and checks that
// structs and prototypes agree.
#![allow(dead_code)]

use std::ffi::{c_int, c_void, CStr};

use super::mvr_attn::{mvr_last_error, MvrPagedAttentionArgs, MvrRopeAppendArgs, MVR_OK};

#[repr(C)]
pub struct MvrDraftTrees {
    pub masks: *const u32, // device [total_q][mask_words]
    pub mask_words: i32,   // >= ceil(max_q_len / 32)
}

#[repr(C)]
pub struct MvrHeadNorms {
    pub q_weight: *const c_void, // [head_dim], activation dtype; null: queries are not normalised
    pub k_weight: *const c_void,
    pub eps: f32,
    pub positions: *const i32, // device [total_q]; null: each token's cache slot
}

#[repr(C)]
pub struct MvrCompactDraftsArgs {
    pub dtype: i32, // MVR_DTYPE_*
    pub num_layers: i32,
    pub num_seqs: i32,
    pub num_kv_heads: i32,
    pub head_dim: i32,
    pub page_size: i32,
    pub num_pages: i64,
    pub max_pages_per_seq: i32,
    pub max_seq_len: i32,
    pub max_accepted: i32,
    pub key_pool: *mut c_void,
    pub value_pool: *mut c_void,
    pub block_tables: *const i32, // device [num_layers][num_seqs][max_pages_per_seq]
    pub seq_lens: *const i32,
    pub cu_q_lens: *const i32,
    pub accepted: *const i32, // device [num_seqs][max_accepted], ascending
    pub accepted_lens: *const i32,
    pub new_seq_lens: *mut i32, // device [num_seqs], written; null: not wanted
    pub stream: *mut c_void,
}

#[repr(C)]
pub struct MvrCopyPagesArgs {
    pub dtype: i32,
    pub num_copies: i32,
    pub num_kv_heads: i32,
    pub head_dim: i32,
    pub page_size: i32,
    pub num_pages: i64,
    pub key_pool: *mut c_void,
    pub value_pool: *mut c_void,
    pub src_pages: *const i32,
    pub dst_pages: *const i32,
    pub tokens: *const i32, // device [num_copies]; null: whole pages
    pub stream: *mut c_void,
}

extern "C" {
    pub fn mvr_paged_attention_tree(args: *const MvrPagedAttentionArgs, trees: *const MvrDraftTrees) -> c_int;
    pub fn mvr_paged_attention_tree_workspace_size(args: *const MvrPagedAttentionArgs,
                                                   trees: *const MvrDraftTrees) -> usize;
    pub fn mvr_paged_attention_tree_validate(args: *const MvrPagedAttentionArgs, trees: *const MvrDraftTrees,
                                             block_tables_host: *const i32, seq_lens_host: *const i32,
                                             cu_q_lens_host: *const i32, masks_host: *const u32) -> c_int;
    pub fn mvr_norm_rope_append(args: *const MvrRopeAppendArgs, norms: *const MvrHeadNorms) -> c_int;
    pub fn mvr_norm_rope_append_validate(args: *const MvrRopeAppendArgs, norms: *const MvrHeadNorms,
                                         block_tables_host: *const i32, seq_lens_host: *const i32,
                                         cu_q_lens_host: *const i32, positions_host: *const i32,
                                         page_writable_host: *const u8) -> c_int;
    pub fn mvr_compact_drafts(args: *const MvrCompactDraftsArgs) -> c_int;
    pub fn mvr_compact_drafts_validate(args: *const MvrCompactDraftsArgs, block_tables_host: *const i32,
                                       seq_lens_host: *const i32, cu_q_lens_host: *const i32,
                                       accepted_host: *const i32, accepted_lens_host: *const i32) -> c_int;
    pub fn mvr_copy_pages(args: *const MvrCopyPagesArgs) -> c_int;
    pub fn mvr_copy_pages_validate(args: *const MvrCopyPagesArgs, src_pages_host: *const i32,
                                   dst_pages_host: *const i32, tokens_host: *const i32) -> c_int;
}

/// The library's message for a failed call, as candle_core::bail! would carry it.
fn check(rc: c_int) -> candle_core::Result<()> {
    if rc == MVR_OK {
        return Ok(());
    }
    let msg = unsafe { CStr::from_ptr(mvr_last_error()) }.to_string_lossy().into_owned();
    candle_core::bail!("{msg} (mvr_attn error {rc})")
}

pub fn tree_workspace_size(args: &MvrPagedAttentionArgs, trees: &MvrDraftTrees) -> usize {
    unsafe { mvr_paged_attention_tree_workspace_size(args, trees) }
}

/// Attention of every request's drafted tree, each draft on the cache and the drafts that its mask names.
pub fn paged_attention_tree(args: &MvrPagedAttentionArgs, trees: &MvrDraftTrees) -> candle_core::Result<()> {
    check(unsafe { mvr_paged_attention_tree(args, trees) })
}

/// rope_append with norms of Q and K per head before it and a rotary position for each token.
pub fn norm_rope_append(args: &MvrRopeAppendArgs, norms: &MvrHeadNorms) -> candle_core::Result<()> {
    check(unsafe { mvr_norm_rope_append(args, norms) })
}

/// The accepted drafts' rows to the front of the drafts' slots, in the pages of every layer.
pub fn compact_drafts(args: &MvrCompactDraftsArgs) -> candle_core::Result<()> {
    check(unsafe { mvr_compact_drafts(args) })
}

/// Copies of pages, for forked requests.
pub fn copy_pages(args: &MvrCopyPagesArgs) -> candle_core::Result<()> {
    check(unsafe { mvr_copy_pages(args) })
}
