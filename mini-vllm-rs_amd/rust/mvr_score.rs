// Rust binding of the calls on scores of libmvr_attn.so (C ABI: include/mvr_score.h).
//
// Drop-in module for lun0522/mini-vllm-rs beside mvr_attn.rs
// (src/models/backends/mvr_score.rs).  Its callers are the attention of models whose
// scores are capped, sloped or masked (in the place of forward_paged_attention,
// src/models/backends/common.rs:739-817), and a cache manager that cuts requests to
// the tokens which got most attention (beside kv_cache/paged_cache.rs).
//
// tests/test_score_api.py parses this file and the header and checks that structs and
// prototypes agree.
#![allow(dead_code)]

use std::ffi::{c_int, c_void, CStr};

use super::mvr_attn::{mvr_last_error, MvrPagedAttentionArgs, MVR_OK};

#[repr(C)]
pub struct MvrScoreRules {
    pub cap: f32,                // 0: scores are not capped
    pub window: i32,             // 0: any number of keys
    pub slopes: *const f32,      // device [num_q_heads]; null: none
    pub first_keys: *const i32,  // device [total_q]; null: 0
    pub prefix_lens: *const i32, // device [num_seqs]; null: none
    pub lse: *mut f32,           // device, (head h, token n) at h * lse_stride_head + n; null: not wanted
    pub lse_stride_head: i64,
}

#[repr(C)]
pub struct MvrKeyWeights {
    pub weights: *mut f32, // device [num_pages][num_kv_heads][page_size], updated
    pub decay: f32,
    pub fresh_from: *const i32, // device [num_seqs]; null: seq_len - q_len
}

#[repr(C)]
pub struct MvrSelectTokensArgs {
    pub num_layers: i32,
    pub num_seqs: i32,
    pub num_kv_heads: i32,
    pub page_size: i32,
    pub num_pages: i64,
    pub max_pages_per_seq: i32,
    pub max_seq_len: i32,
    pub max_moves: i32,
    pub recent: i32,
    pub first: i32,
    pub weights: *const f32,      // device [num_pages][num_kv_heads][page_size]
    pub positions: *mut i32,      // same shape; of slots from kept_lens on written
    pub block_tables: *const i32, // device [num_layers][num_seqs][max_pages_per_seq]
    pub seq_lens: *const i32,
    pub next_positions: *const i32, // null: seq_lens
    pub kept_lens: *const i32,      // null: 0
    pub keep_lens: *const i32,
    pub moves: *mut i32,        // device [num_layers][num_seqs][num_kv_heads][max_moves][2], written
    pub num_moves: *mut i32,    // device [num_layers][num_seqs][num_kv_heads], written
    pub new_seq_lens: *mut i32, // device [num_seqs], written; null: not wanted
    pub stream: *mut c_void,
}

#[repr(C)]
pub struct MvrMoveTokensArgs {
    pub dtype: i32, // MVR_DTYPE_*
    pub num_layers: i32,
    pub num_seqs: i32,
    pub num_kv_heads: i32,
    pub head_dim: i32,
    pub page_size: i32,
    pub num_pages: i64,
    pub max_pages_per_seq: i32,
    pub max_moves: i32,
    pub key_pool: *mut c_void,
    pub value_pool: *mut c_void,
    pub weights: *mut f32,   // null: none to move
    pub positions: *mut i32, // null: none to move
    pub block_tables: *const i32,
    pub moves: *const i32,
    pub num_moves: *const i32,
    pub stream: *mut c_void,
}

extern "C" {
    pub fn mvr_paged_attention_scored(args: *const MvrPagedAttentionArgs, rules: *const MvrScoreRules) -> c_int;
    pub fn mvr_paged_attention_scored_workspace_size(args: *const MvrPagedAttentionArgs,
                                                     rules: *const MvrScoreRules) -> usize;
    pub fn mvr_paged_attention_scored_validate(args: *const MvrPagedAttentionArgs, rules: *const MvrScoreRules,
                                               block_tables_host: *const i32, seq_lens_host: *const i32,
                                               cu_q_lens_host: *const i32, first_keys_host: *const i32,
                                               prefix_lens_host: *const i32, slopes_host: *const f32) -> c_int;
    pub fn mvr_attention_weights(args: *const MvrPagedAttentionArgs, rules: *const MvrScoreRules,
                                 weights: *const MvrKeyWeights) -> c_int;
    pub fn mvr_attention_weights_validate(args: *const MvrPagedAttentionArgs, rules: *const MvrScoreRules,
                                          weights: *const MvrKeyWeights, block_tables_host: *const i32,
                                          seq_lens_host: *const i32, cu_q_lens_host: *const i32,
                                          first_keys_host: *const i32, prefix_lens_host: *const i32,
                                          slopes_host: *const f32, fresh_from_host: *const i32) -> c_int;
    pub fn mvr_select_tokens(args: *const MvrSelectTokensArgs) -> c_int;
    pub fn mvr_select_tokens_validate(args: *const MvrSelectTokensArgs, block_tables_host: *const i32,
                                      seq_lens_host: *const i32, next_positions_host: *const i32,
                                      kept_lens_host: *const i32, keep_lens_host: *const i32) -> c_int;
    pub fn mvr_move_tokens(args: *const MvrMoveTokensArgs) -> c_int;
    pub fn mvr_move_tokens_validate(args: *const MvrMoveTokensArgs, block_tables_host: *const i32,
                                    moves_host: *const i32, num_moves_host: *const i32) -> c_int;
}

/// The library's message for a failed call, as candle_core::bail! would carry it.
fn check(rc: c_int) -> candle_core::Result<()> {
    if rc == MVR_OK {
        return Ok(());
    }
    let msg = unsafe { CStr::from_ptr(mvr_last_error()) }.to_string_lossy().into_owned();
    candle_core::bail!("{msg} (mvr_attn error {rc})")
}

pub fn scored_workspace_size(args: &MvrPagedAttentionArgs, rules: &MvrScoreRules) -> usize {
    unsafe { mvr_paged_attention_scored_workspace_size(args, rules) }
}

/// Attention with capped, sloped or masked scores, and the rows' log-sum-exps.
pub fn paged_attention_scored(args: &MvrPagedAttentionArgs, rules: &MvrScoreRules) -> candle_core::Result<()> {
    check(unsafe { mvr_paged_attention_scored(args, rules) })
}

/// What each cached key got from these rows, added to what it had.
pub fn attention_weights(args: &MvrPagedAttentionArgs, rules: &MvrScoreRules,
                         weights: &MvrKeyWeights) -> candle_core::Result<()> {
    check(unsafe { mvr_attention_weights(args, rules, weights) })
}

/// Which tokens of every layer, request and KV head stay, as moves.
pub fn select_tokens(args: &MvrSelectTokensArgs) -> candle_core::Result<()> {
    check(unsafe { mvr_select_tokens(args) })
}

/// The moves of K and V rows, weights and positions.
pub fn move_tokens(args: &MvrMoveTokensArgs) -> candle_core::Result<()> {
    check(unsafe { mvr_move_tokens(args) })
}
