/*
 * mvr_draft — the calls of speculative decoding with a tree of drafted
 * tokens, and of forked requests, on the paged KV cache of mvr_attn.h.
 *
 * The reference drafts and verifies a chain: the drafts of a request are its
 * last q_len tokens, and draft i sees the drafts before it
 * (generation/text_generation.rs:981-1066); rejected drafts are dropped by
 * truncating the cache (text_generation.rs:531-537).  A tree verifies several
 * continuations at once.  One step of a layer is then
 *   mvr_norm_rope_append      norms of Q and K per head, rotation at a position
 *                             of each token's own (a node's depth, which is not
 *                             its cache slot), append to the pages;
 *   mvr_paged_attention_tree  every node attends the cache and its ancestors;
 * and once per step, for the tables of all layers,
 *   mvr_compact_drafts        the accepted path moves to the front of the
 *                             drafts' slots, and the new lengths come out;
 *   mvr_copy_pages            copies of pages for a request that is forked or
 *                             whose last page is shared.
 *
 * Pools, block tables, lengths, strides, status codes, mvr_last_error(), the
 * streams and the rules on device tables are those of mvr_attn.h: every call
 * is stream-ordered and asynchronous and allocates nothing, works on the
 * current device, can be captured into a graph, and with
 * MVR_ATTN_CHECKED=true (a development mode, not under capture) checks its
 * device tables on the host first.  Kernels read and write no page outside the
 * pool: an attention call reads the last page in place of one outside, the
 * calls that write leave such rows out.  Requests must own the pages that a
 * call writes: two writers of one page race, and so do calls on different
 * streams that are not ordered, where one of them writes what the other uses.
 */
#ifndef MVR_DRAFT_H
#define MVR_DRAFT_H

#include "mvr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Attention of drafted trees ------------------------------------------ */

/* Which drafts each draft sees.  The q_len drafts of request b are its last
   q_len tokens, in the cache slots seq_len - q_len .. seq_len - 1 (appended
   before this call).  Query i of the request sees every token before them, and
   draft slot s (0 <= s < q_len) iff bit s % 32 of word s / 32 of its mask row
   is set: its ancestors and itself for a tree, any set in general.  Bits from
   q_len on are ignored.  A query that sees no key at all has output 0. */
typedef struct mvr_draft_trees {
  const uint32_t* masks; /* device [total_q][mask_words], a row per packed query token */
  int32_t mask_words;    /* words per row, >= ceil(max_q_len / 32) */
} mvr_draft_trees;

/* mvr_paged_attention with the drafts' own masks in place of the causal one.
   Same arguments, layouts, dtypes, head dimensions (multiples of 32 up to
   256), page sizes (any; nothing is repacked) and hints.  Scores, softmax state
   and sums are held in 32 bits.  F16 probabilities enter the product with V with
   20 bits; where requests have more than 32 rows (query heads per KV head x
   drafts) the plan may round them to F16, and the sum is then that of the
   rounded ones.  Differences to mvr_paged_attention:
     - a request may have q_len 0 (no drafts this step): nothing is computed
       for it, so total_q, where given, lies in [0, num_seqs * max_q_len].  All
       of them may; max_q_len is 1 at least and q, out and masks are there even
       so (a step without any token can leave the call out);
     - rows of q and out from cu_q_lens[num_seqs] on are neither read nor
       written;
     - a device q_len above max_q_len is clamped to it;
     - a NaN or an infinity in the K or V row of a draft reaches only the rows
       that see the draft.
   Host tables (seq_lens_host, cu_q_lens_host) and sum_seq_lens only shape the
   launch; rows are computed from the device tables whatever they hold. */
int mvr_paged_attention_tree(const mvr_paged_attention_args* args, const mvr_draft_trees* trees);

/* Bytes of workspace that the call needs (0: none; contents need no
   initialisation and are dead after the call).  Depends on the scalars and the
   hints.  With less workspace, or none, the call still runs: it splits the
   keys as far as its workspace allows, down to not at all.  Calls that share
   a workspace must not overlap in time. */
size_t mvr_paged_attention_tree_workspace_size(const mvr_paged_attention_args* args, const mvr_draft_trees* trees);

/* Host-side checks of the tables the device will read: lengths and pages as
   mvr_paged_attention_validate does (q_len 0 allowed), and, where masks_host
   is given, that every query sees itself (a row that does not see its own slot
   is legal, but in a tree it is a mistake).  Any pointer may be NULL to skip
   its checks.  Launches nothing. */
int mvr_paged_attention_tree_validate(const mvr_paged_attention_args* args, const mvr_draft_trees* trees,
                                      const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                      const int32_t* cu_q_lens_host, const uint32_t* masks_host);

/* ---- Norm, rotation and append ------------------------------------------- */

typedef struct mvr_head_norms {
  const void* q_weight;     /* [head_dim], activation dtype; NULL: queries are not normalised */
  const void* k_weight;     /* [head_dim]; NULL: keys are not normalised */
  float eps;                /* added to the mean square; >= 0 and finite */
  const int32_t* positions; /* device [total_q]: rotary position of each packed token; NULL: its cache slot */
} mvr_head_norms;

/* mvr_rope_append with a root-mean-square norm of every query and key row
   before the rotation, and a rotary position for each token:
     y = x * weight / sqrt(mean(x^2) + eps),
     (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of rope_type,
   in 32 bits, rounded once where it is written (mvr_rope_append, whose
   rounding follows the reference's kernels, rounds every product and sum).
   The row of token i of request b goes to slot seq_len - q_len + i, wherever
   it is rotated to.  Arguments are mvr_rope_append's; here
     - a request may have q_len 0, and total_q, 1 at least, may exceed
       cu_q_lens[num_seqs] (a padded batch): rows from there on do not matter
       and are not written.  A step without any token makes no call, or one on
       a padded batch;
     - rope_len need only cover the positions: rows whose position is outside
       [0, rope_len), or whose slot is outside [0, max_seq_len), or whose page
       is outside the pool, are left out. */
int mvr_norm_rope_append(const mvr_rope_append_args* args, const mvr_head_norms* norms);

/* Host-side checks of the tables: mvr_rope_append_validate's (q_len 0 and a
   padded total_q allowed), and positions inside the rotary tables.  Any pointer
   may be NULL to skip its checks.  Launches nothing. */
int mvr_norm_rope_append_validate(const mvr_rope_append_args* args, const mvr_head_norms* norms,
                                  const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                  const int32_t* cu_q_lens_host, const int32_t* positions_host,
                                  const uint8_t* page_writable_host);

/* ---- Compaction of accepted drafts --------------------------------------- */

/* After verification: of the q_len drafts of request b (slots first = seq_len -
   q_len on), the accepted_lens[b] ones whose indices accepted[b] lists, in
   strictly ascending order, stay; their K and V rows move to slots first,
   first + 1, ... in the pages of every layer.  Rows are copied bit for bit (a
   node at depth d was rotated for position first + d, which is its new slot).
   Pages that the new length leaves empty are the caller's to free. */
typedef struct mvr_compact_drafts_args {
  int32_t dtype;             /* mvr_dtype */
  int32_t num_layers;        /* block tables per request: one for each layer that shares the pools, >= 1 */
  int32_t num_seqs;
  int32_t num_kv_heads;
  int32_t head_dim;          /* any positive value */
  int32_t page_size;         /* any positive value */
  int64_t num_pages;
  int32_t max_pages_per_seq; /* row stride of block_tables */
  int32_t max_seq_len;       /* >= every seq_len */
  int32_t max_accepted;      /* row stride of accepted, >= every accepted_lens */
  void* key_pool;            /* [num_pages, 1, num_kv_heads, page_size, head_dim] */
  void* value_pool;
  const int32_t* block_tables;  /* device [num_layers][num_seqs][max_pages_per_seq] */
  const int32_t* seq_lens;      /* device [num_seqs], drafts included */
  const int32_t* cu_q_lens;     /* device [num_seqs + 1]; q_len 0 allowed */
  const int32_t* accepted;      /* device [num_seqs][max_accepted]: indices in [0, q_len), strictly ascending */
  const int32_t* accepted_lens; /* device [num_seqs], 0 .. min(q_len, max_accepted) */
  int32_t* new_seq_lens;        /* device [num_seqs], written: seq_len - q_len + accepted_lens; NULL: not wanted; must
                                   overlap none of the tables above */
  void* stream;
} mvr_compact_drafts_args;

/* One launch for all layers.  An index outside [0, q_len), one that is not
   above the index before it, or a row whose page is outside the pool is left
   out (only a broken table holds one); an accepted_lens outside its range is
   clamped into it. */
int mvr_compact_drafts(const mvr_compact_drafts_args* args);

/* Host-side checks of the tables: lengths, indices ascending and below q_len,
   page ids inside the pool, and no page that is written for two requests or
   layers.  Any pointer may be NULL to skip its checks.  Launches nothing. */
int mvr_compact_drafts_validate(const mvr_compact_drafts_args* args, const int32_t* block_tables_host,
                                const int32_t* seq_lens_host, const int32_t* cu_q_lens_host,
                                const int32_t* accepted_host, const int32_t* accepted_lens_host);

/* ---- Copies of pages ----------------------------------------------------- */

typedef struct mvr_copy_pages_args {
  int32_t dtype;          /* mvr_dtype */
  int32_t num_copies;     /* >= 0 */
  int32_t num_kv_heads;
  int32_t head_dim;       /* any positive value */
  int32_t page_size;      /* any positive value */
  int64_t num_pages;
  void* key_pool;
  void* value_pool;
  const int32_t* src_pages; /* device [num_copies] */
  const int32_t* dst_pages; /* device [num_copies]: all different, none of them a source of this call */
  const int32_t* tokens;    /* device [num_copies]: leading tokens to copy, clamped to 0 .. page_size; NULL: whole pages */
  void* stream;
} mvr_copy_pages_args;

/* Copies K and V pages bit for bit: for a fork the pages of all layers in one
   launch, the partly filled ones up to their tokens (the destination's other
   slots keep what they hold).  A copy with a page outside the pool is left
   out. */
int mvr_copy_pages(const mvr_copy_pages_args* args);

/* Host-side checks: page ids inside the pool, destinations all different and
   none of them a source, token counts within a page.  Any pointer may be NULL
   to skip its checks.  Launches nothing. */
int mvr_copy_pages_validate(const mvr_copy_pages_args* args, const int32_t* src_pages_host,
                            const int32_t* dst_pages_host, const int32_t* tokens_host);

#ifdef __cplusplus
}
#endif
#endif /* MVR_DRAFT_H */
