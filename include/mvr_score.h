/*
 * mvr_score — attention over the paged KV cache of mvr_attn.h whose scores are
 * bent or masked as models do it, the attention that each cached token gets, and
 * the cut of a cache to the tokens that got most.
 *
 * mvr_paged_attention is the softmax of scale * q . k under the causal mask.
 * Models cap those scores, lower them with the distance, or look at a window, at
 * one document of a packed prompt, at a prefix both ways; and a server whose
 * caches outgrow its memory keeps, of each layer, request and KV head, the tokens
 * that the queries looked at.  One step of a layer is then
 *   mvr_norm_rope_append         append, rotated at positions of the tokens' own
 *                                (mvr_draft.h): in a cache that was cut, a token's
 *                                slot is not its position;
 *   mvr_paged_attention_scored   the attention, and every row's log-sum-exp;
 *   mvr_attention_weights        what each key got from these rows, added up in a
 *                                pool beside the keys;
 * and where a request has outgrown its budget, for the tables of all layers,
 *   mvr_select_tokens            which tokens stay, as a list of moves;
 *   mvr_move_tokens              the moves of their K and V rows, weights and
 *                                positions into the slots that become free.
 *
 * Pools, block tables, lengths, strides, status codes, mvr_last_error(), the
 * streams and the rules on device tables are those of mvr_attn.h: every call is
 * stream-ordered and asynchronous and allocates nothing, works on the current
 * device, can be captured into a graph, and with MVR_ATTN_CHECKED=true (a
 * development mode, not under capture) checks its device tables on the host first.
 * Kernels read and write no page outside the pool: what would be read from one
 * outside is read from the last page, what would be written to one is left out.
 * Requests must own the pages that a call writes: two writers of one page race, and
 * so do calls on different streams that are not ordered, where one of them writes
 * what the other uses.
 */
#ifndef MVR_SCORE_H
#define MVR_SCORE_H

#include "mvr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Attention with bent and masked scores -------------------------------- */

/* Query i of request b lies in slot p = seq_len - q_len + i.  It sees the keys j
   with first <= j < last,
     last  = max(p + 1, min(prefix_lens[b], seq_len)),
     first = max(0, first_keys[n], p - window + 1)      (n: its packed token),
   each part only where it is given, with the score
     s = scale * q . k_j,   s = cap * tanh(s / cap),   s - slopes[h] * |p - j|.
   Distances and windows count cache slots: after a cut, whose moves change the
   order, only the cap and masks that end before the moved slots mean what they say.
   A query that sees no key has output 0 and log-sum-exp -infinity; so have those in
   slots below 0, of requests shorter than their query tokens (length 0 among them),
   which the checks refuse. */
typedef struct mvr_score_rules {
  float cap;                  /* > 0; 0: scores are not capped */
  int32_t window;             /* keys that a query sees at most, up to itself; 0: any number */
  const float* slopes;        /* device [num_q_heads], finite; NULL: none */
  const int32_t* first_keys;  /* device [total_q]: the first key of the token's document; NULL: 0 */
  const int32_t* prefix_lens; /* device [num_seqs]: leading keys that all queries of the request see; NULL: none */
  float* lse;                 /* device, log of the sum of e^score of (q head h, packed token n) at
                                 h * lse_stride_head + n; mvr_paged_attention_scored writes it (NULL: not wanted),
                                 mvr_attention_weights reads it */
  int64_t lse_stride_head;    /* elements */
} mvr_score_rules;

/* mvr_paged_attention under the rules above.  Same arguments, layouts, dtypes, head
   dimensions (multiples of 32 up to 256), page sizes (any; nothing is repacked) and
   hints.  Scores, softmax state and sums are held in 32 bits.  F16 probabilities
   enter the product with V with 20 bits, and calls of many rows round them to F16 for
   it (in steps of 2^-31 of a row's largest, where they are that small), not for the
   sum that divides them: their outputs are up to 1.4 times as far from the formula.
   A cap adds an error of 2^-20 of the capped score at most.  Differences to mvr_paged_attention:
     - a request may have q_len 0: nothing is computed for it, so total_q, where
       given, lies in [0, num_seqs * max_q_len];
     - rows of q, out and lse from cu_q_lens[num_seqs] on are neither read nor
       written;
     - a device q_len above max_q_len is clamped to it;
     - a launch holds 2^24 tiles of 16 rows (a row: a query token and a query head of
       its KV head's group), or up to an eighth less: calls of more are refused, counted by
       total_q where it and cu_q_lens are given, else by max_q_len for every request;
     - a NaN or an infinity in the K or V row of a key reaches only the rows that
       see the key.  An infinity in a V row may come out of those as an infinity or as a
       NaN (it is multiplied by a probability in parts, which may be 0): which of them is
       the plan's, and may change with the hints.
   Host tables (seq_lens_host, cu_q_lens_host) and sum_seq_lens only shape the
   launch, and with it the order of sums and the rounding of probabilities; rows are computed from the device tables whatever they hold. */
int mvr_paged_attention_scored(const mvr_paged_attention_args* args, const mvr_score_rules* rules);

/* Bytes of workspace that the call needs (0: none; 96 MiB at most; contents need no
   initialisation and are dead after the call).  Depends on the scalars and the
   hints.  With less workspace, or none, the call still runs: it splits the keys as
   far as its workspace allows, down to not at all.  Calls that share a workspace
   must not overlap in time. */
size_t mvr_paged_attention_scored_workspace_size(const mvr_paged_attention_args* args, const mvr_score_rules* rules);

/* Host-side checks of the tables the device will read: lengths and pages as
   mvr_paged_attention_validate does (q_len 0 allowed), first keys and prefixes that
   are not negative, finite slopes.  Any pointer may be NULL to skip its checks.
   Launches nothing. */
int mvr_paged_attention_scored_validate(const mvr_paged_attention_args* args, const mvr_score_rules* rules,
                                        const int32_t* block_tables_host, const int32_t* seq_lens_host,
                                        const int32_t* cu_q_lens_host, const int32_t* first_keys_host,
                                        const int32_t* prefix_lens_host, const float* slopes_host);

/* ---- The weight that keys get ---------------------------------------------- */

typedef struct mvr_key_weights {
  float* weights;            /* device [num_pages][num_kv_heads][page_size], updated */
  float decay;               /* what a key had is multiplied by it; finite, >= 0; 1 for plain sums, 0 for these rows' alone */
  const int32_t* fresh_from; /* device [num_seqs]: slots from here on had nothing yet (their weights are not read); NULL:
                                the request's query tokens, seq_len - q_len */
} mvr_key_weights;

/* For every key j < seq_len of every request and KV head,
     weights_j <- (j < fresh_from ? decay * weights_j : 0) + sum e^(score - lse)
   over the query rows that see the key (all of the request's tokens in the call and
   all query heads of the KV head), with the scores of mvr_paged_attention_scored
   under the same rules and the log-sum-exps that it wrote.  The arguments are that
   call's (value_pool, out and workspace are not used), or those of its last tokens
   alone: q, lse and cu_q_lens then start at the first of them.  Rows whose
   log-sum-exp is -infinity count nothing.  Sums are held in 32 bits, in an order
   that does not change from call to call.  Requests without query tokens are left as
   they are. */
int mvr_attention_weights(const mvr_paged_attention_args* args, const mvr_score_rules* rules,
                          const mvr_key_weights* weights);

/* Host-side checks of the tables: mvr_paged_attention_scored_validate's, fresh_from
   not negative, and no page whose weights would be updated for two requests.  Any
   pointer may be NULL to skip its checks.  Launches nothing. */
int mvr_attention_weights_validate(const mvr_paged_attention_args* args, const mvr_score_rules* rules,
                                   const mvr_key_weights* weights, const int32_t* block_tables_host,
                                   const int32_t* seq_lens_host, const int32_t* cu_q_lens_host,
                                   const int32_t* first_keys_host, const int32_t* prefix_lens_host,
                                   const float* slopes_host, const int32_t* fresh_from_host);

/* ---- Which tokens stay ------------------------------------------------------ */

/* Every layer and KV head of a request chooses its own keep_lens[b] tokens: those
   whose position is below `first` or among the last `recent` ones before all others
   (where they are too many, those in the lower slots), the others by descending weight
   (NaN counts as -infinity), at equal weights those in the lower slots.  Tokens that stay and lie below the new length stay where they are; the
   others move into the slots there that become free, both in ascending order, which
   is as few rows as can be moved, and in any order of execution the same.
   positions holds the position of each token in slots below kept_lens (what an
   earlier call left, moved with the rows); those of the tokens appended since are
   written here: the last slot holds position next_positions - 1, the one before it
   next_positions - 2, ... */
typedef struct mvr_select_tokens_args {
  int32_t num_layers;        /* block tables per request: one for each layer that shares the pools, >= 1 */
  int32_t num_seqs;
  int32_t num_kv_heads;
  int32_t page_size;         /* any positive value */
  int64_t num_pages;
  int32_t max_pages_per_seq; /* row stride of block_tables */
  int32_t max_seq_len;       /* >= every seq_len */
  int32_t max_moves;         /* moves that a row of `moves` holds, >= 1 */
  int32_t recent;            /* >= 0 */
  int32_t first;             /* >= 0 */
  const float* weights;      /* device [num_pages][num_kv_heads][page_size] */
  int32_t* positions;        /* device, same shape; of slots from kept_lens on written */
  const int32_t* block_tables;   /* device [num_layers][num_seqs][max_pages_per_seq] */
  const int32_t* seq_lens;       /* device [num_seqs] */
  const int32_t* next_positions; /* device [num_seqs]: position of the next token to come; NULL: seq_lens (no token
                                    was dropped before) */
  const int32_t* kept_lens;      /* device [num_seqs]: slots whose positions are known (above seq_len: all); NULL: 0 */
  const int32_t* keep_lens;      /* device [num_seqs]: tokens to keep; not below seq_len: all stay */
  int32_t* moves;                /* device [num_layers][num_seqs][num_kv_heads][max_moves][2]: from slot, to slot */
  int32_t* num_moves;            /* device [num_layers][num_seqs][num_kv_heads], written */
  int32_t* new_seq_lens;         /* device [num_seqs], written; NULL: not wanted */
  void* stream;
} mvr_select_tokens_args;

/* One launch for all layers.  A request that might need more than max_moves moves
   (min(keep_lens, seq_len - keep_lens) of them) is not cut: it has no moves, and its
   new length is its old one.  Entries of `moves` behind num_moves are not written.
   Written arrays must not overlap the tables or each other. */
int mvr_select_tokens(const mvr_select_tokens_args* args);

/* Host-side checks of the tables: lengths, positions that cover the tokens
   (next_positions >= seq_len >= kept_lens >= 0), protected tokens that fit (first +
   recent <= keep_lens, where a request is cut), room for the moves, page ids inside
   the pool, and no page of two requests or layers.  Any pointer may be NULL to skip
   its checks.  Launches nothing. */
int mvr_select_tokens_validate(const mvr_select_tokens_args* args, const int32_t* block_tables_host,
                               const int32_t* seq_lens_host, const int32_t* next_positions_host,
                               const int32_t* kept_lens_host, const int32_t* keep_lens_host);

/* ---- Moves of tokens -------------------------------------------------------- */

typedef struct mvr_move_tokens_args {
  int32_t dtype;             /* mvr_dtype of the pools */
  int32_t num_layers;
  int32_t num_seqs;
  int32_t num_kv_heads;
  int32_t head_dim;          /* any positive value */
  int32_t page_size;         /* any positive value */
  int64_t num_pages;
  int32_t max_pages_per_seq; /* row stride of block_tables */
  int32_t max_moves;
  void* key_pool;            /* [num_pages, 1, num_kv_heads, page_size, head_dim] */
  void* value_pool;
  float* weights;            /* [num_pages][num_kv_heads][page_size]; NULL: none to move */
  int32_t* positions;        /* same shape; NULL: none to move */
  const int32_t* block_tables; /* device [num_layers][num_seqs][max_pages_per_seq] */
  const int32_t* moves;        /* device [num_layers][num_seqs][num_kv_heads][max_moves][2]: from slot, to slot */
  const int32_t* num_moves;    /* device [num_layers][num_seqs][num_kv_heads], clamped into 0 .. max_moves */
  void* stream;
} mvr_move_tokens_args;

/* Copies each KV head's K and V rows, weights and positions from slot to slot, bit
   for bit, for all layers in one launch: mvr_select_tokens's moves, or any others
   among which no slot is moved to twice, or both to and from.  A move with a slot
   outside the block table's row or a page outside the pool is left out.  Pages that
   the new length leaves empty are the caller's to free. */
int mvr_move_tokens(const mvr_move_tokens_args* args);

/* Host-side checks: slots inside the block tables, page ids inside the pool, no slot
   moved to twice, or both to and from, of one row of moves.  Any pointer may be NULL
   to skip its checks.  Launches nothing. */
int mvr_move_tokens_validate(const mvr_move_tokens_args* args, const int32_t* block_tables_host,
                             const int32_t* moves_host, const int32_t* num_moves_host);

#ifdef __cplusplus
}
#endif
#endif /* MVR_SCORE_H */
