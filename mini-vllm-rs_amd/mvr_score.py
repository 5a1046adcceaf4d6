"""Python binding of the calls on scores of libmvr_attn.so (C ABI in include/mvr_score.h).

Attention whose scores are capped, sloped or masked, and a cache that is cut to the tokens which got most attention:
  * paged_attention_scored(...)  attention with a cap, slopes, a window, documents, a prefix, and the rows' log-sum-exps
                                 (beside mvr_attn.paged_attention);
  * attention_weights(...)       what each cached key got from these rows, added to what it had;
and where a request has outgrown its budget, over the block tables of all layers,
  * select_tokens(...)           which tokens of each KV head stay, as moves into the slots that become free;
  * move_tokens(...)             the moves of their K and V rows, weights and positions (beside mvr_draft.compact_drafts).

make_*_call(...) builds the argument block (and workspace) of one call once: the object that it returns (mvr_draft.Call)
makes the call, on the stream that is current then unless it was given one.  The functions above build one and call it.
Tensors are torch tensors on one GPU; errors are mvr_attn.MvrError.  A call on tensors without rows launches nothing.
"""
from __future__ import annotations

import ctypes

import mvr_attn as M
import mvr_draft as D
from mvr_draft import _check, _host_table, _lengths, _pools, _raw_current_stream, _refuse, _rows_read, _same_device, \
    _scope, _table

EXPORTED_SYMBOLS = (
    "mvr_paged_attention_scored",
    "mvr_paged_attention_scored_workspace_size",
    "mvr_paged_attention_scored_validate",
    "mvr_attention_weights",
    "mvr_attention_weights_validate",
    "mvr_select_tokens",
    "mvr_select_tokens_validate",
    "mvr_move_tokens",
    "mvr_move_tokens_validate",
)


class ScoreRules(ctypes.Structure):
    _fields_ = [
        ("cap", ctypes.c_float),
        ("window", ctypes.c_int32),
        ("slopes", ctypes.c_void_p),
        ("first_keys", ctypes.c_void_p),
        ("prefix_lens", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("lse_stride_head", ctypes.c_int64),
    ]


class KeyWeights(ctypes.Structure):
    _fields_ = [
        ("weights", ctypes.c_void_p),
        ("decay", ctypes.c_float),
        ("fresh_from", ctypes.c_void_p),
    ]


class SelectTokensArgs(ctypes.Structure):
    _fields_ = [
        ("num_layers", ctypes.c_int32),
        ("num_seqs", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int64),
        ("max_pages_per_seq", ctypes.c_int32),
        ("max_seq_len", ctypes.c_int32),
        ("max_moves", ctypes.c_int32),
        ("recent", ctypes.c_int32),
        ("first", ctypes.c_int32),
        ("weights", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("next_positions", ctypes.c_void_p),
        ("kept_lens", ctypes.c_void_p),
        ("keep_lens", ctypes.c_void_p),
        ("moves", ctypes.c_void_p),
        ("num_moves", ctypes.c_void_p),
        ("new_seq_lens", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class MoveTokensArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("num_layers", ctypes.c_int32),
        ("num_seqs", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int64),
        ("max_pages_per_seq", ctypes.c_int32),
        ("max_moves", ctypes.c_int32),
        ("key_pool", ctypes.c_void_p),
        ("value_pool", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("moves", ctypes.c_void_p),
        ("num_moves", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


STRUCTS = {  # C typedef -> ctypes mirror
    "mvr_score_rules": ScoreRules,
    "mvr_key_weights": KeyWeights,
    "mvr_select_tokens_args": SelectTokensArgs,
    "mvr_move_tokens_args": MoveTokensArgs,
}

_typed = False


def load_library():
    """libmvr_attn.so with the prototypes of this header too; raises if it was not built."""
    global _typed
    lib = D.load_library()
    if not _typed:
        ptr, table = ctypes.POINTER, ctypes.c_void_p
        attn, rules, weights = ptr(M.PagedAttentionArgs), ptr(ScoreRules), ptr(KeyWeights)
        select, move = ptr(SelectTokensArgs), ptr(MoveTokensArgs)
        for name, args in (("mvr_paged_attention_scored", [attn, rules]),
                           ("mvr_paged_attention_scored_workspace_size", [attn, rules]),
                           ("mvr_paged_attention_scored_validate", [attn, rules] + [table] * 6),
                           ("mvr_attention_weights", [attn, rules, weights]),
                           ("mvr_attention_weights_validate", [attn, rules, weights] + [table] * 7),
                           ("mvr_select_tokens", [select]),
                           ("mvr_select_tokens_validate", [select] + [table] * 5),
                           ("mvr_move_tokens", [move]),
                           ("mvr_move_tokens_validate", [move] + [table] * 3)):
            f = getattr(lib, name)
            f.argtypes = args
            f.restype = ctypes.c_size_t if name.endswith("workspace_size") else ctypes.c_int
        _typed = True
    return lib


def _need(**tensors):
    """Tensors that a call cannot do without."""
    for name, t in tensors.items():
        if t is None:
            _refuse(f"{name} is missing")


def _floats(t, shape, name):
    """A contiguous float32 device tensor of the given shape."""
    if t is None:
        return None
    if str(t.dtype) != "torch.float32" or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        _refuse(f"{name} must be a contiguous float32 tensor of shape {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _score_rules(q, num_seqs, lse, cap, slopes, window, first_keys, prefix_lens):
    r = ScoreRules()
    r.cap, r.window = cap, window
    r.slopes = _floats(slopes, (q.shape[0],), "slopes")
    r.first_keys = _table(first_keys, (q.shape[1],), "first_keys")
    r.prefix_lens = _table(prefix_lens, (num_seqs,), "prefix_lens")
    if lse is not None:
        if str(lse.dtype) != "torch.float32" or tuple(lse.shape) != tuple(q.shape[:2]) or \
                (lse.shape[1] > 1 and lse.stride(1) != 1):
            _refuse(f"lse must be a float32 tensor of shape {tuple(q.shape[:2])} with unit last stride, not {lse.dtype} "
                    f"{tuple(lse.shape)}")
        r.lse, r.lse_stride_head = lse.data_ptr(), lse.stride(0) if lse.shape[0] > 1 else max(1, lse.shape[1])
    return r


def _padded(a, max_q_len):
    """Rows behind the last request (a padded batch): the token count bounds nothing."""
    if a.total_q > a.num_seqs * max_q_len:
        a.total_q = 0
    return a


def make_scored_call(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out, lse=None, *, max_q_len: int,
                     max_seq_len: int, scale: float = 0.0, cap: float = 0.0, slopes=None, window: int = 0,
                     first_keys=None, prefix_lens=None, workspace=None, stream=None, sum_seq_lens: int = 0,
                     seq_lens_host=None, cu_q_lens_host=None) -> D.Call:
    """q / out [Hq, tokens, D] (unit last stride); pools [num_pages, 1, Hkv, page_size, D]; block_tables int32
    [num_seqs, max_pages]; seq_lens [num_seqs] and cu_q_lens [num_seqs + 1] int32; lse float32 [Hq, tokens], written, or
    None; cap: 0 for none; slopes float32 [Hq] or None; window: keys a query sees at most, 0 for all; first_keys int32
    [tokens] or None: where the token's document starts; prefix_lens int32 [num_seqs] or None: leading keys that all of a
    request's queries see.
    workspace: bytes of device memory to use (allocated where none is given; with too few the keys are split less)."""
    _need(q=q, key_pool=key_pool, value_pool=value_pool, block_tables=block_tables, out=out)
    _pools(key_pool, value_pool)
    if out.shape != q.shape or not q.dtype == out.dtype == key_pool.dtype:
        _refuse("q, out and the pools must have one dtype, q and out one shape")
    if key_pool.shape[4] != q.shape[2]:
        _refuse(f"q has head_dim {q.shape[2]}, the pools {key_pool.shape[4]}")
    _lengths(block_tables, seq_lens, cu_q_lens)
    r = _score_rules(q, block_tables.shape[0], lse, cap, slopes, window, first_keys, prefix_lens)
    tensors = (q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out, lse, slopes, first_keys, prefix_lens)
    device = _same_device(*tensors, workspace)
    lib = load_library()
    with _scope(device, stream):
        a = _padded(M.make_args(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out, max_q_len=max_q_len,
                                max_seq_len=max_seq_len, scale=scale, stream=stream, sum_seq_lens=sum_seq_lens,
                                seq_lens_host=seq_lens_host, cu_q_lens_host=cu_q_lens_host), max_q_len)
        need = int(lib.mvr_paged_attention_scored_workspace_size(ctypes.byref(a), ctypes.byref(r)))
        made_on = None
        if need and workspace is None:
            workspace, made_on = M.new_workspace(need, device), _raw_current_stream(device.index)
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return D.Call("mvr_paged_attention_scored", a, r, tensors, device, stream, workspace=workspace,
                  workspace_stream=made_on, empty=q.shape[1] == 0)


def paged_attention_scored(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out=None, lse=None, *,
                           max_q_len: int, max_seq_len: int, scale: float = 0.0, cap: float = 0.0, slopes=None,
                           window: int = 0, first_keys=None, prefix_lens=None, workspace=None, stream=None,
                           sum_seq_lens: int = 0, seq_lens_host=None, cu_q_lens_host=None):
    """Attention with bent and masked scores; returns out [Hq, tokens, D] in q's dtype and lse [Hq, tokens].  (Rows behind
    the last request are left as they are: uninitialised in tensors made here.)"""
    _need(q=q)
    torch = M._torch()
    with _scope(_same_device(q), stream):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if lse is None:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    make_scored_call(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out, lse, max_q_len=max_q_len,
                     max_seq_len=max_seq_len, scale=scale, cap=cap, slopes=slopes, window=window, first_keys=first_keys,
                     prefix_lens=prefix_lens, workspace=workspace, stream=stream, sum_seq_lens=sum_seq_lens,
                     seq_lens_host=seq_lens_host, cu_q_lens_host=cu_q_lens_host)()
    return out, lse


def _token_pool(t, dtype, pages, hkv, page_size, name):
    """A pool of one number per page, KV head and token."""
    if t is not None and (str(t.dtype) != dtype or not t.is_contiguous() or tuple(t.shape) != (pages, hkv, page_size)):
        _refuse(f"{name} must be a contiguous {dtype} tensor of shape {(pages, hkv, page_size)}, not {t.dtype} "
                f"{tuple(t.shape)}")
    return t.data_ptr() if t is not None else None


def make_weights_call(q, lse, key_pool, weights, block_tables, seq_lens, cu_q_lens, fresh_from=None, *, max_q_len: int,
                      max_seq_len: int, decay: float = 1.0, scale: float = 0.0, cap: float = 0.0, slopes=None,
                      window: int = 0, first_keys=None, prefix_lens=None, stream=None, seq_lens_host=None,
                      cu_q_lens_host=None) -> D.Call:
    """The rows of an attention call (or its last tokens': q, lse, cu_q_lens and first_keys of those), its lse and its
    rules; weights float32 [num_pages, Hkv, page_size], updated; fresh_from int32 [num_seqs]: slots from here on had no
    weight yet, or None: the query tokens'."""
    _need(q=q, lse=lse, key_pool=key_pool, weights=weights, block_tables=block_tables)
    pages, _, hkv, page_size, d = _pools(key_pool, key_pool)
    if q.dtype != key_pool.dtype or q.dim() != 3 or d != q.shape[2]:
        _refuse("q must be [num_q_heads, tokens, head_dim] in the pool's dtype")
    _lengths(block_tables, seq_lens, cu_q_lens)
    r = _score_rules(q, block_tables.shape[0], lse, cap, slopes, window, first_keys, prefix_lens)
    w = KeyWeights(_token_pool(weights, "torch.float32", pages, hkv, page_size, "weights"), decay,
                   _table(fresh_from, (block_tables.shape[0],), "fresh_from"))
    tensors = (q, lse, key_pool, weights, block_tables, seq_lens, cu_q_lens, fresh_from, slopes, first_keys, prefix_lens)
    device = _same_device(*tensors)
    load_library()
    with _scope(device, stream):
        a = _padded(M.make_args(q, key_pool, key_pool, block_tables, seq_lens, cu_q_lens, q, max_q_len=max_q_len,
                                max_seq_len=max_seq_len, scale=scale, stream=stream, seq_lens_host=seq_lens_host,
                                cu_q_lens_host=cu_q_lens_host), max_q_len)
    return D.Call("mvr_attention_weights", a, (r, w), tensors, device, stream, empty=q.shape[1] == 0)


def attention_weights(q, lse, key_pool, weights, block_tables, seq_lens, cu_q_lens, fresh_from=None, *, max_q_len: int,
                      max_seq_len: int, decay: float = 1.0, scale: float = 0.0, cap: float = 0.0, slopes=None,
                      window: int = 0, first_keys=None, prefix_lens=None, stream=None, seq_lens_host=None,
                      cu_q_lens_host=None):
    """Adds what each key got from these rows to its weight; returns weights."""
    make_weights_call(q, lse, key_pool, weights, block_tables, seq_lens, cu_q_lens, fresh_from, max_q_len=max_q_len,
                      max_seq_len=max_seq_len, decay=decay, scale=scale, cap=cap, slopes=slopes, window=window,
                      first_keys=first_keys, prefix_lens=prefix_lens, stream=stream, seq_lens_host=seq_lens_host,
                      cu_q_lens_host=cu_q_lens_host)()
    return weights


def _layer_tables(block_tables):
    """[layers, num_seqs, max_pages]; [num_seqs, max_pages] is one layer."""
    tables = block_tables if block_tables.dim() == 3 else block_tables.unsqueeze(0)
    _table(tables, (None, None, None), "block_tables")
    return tables


def _moves(moves, num_moves, rows):
    return _table(moves, (*rows, None, 2), "moves"), _table(num_moves, rows, "num_moves")


def make_select_call(weights, positions, block_tables, seq_lens, next_positions, kept_lens, keep_lens, moves, num_moves,
                     new_seq_lens=None, *, recent: int, max_seq_len: int, first: int = 0, stream=None) -> D.Call:
    """weights float32 and positions int32 [num_pages, Hkv, page_size]; block_tables int32 [layers, num_seqs, max_pages],
    or [num_seqs, max_pages] for one layer; seq_lens, next_positions (None: seq_lens), kept_lens (None: 0), keep_lens
    int32 [num_seqs]; written: moves int32 [layers, num_seqs, Hkv, most, 2], num_moves [layers, num_seqs, Hkv],
    new_seq_lens [num_seqs] or None."""
    _need(weights=weights, positions=positions, block_tables=block_tables, seq_lens=seq_lens, keep_lens=keep_lens,
          moves=moves, num_moves=num_moves)
    if weights.dim() != 3:
        _refuse("weights must be [num_pages, num_kv_heads, page_size]")
    pages, hkv, page_size = weights.shape
    tables = _layer_tables(block_tables)
    a = SelectTokensArgs()
    a.num_layers, a.num_seqs, a.max_pages_per_seq = tables.shape
    a.num_kv_heads, a.page_size, a.num_pages = hkv, page_size, pages
    a.max_seq_len, a.recent, a.first = max_seq_len, recent, first
    a.weights = _token_pool(weights, "torch.float32", pages, hkv, page_size, "weights")
    a.positions = _token_pool(positions, "torch.int32", pages, hkv, page_size, "positions")
    a.block_tables = tables.data_ptr()
    a.moves, a.num_moves = _moves(moves, num_moves, (a.num_layers, a.num_seqs, hkv))
    a.max_moves = moves.shape[3]
    for name, t in (("seq_lens", seq_lens), ("next_positions", next_positions), ("kept_lens", kept_lens),
                    ("keep_lens", keep_lens), ("new_seq_lens", new_seq_lens)):
        setattr(a, name, _table(t, (a.num_seqs,), name))
    tensors = (weights, positions, block_tables, seq_lens, next_positions, kept_lens, keep_lens, moves, num_moves,
               new_seq_lens)
    load_library()
    return D.Call("mvr_select_tokens", a, None, tensors, _same_device(*tensors), stream)


def select_tokens(weights, positions, block_tables, seq_lens, next_positions, kept_lens, keep_lens, *, recent: int,
                  max_seq_len: int, max_moves: int, first: int = 0, stream=None):
    """Which tokens stay: returns moves [layers, num_seqs, Hkv, max_moves, 2] (behind num_moves: uninitialised),
    num_moves [layers, num_seqs, Hkv] and the new lengths [num_seqs]."""
    _need(weights=weights, block_tables=block_tables, seq_lens=seq_lens)
    if weights.dim() != 3 or max_moves < 1:
        _refuse("weights must be [num_pages, num_kv_heads, page_size], and max_moves positive")
    torch, tables = M._torch(), _layer_tables(block_tables)
    with _scope(_same_device(weights), stream):
        rows = (tables.shape[0], tables.shape[1], weights.shape[1])
        moves = torch.empty(rows + (max_moves, 2), dtype=torch.int32, device=weights.device)
        num_moves = torch.empty(rows, dtype=torch.int32, device=weights.device)
        new_seq_lens = torch.empty_like(seq_lens)
    make_select_call(weights, positions, block_tables, seq_lens, next_positions, kept_lens, keep_lens, moves, num_moves,
                     new_seq_lens, recent=recent, first=first, max_seq_len=max_seq_len, stream=stream)()
    return moves, num_moves, new_seq_lens


def make_move_call(key_pool, value_pool, weights, positions, block_tables, moves, num_moves, *, stream=None) -> D.Call:
    """Pools [num_pages, 1, Hkv, page_size, D]; weights float32, positions int32 [num_pages, Hkv, page_size] or None;
    block_tables, moves and num_moves as for make_select_call."""
    _need(key_pool=key_pool, value_pool=value_pool, block_tables=block_tables, moves=moves, num_moves=num_moves)
    pages, _, hkv, page_size, d = _pools(key_pool, value_pool)
    tables = _layer_tables(block_tables)
    a = MoveTokensArgs()
    a.dtype = M.dtype_code(key_pool)
    a.num_layers, a.num_seqs, a.max_pages_per_seq = tables.shape
    a.num_kv_heads, a.head_dim, a.page_size, a.num_pages = hkv, d, page_size, pages
    a.key_pool, a.value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    a.weights = _token_pool(weights, "torch.float32", pages, hkv, page_size, "weights")
    a.positions = _token_pool(positions, "torch.int32", pages, hkv, page_size, "positions")
    a.block_tables = tables.data_ptr()
    a.moves, a.num_moves = _moves(moves, num_moves, (a.num_layers, a.num_seqs, hkv))
    a.max_moves = moves.shape[3]
    tensors = (key_pool, value_pool, weights, positions, block_tables, moves, num_moves)
    load_library()
    return D.Call("mvr_move_tokens", a, None, tensors, _same_device(*tensors), stream)


def move_tokens(key_pool, value_pool, weights, positions, block_tables, moves, num_moves, *, stream=None) -> None:
    """Copies the K and V rows, weights and positions of each KV head from slot to slot."""
    make_move_call(key_pool, value_pool, weights, positions, block_tables, moves, num_moves, stream=stream)()


def _rule_tables(keep, a, cu_q_lens_host, first_keys_host, prefix_lens_host, slopes_host):
    return (_host_table(keep, first_keys_host, "first_keys_host", _rows_read(a, cu_q_lens_host, a.max_q_len)),
            _host_table(keep, prefix_lens_host, "prefix_lens_host", a.num_seqs),
            _host_table(keep, slopes_host, "slopes_host", a.num_q_heads, "float32"))


def _length_tables(keep, a, block_tables_host, seq_lens_host, cu_q_lens_host):
    return (_host_table(keep, block_tables_host, "block_tables_host", a.num_seqs * a.max_pages_per_seq),
            _host_table(keep, seq_lens_host, "seq_lens_host", a.num_seqs),
            _host_table(keep, cu_q_lens_host, "cu_q_lens_host", a.num_seqs + 1))


def validate_scored(args: M.PagedAttentionArgs, rules: ScoreRules, block_tables_host=None, seq_lens_host=None,
                    cu_q_lens_host=None, first_keys_host=None, prefix_lens_host=None, slopes_host=None) -> None:
    """Host-side checks of an attention call's tables (numpy arrays or None); raises MvrError."""
    keep = []
    tables = _length_tables(keep, args, block_tables_host, seq_lens_host, cu_q_lens_host) + \
        _rule_tables(keep, args, cu_q_lens_host, first_keys_host, prefix_lens_host, slopes_host)
    _check(load_library().mvr_paged_attention_scored_validate(ctypes.byref(args), ctypes.byref(rules), *tables))


def validate_weights(args: M.PagedAttentionArgs, rules: ScoreRules, weights: KeyWeights, block_tables_host=None,
                     seq_lens_host=None, cu_q_lens_host=None, first_keys_host=None, prefix_lens_host=None,
                     slopes_host=None, fresh_from_host=None) -> None:
    """Host-side checks of a weights call's tables (numpy arrays or None); raises MvrError."""
    keep = []
    tables = _length_tables(keep, args, block_tables_host, seq_lens_host, cu_q_lens_host) + \
        _rule_tables(keep, args, cu_q_lens_host, first_keys_host, prefix_lens_host, slopes_host) + \
        (_host_table(keep, fresh_from_host, "fresh_from_host", args.num_seqs),)
    _check(load_library().mvr_attention_weights_validate(ctypes.byref(args), ctypes.byref(rules), ctypes.byref(weights),
                                                         *tables))


def validate_select(args: SelectTokensArgs, block_tables_host=None, seq_lens_host=None, next_positions_host=None,
                    kept_lens_host=None, keep_lens_host=None) -> None:
    """Host-side checks of a selection's tables (numpy arrays or None); raises MvrError."""
    keep, n = [], args.num_seqs
    tables = (_host_table(keep, block_tables_host, "block_tables_host", args.num_layers * n * args.max_pages_per_seq),
              _host_table(keep, seq_lens_host, "seq_lens_host", n),
              _host_table(keep, next_positions_host, "next_positions_host", n),
              _host_table(keep, kept_lens_host, "kept_lens_host", n), _host_table(keep, keep_lens_host, "keep_lens_host", n))
    _check(load_library().mvr_select_tokens_validate(ctypes.byref(args), *tables))


def validate_move(args: MoveTokensArgs, block_tables_host=None, moves_host=None, num_moves_host=None) -> None:
    """Host-side checks of a list of moves (numpy arrays or None); raises MvrError."""
    keep, rows = [], args.num_layers * args.num_seqs
    tables = (_host_table(keep, block_tables_host, "block_tables_host", rows * args.max_pages_per_seq),
              _host_table(keep, moves_host, "moves_host", rows * args.num_kv_heads * args.max_moves * 2),
              _host_table(keep, num_moves_host, "num_moves_host", rows * args.num_kv_heads))
    _check(load_library().mvr_move_tokens_validate(ctypes.byref(args), *tables))
