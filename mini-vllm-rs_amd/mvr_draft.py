"""Python binding of the drafted-tree calls of libmvr_attn.so (C ABI in include/mvr_draft.h).

One step of speculative decoding with a tree of drafts, per layer and over all requests of a batch:
  * norm_rope_append(...)      norms of the new Q and K rows per head, rotation at a position of each token's own,
                               append to the pages (beside mvr_attn.rope_append);
  * paged_attention_tree(...)  each draft attends the cache and the drafts that its mask names (beside
                               mvr_attn.paged_attention);
and per step, over the block tables of all layers:
  * compact_drafts(...)        the accepted drafts' rows move to the front of the drafts' slots;
  * copy_pages(...)            copies of pages, for forked requests.

make_*_call(...) builds the argument block (and workspace) of one call once: the object that it returns makes the call,
on the stream that is current then unless it was given one, as a runner repeats it step by step or records it into a
graph.  The functions above build one and call it.  Tensors are torch tensors on one GPU; errors are mvr_attn.MvrError.
A call on tensors without rows (no request has a draft this step) launches nothing.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional

import mvr_attn as M
from mvr_attn import MVR_E_INVALID_ARGUMENT, ROPE_INTERLEAVED, ROPE_NEOX, MvrError  # noqa: F401

EXPORTED_SYMBOLS = (
    "mvr_paged_attention_tree",
    "mvr_paged_attention_tree_workspace_size",
    "mvr_paged_attention_tree_validate",
    "mvr_norm_rope_append",
    "mvr_norm_rope_append_validate",
    "mvr_compact_drafts",
    "mvr_compact_drafts_validate",
    "mvr_copy_pages",
    "mvr_copy_pages_validate",
)


class DraftTrees(ctypes.Structure):
    _fields_ = [
        ("masks", ctypes.c_void_p),
        ("mask_words", ctypes.c_int32),
    ]


class HeadNorms(ctypes.Structure):
    _fields_ = [
        ("q_weight", ctypes.c_void_p),
        ("k_weight", ctypes.c_void_p),
        ("eps", ctypes.c_float),
        ("positions", ctypes.c_void_p),
    ]


class CompactDraftsArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("num_layers", ctypes.c_int32),
        ("num_seqs", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int64),
        ("max_pages_per_seq", ctypes.c_int32),
        ("max_seq_len", ctypes.c_int32),
        ("max_accepted", ctypes.c_int32),
        ("key_pool", ctypes.c_void_p),
        ("value_pool", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("cu_q_lens", ctypes.c_void_p),
        ("accepted", ctypes.c_void_p),
        ("accepted_lens", ctypes.c_void_p),
        ("new_seq_lens", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class CopyPagesArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int32),
        ("num_copies", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int64),
        ("key_pool", ctypes.c_void_p),
        ("value_pool", ctypes.c_void_p),
        ("src_pages", ctypes.c_void_p),
        ("dst_pages", ctypes.c_void_p),
        ("tokens", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


STRUCTS = {  # C typedef -> ctypes mirror
    "mvr_draft_trees": DraftTrees,
    "mvr_head_norms": HeadNorms,
    "mvr_compact_drafts_args": CompactDraftsArgs,
    "mvr_copy_pages_args": CopyPagesArgs,
}

_typed = False


def load_library():
    """libmvr_attn.so with the prototypes of this header too; raises if it was not built."""
    global _typed
    lib = M.load_library()
    if not _typed:
        ptr, table = ctypes.POINTER, ctypes.c_void_p
        attn, trees = ptr(M.PagedAttentionArgs), ptr(DraftTrees)
        rope, norms = ptr(M.RopeAppendArgs), ptr(HeadNorms)
        compact, copy = ptr(CompactDraftsArgs), ptr(CopyPagesArgs)
        for name, args in (("mvr_paged_attention_tree", [attn, trees]),
                           ("mvr_paged_attention_tree_workspace_size", [attn, trees]),
                           ("mvr_paged_attention_tree_validate", [attn, trees] + [table] * 4),
                           ("mvr_norm_rope_append", [rope, norms]),
                           ("mvr_norm_rope_append_validate", [rope, norms] + [table] * 5),
                           ("mvr_compact_drafts", [compact]),
                           ("mvr_compact_drafts_validate", [compact] + [table] * 5),
                           ("mvr_copy_pages", [copy]),
                           ("mvr_copy_pages_validate", [copy] + [table] * 3)):
            f = getattr(lib, name)
            f.argtypes = args
            f.restype = ctypes.c_size_t if name.endswith("workspace_size") else ctypes.c_int
        _typed = True
    return lib


def _check(rc: int) -> None:
    if rc != 0:
        raise MvrError(rc, load_library().mvr_last_error().decode())


def _refuse(message: str):
    raise MvrError(MVR_E_INVALID_ARGUMENT, message)


def _same_device(*tensors):
    """The one GPU of all tensors."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        _refuse(f"tensors on different devices: {sorted(map(str, devices))}")
    device = devices.pop()
    if device.type != "cuda":
        _refuse(f"tensors must be on a GPU, not on {device}")
    return device


def _table(t, shape, name):
    """A contiguous int32 device table of at least the given shape (None entries: any)."""
    if t is None:
        return None
    if str(t.dtype) not in ("torch.int32", "torch.uint32") or not t.is_contiguous() or t.dim() != len(shape) or \
            any(want is not None and have != want for have, want in zip(t.shape, shape)):
        _refuse(f"{name} must be a contiguous int32 tensor of shape {tuple('*' if x is None else x for x in shape)}, "
                f"not {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _lengths(block_tables, seq_lens, cu_q_lens):
    _table(block_tables, (None, None), "block_tables")
    _table(seq_lens, (block_tables.shape[0],), "seq_lens")
    _table(cu_q_lens, (block_tables.shape[0] + 1,), "cu_q_lens")


def _pools(key_pool, value_pool):
    if key_pool.dim() != 5 or key_pool.shape[1] != 1 or value_pool.shape != key_pool.shape:
        _refuse("pools must be [num_pages, 1, num_kv_heads, page_size, head_dim]")
    if not key_pool.is_contiguous() or not value_pool.is_contiguous():
        _refuse("pools must be contiguous")
    if key_pool.dtype != value_pool.dtype:
        _refuse("pools of different dtypes")
    return key_pool.shape


class Call:
    """One call of the library, its argument block (`args`, and `extra` where the entry point takes a second one, or a
    tuple of more) made and its tensors kept.  Calling it launches on `stream`, or on the stream that is current then.
    One thread at a time may call it (another makes a Call of its own), and where there is a `workspace`, its launches must
    not overlap in time, nor may those of Calls that share one.  A graph that recorded a launch reads the argument block's
    tensors and writes the workspace at every replay: keep the Call as long as the graph.
    workspace_stream: handle of the stream whose memory the workspace is, where this module made it; None: the caller's.
    empty: its tensors have no rows, there is nothing to launch."""

    def __init__(self, name, args, extra, tensors, device, stream, workspace=None, workspace_stream=None, empty=False):
        self._function = getattr(load_library(), name)
        self.args, self.extra, self.workspace = args, extra, workspace
        extras = extra if isinstance(extra, tuple) else () if extra is None else (extra,)
        self._refs = tuple(ctypes.byref(block) for block in (args, *extras))
        self._tensors = tuple(t for t in tensors if t is not None)
        if workspace is not None and workspace_stream is None:
            self._tensors += (workspace,)
        self._device, self._stream, self._empty = device, stream, empty
        # Streams that the workspace made here is known to be used on (the allocator's record lasts until it is freed).
        self._known = None if workspace_stream is None else {workspace_stream}
        self._cuda = M._torch().cuda
        if stream is not None and stream.device != device:
            _refuse(f"a stream of {stream.device} for tensors of {device}")

    def __call__(self):
        if self._empty:
            return
        cuda, index = self._cuda, self._device.index
        if cuda.current_device() != index:
            with cuda.device(self._device):
                return self()
        current = _raw_current_stream(index)
        launch = current if self._stream is None else self._stream.cuda_stream
        self.args.stream = launch
        # Memory that is freed while kernels of another stream than its own still use it must not be handed out meanwhile.
        if launch != current:
            for t in self._tensors:
                t.record_stream(self._stream)
        if self._known is not None and launch not in self._known:
            self.workspace.record_stream(self._stream or cuda.current_stream(index))
            self._known.add(launch)
        _check(self._function(*self._refs))


def _raw_current_stream(index):
    """Handle of the device's current stream.  (torch.cuda.current_stream() makes a Stream object: 2.7 us against 0.1,
    where a whole small call takes 3.)"""
    global _raw_stream
    if _raw_stream is None:
        torch = M._torch()
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _raw_stream(index)


_raw_stream = None


def _scope(device, stream):
    """Allocations of a call, made where it runs."""
    torch = M._torch()
    stack = contextlib.ExitStack()
    stack.enter_context(torch.cuda.device(device))
    if stream is not None:
        stack.enter_context(torch.cuda.stream(stream))
    return stack


def make_tree_call(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, masks, out, *, max_q_len: int,
                   max_seq_len: int, scale: float = 0.0, workspace=None, stream=None, sum_seq_lens: int = 0,
                   seq_lens_host=None, cu_q_lens_host=None) -> Call:
    """q / out [Hq, tokens, D] (unit last stride); pools [num_pages, 1, Hkv, page_size, D]; block_tables int32
    [num_seqs, max_pages]; seq_lens [num_seqs] (drafts included) and cu_q_lens [num_seqs + 1] int32; masks int32 or
    uint32 [tokens, words], bit s % 32 of word s / 32 of row n: packed token n sees draft slot s of its request.
    workspace: bytes of device memory to use (allocated where none is given; with too few the keys are split less)."""
    _pools(key_pool, value_pool)
    if out.shape != q.shape or not q.dtype == out.dtype == key_pool.dtype:
        _refuse("q, out and the pools must have one dtype, q and out one shape")
    if key_pool.shape[4] != q.shape[2]:
        _refuse(f"q has head_dim {q.shape[2]}, the pools {key_pool.shape[4]}")
    _lengths(block_tables, seq_lens, cu_q_lens)
    t = DraftTrees(_table(masks, (q.shape[1], None), "masks"), masks.shape[1])
    device = _same_device(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, masks, out, workspace)
    with _scope(device, stream):
        a = M.make_args(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, out, max_q_len=max_q_len,
                        max_seq_len=max_seq_len, scale=scale, stream=stream, sum_seq_lens=sum_seq_lens,
                        seq_lens_host=seq_lens_host, cu_q_lens_host=cu_q_lens_host)
        if a.total_q > a.num_seqs * max_q_len:  # rows behind the last request (a padded batch)
            a.total_q = 0
        need = int(load_library().mvr_paged_attention_tree_workspace_size(ctypes.byref(a), ctypes.byref(t)))
        made_on = None
        if need and workspace is None:
            workspace, made_on = M.new_workspace(need, device), _raw_current_stream(device.index)
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return Call("mvr_paged_attention_tree", a, t,
                (q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, masks, out), device, stream, workspace=workspace,
                workspace_stream=made_on, empty=q.shape[1] == 0)


def paged_attention_tree(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, masks, out=None, *,
                         max_q_len: int, max_seq_len: int, scale: float = 0.0, workspace=None, stream=None,
                         sum_seq_lens: int = 0, seq_lens_host=None, cu_q_lens_host=None):
    """Attention of drafted trees; returns out [Hq, tokens, D] in q's dtype.  (Rows behind the last request are left as
    they are: uninitialised in an out made here.)"""
    if out is None:
        with _scope(q.device, stream):
            out = M._torch().empty_like(q, memory_format=M._torch().contiguous_format)
    make_tree_call(q, key_pool, value_pool, block_tables, seq_lens, cu_q_lens, masks, out, max_q_len=max_q_len,
                   max_seq_len=max_seq_len, scale=scale, workspace=workspace, stream=stream,
                   sum_seq_lens=sum_seq_lens, seq_lens_host=seq_lens_host, cu_q_lens_host=cu_q_lens_host)()
    return out


def make_norm_rope_append_call(q, k, v, q_weight, k_weight, cos_table, sin_table, block_tables, seq_lens, cu_q_lens,
                               key_pool, value_pool, q_out, *, eps: float, max_seq_len: int, positions=None,
                               rope_type: int = ROPE_NEOX, stream=None) -> Call:
    """q / q_out [Hq, tokens, D] (q_out may be q), k / v [Hkv, tokens, D] (unit last stride); q_weight / k_weight [D] or
    None (no norm); cos / sin [rope_len, D/2]; positions int32 [tokens] or None (each token's cache slot); the rest as
    for mvr_attn.rope_append."""
    _pools(key_pool, value_pool)
    hkv, d = key_pool.shape[2], key_pool.shape[4]
    for t in (q, k, v, q_out, q_weight, k_weight, cos_table, sin_table, key_pool):
        if t is not None and t.dtype != q.dtype:
            _refuse("q, k, v, q_out, the weights, the rotary tables and the pools must have one dtype")
    for t in (q_weight, k_weight):
        if t is not None and (tuple(t.shape) != (d,) or not t.is_contiguous()):
            _refuse(f"norm weights must be contiguous vectors of head_dim {d}")
    if q.dim() != 3 or q_out.shape != q.shape or tuple(k.shape) != (hkv, q.shape[1], d) or v.shape != k.shape or \
            q.shape[2] != d:
        _refuse("q and q_out must be [Hq, tokens, head_dim], k and v [Hkv, tokens, head_dim]")
    if tuple(cos_table.shape[1:]) != (d // 2,) or sin_table.shape != cos_table.shape:
        _refuse("rotary tables must be [rope_len, head_dim / 2]")
    _lengths(block_tables, seq_lens, cu_q_lens)
    n = HeadNorms(q_weight.data_ptr() if q_weight is not None else None,
                  k_weight.data_ptr() if k_weight is not None else None, eps,
                  _table(positions, (q.shape[1],), "positions"))
    device = _same_device(q, k, v, q_weight, k_weight, cos_table, sin_table, block_tables, seq_lens, cu_q_lens,
                          key_pool, value_pool, q_out, positions)
    with _scope(device, stream):
        a = M.make_rope_append_args(q, k, v, cos_table, sin_table, block_tables, seq_lens, cu_q_lens, key_pool,
                                    value_pool, q_out, max_seq_len=max_seq_len, rope_type=rope_type, stream=stream)
    return Call("mvr_norm_rope_append", a, n,
                (q, k, v, q_weight, k_weight, cos_table, sin_table, block_tables, seq_lens, cu_q_lens, key_pool,
                 value_pool, q_out, positions), device, stream, empty=q.shape[1] == 0)


def norm_rope_append(q, k, v, q_weight, k_weight, cos_table, sin_table, block_tables, seq_lens, cu_q_lens, key_pool,
                     value_pool, q_out=None, *, eps: float, max_seq_len: int, positions=None,
                     rope_type: int = ROPE_NEOX, stream=None):
    """Normalises and rotates q into q_out (a new tensor unless given; may be q itself) and k into its page slots,
    beside v; returns q_out."""
    if q_out is None:
        with _scope(q.device, stream):
            q_out = M._torch().empty_like(q, memory_format=M._torch().contiguous_format)
    make_norm_rope_append_call(q, k, v, q_weight, k_weight, cos_table, sin_table, block_tables, seq_lens, cu_q_lens,
                               key_pool, value_pool, q_out, eps=eps, max_seq_len=max_seq_len, positions=positions,
                               rope_type=rope_type, stream=stream)()
    return q_out


def make_compact_drafts_call(key_pool, value_pool, block_tables, seq_lens, cu_q_lens, accepted, accepted_lens,
                             new_seq_lens=None, *, max_seq_len: int, stream=None) -> Call:
    """block_tables int32 [layers, num_seqs, max_pages], or [num_seqs, max_pages] for one layer; accepted int32
    [num_seqs, most], ascending draft indices; accepted_lens [num_seqs]; new_seq_lens [num_seqs] or None, written."""
    n, _, hkv, page_size, d = _pools(key_pool, value_pool)
    a = CompactDraftsArgs()
    a.dtype = M.dtype_code(key_pool)
    tables = block_tables if block_tables.dim() == 3 else block_tables.unsqueeze(0)
    a.block_tables = _table(tables, (None, None, None), "block_tables")
    a.num_layers, a.num_seqs, a.max_pages_per_seq = tables.shape
    a.num_kv_heads, a.head_dim, a.page_size, a.num_pages = hkv, d, page_size, n
    a.max_seq_len = max_seq_len
    a.accepted = _table(accepted, (a.num_seqs, None), "accepted")
    a.max_accepted = accepted.shape[1]
    a.key_pool, a.value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    a.seq_lens = _table(seq_lens, (a.num_seqs,), "seq_lens")
    a.cu_q_lens = _table(cu_q_lens, (a.num_seqs + 1,), "cu_q_lens")
    a.accepted_lens = _table(accepted_lens, (a.num_seqs,), "accepted_lens")
    a.new_seq_lens = _table(new_seq_lens, (a.num_seqs,), "new_seq_lens")
    device = _same_device(key_pool, value_pool, block_tables, seq_lens, cu_q_lens, accepted, accepted_lens, new_seq_lens)
    return Call("mvr_compact_drafts", a, None, (key_pool, value_pool, block_tables, seq_lens, cu_q_lens, accepted,
                                                accepted_lens, new_seq_lens), device, stream)


def compact_drafts(key_pool, value_pool, block_tables, seq_lens, cu_q_lens, accepted, accepted_lens,
                   new_seq_lens=None, *, max_seq_len: int, stream=None):
    """Moves the accepted drafts' rows to the front of the drafts' slots in every layer; returns the new lengths (a new
    tensor unless given)."""
    if new_seq_lens is None:
        with _scope(seq_lens.device, stream):
            new_seq_lens = M._torch().empty_like(seq_lens)
    make_compact_drafts_call(key_pool, value_pool, block_tables, seq_lens, cu_q_lens, accepted, accepted_lens,
                             new_seq_lens, max_seq_len=max_seq_len, stream=stream)()
    return new_seq_lens


def make_copy_pages_call(key_pool, value_pool, src_pages, dst_pages, tokens=None, *, stream=None) -> Call:
    """src_pages, dst_pages int32 [copies]; tokens int32 [copies]: leading tokens of each page to copy (None: all)."""
    n, _, hkv, page_size, d = _pools(key_pool, value_pool)
    a = CopyPagesArgs()
    a.dtype = M.dtype_code(key_pool)
    a.num_copies = src_pages.shape[0]
    a.num_kv_heads, a.head_dim, a.page_size, a.num_pages = hkv, d, page_size, n
    a.key_pool, a.value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    a.src_pages = _table(src_pages, (None,), "src_pages")
    a.dst_pages = _table(dst_pages, (a.num_copies,), "dst_pages")
    a.tokens = _table(tokens, (a.num_copies,), "tokens")
    device = _same_device(key_pool, value_pool, src_pages, dst_pages, tokens)
    return Call("mvr_copy_pages", a, None, (key_pool, value_pool, src_pages, dst_pages, tokens), device, stream)


def copy_pages(key_pool, value_pool, src_pages, dst_pages, tokens=None, *, stream=None) -> None:
    """Copies K and V pages src_pages[i] to dst_pages[i]."""
    make_copy_pages_call(key_pool, value_pool, src_pages, dst_pages, tokens, stream=stream)()


def _host_table(keep, x, name, entries, dtype="int32"):
    """Address of a host table of at least `entries` entries, as the library reads it."""
    if x is None:
        return None
    import numpy as np

    x = np.ascontiguousarray(x, dtype=dtype)
    if x.size < entries:
        _refuse(f"{name} must hold {entries} entries, not {x.size}")
    keep.append(x)
    return x.ctypes.data


def _rows_read(args, cu_q_lens_host, alone):
    """Rows of a per-token table that a check reads: the requests' tokens; `alone` of one request without cu_q_lens."""
    if cu_q_lens_host is None:
        return alone if args.num_seqs == 1 else 0
    rows = max((int(x) for x in cu_q_lens_host), default=0)  # (starts that do not ascend are refused before any row is read)
    return min(rows, args.total_q) if args.total_q > 0 else rows


def validate_tree(args: M.PagedAttentionArgs, trees: DraftTrees, block_tables_host=None, seq_lens_host=None,
                  cu_q_lens_host=None, masks_host=None) -> None:
    """Host-side checks of a tree call's tables (numpy arrays or None); raises MvrError."""
    keep, n = [], args.num_seqs
    tables = (_host_table(keep, block_tables_host, "block_tables_host", n * args.max_pages_per_seq),
              _host_table(keep, seq_lens_host, "seq_lens_host", n),
              _host_table(keep, cu_q_lens_host, "cu_q_lens_host", n + 1))
    if masks_host is not None:
        if masks_host.dtype.itemsize != 4:
            _refuse(f"masks_host must hold 32-bit words, not {masks_host.dtype}")
        masks_host = masks_host.view("uint32")
    masks = _host_table(keep, masks_host, "masks_host",
                        _rows_read(args, cu_q_lens_host, args.max_q_len) * trees.mask_words, "uint32")
    _check(load_library().mvr_paged_attention_tree_validate(ctypes.byref(args), ctypes.byref(trees), *tables, masks))


def validate_norm_rope_append(args: M.RopeAppendArgs, norms: HeadNorms, block_tables_host=None, seq_lens_host=None,
                              cu_q_lens_host=None, positions_host=None, page_writable_host=None) -> None:
    """Host-side checks of an append's tables (numpy arrays or None); raises MvrError."""
    keep, n = [], args.num_seqs
    tables = (_host_table(keep, block_tables_host, "block_tables_host", n * args.max_pages_per_seq),
              _host_table(keep, seq_lens_host, "seq_lens_host", n),
              _host_table(keep, cu_q_lens_host, "cu_q_lens_host", n + 1),
              _host_table(keep, positions_host, "positions_host", _rows_read(args, cu_q_lens_host, args.total_q)),
              _host_table(keep, page_writable_host, "page_writable_host", args.num_pages, "uint8"))
    _check(load_library().mvr_norm_rope_append_validate(ctypes.byref(args), ctypes.byref(norms), *tables))


def validate_compact_drafts(args: CompactDraftsArgs, block_tables_host=None, seq_lens_host=None, cu_q_lens_host=None,
                            accepted_host=None, accepted_lens_host=None) -> None:
    """Host-side checks of a compaction's tables (numpy arrays or None); raises MvrError."""
    keep, n = [], args.num_seqs
    tables = (_host_table(keep, block_tables_host, "block_tables_host", args.num_layers * n * args.max_pages_per_seq),
              _host_table(keep, seq_lens_host, "seq_lens_host", n),
              _host_table(keep, cu_q_lens_host, "cu_q_lens_host", n + 1),
              _host_table(keep, accepted_host, "accepted_host", n * args.max_accepted),
              _host_table(keep, accepted_lens_host, "accepted_lens_host", n))
    _check(load_library().mvr_compact_drafts_validate(ctypes.byref(args), *tables))


def validate_copy_pages(args: CopyPagesArgs, src_pages_host=None, dst_pages_host=None, tokens_host=None) -> None:
    """Host-side checks of a copy's lists (numpy arrays or None); raises MvrError."""
    keep, n = [], args.num_copies
    _check(load_library().mvr_copy_pages_validate(ctypes.byref(args), _host_table(keep, src_pages_host, "src_pages_host", n),
                                                  _host_table(keep, dst_pages_host, "dst_pages_host", n),
                                                  _host_table(keep, tokens_host, "tokens_host", n)))


def tree_masks(parents, cu_q_lens, mask_words: Optional[int] = None):
    """Mask rows (numpy int32 [tokens, words]) of trees: parents[n] is the index, within its request, of packed token
    n's parent (-1: a root), which comes before it; a token sees itself and its ancestors."""
    import numpy as np

    parents, cu = np.asarray(parents), np.asarray(cu_q_lens)
    longest = int((cu[1:] - cu[:-1]).max(initial=0))
    words = mask_words or max(1, math.ceil(longest / 32))
    if words * 32 < longest:
        _refuse(f"mask rows of {words} words cannot hold {longest} drafts")
    masks = np.zeros((len(parents), words), np.uint32)
    for lo, hi in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for i in range(hi - lo):
            p = int(parents[lo + i])
            if not -1 <= p < i:
                _refuse(f"token {lo + i}: parent {p} does not come before it")
            if p >= 0:
                masks[lo + i] = masks[lo + p]
            masks[lo + i, i // 32] |= np.uint32(1 << (i % 32))
    return masks.view(np.int32)
