"""CPU-side checks of the drafted-tree calls: the library exports what include/mvr_draft.h declares, the bindings agree
with it, the host checks refuse bad arguments and tables before any launch."""
import ctypes
import os
import re
import subprocess
import tempfile

import numpy as np
import pytest

import mvr_attn as M
import mvr_draft as D
import test_rust_binding as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mvr_draft.h")
RUST = os.path.join(ROOT, "mini-vllm-rs_amd", "rust", "mvr_draft.rs")
FAKE = 1 << 20  # an aligned address: these calls never launch


# ---- header and bindings ---------------------------------------------------

@pytest.fixture()
def draft_header(monkeypatch):
    """The parsers of the other header's test on this one."""
    monkeypatch.setattr(R, "HEADER", HEADER)
    monkeypatch.setattr(R, "RUST", RUST)


RUST_NAMES = {"mvr_draft_trees": "MvrDraftTrees", "mvr_head_norms": "MvrHeadNorms",
              "mvr_compact_drafts_args": "MvrCompactDraftsArgs", "mvr_copy_pages_args": "MvrCopyPagesArgs",
              "mvr_paged_attention_args": "MvrPagedAttentionArgs", "mvr_rope_append_args": "MvrRopeAppendArgs"}
TYPES = {**R.C_TO_RUST, "const uint32_t*": "*const u32", "int32_t*": "*mut i32"}


def test_library_exports_every_declared_symbol(draft_header):
    declared = set(R.c_functions())
    assert declared == set(D.EXPORTED_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", M.library_path()], capture_output=True, text=True, check=True)
    assert declared <= set(re.findall(r"\bT (mvr_[a-z0-9_]+)$", out.stdout, flags=re.M))
    lib = D.load_library()
    assert all(getattr(lib, name).argtypes for name in declared)


def test_rust_source_matches_the_header(draft_header):
    structs, rust = R.c_structs(), R.rust_structs()
    assert set(structs) == set(D.STRUCTS)
    for name, fields in structs.items():
        assert [(n, TYPES[t]) for n, t in fields] == rust[RUST_NAMES[name]], name
    functions, rust = R.c_functions(), R.rust_functions()
    assert set(rust) == set(functions)
    for name, (ret, args) in functions.items():
        want = [TYPES.get(t) or "*const " + RUST_NAMES[t[len("const "):-1]] for t in args]
        assert (TYPES[ret], want) == rust[name], name


@pytest.mark.skipif(subprocess.run(["which", "gcc"], capture_output=True).returncode != 0, reason="no gcc")
def test_ctypes_mirror_has_the_c_layout(draft_header):
    structs = R.c_structs()
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "mvr_draft.h"', "int main(void) {"]
    for name, fields in structs.items():
        lines.append(f'  printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {n} %zu\\n", offsetof({name}, {n}));' for n, _ in fields]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        open(src, "w").write("\n".join(lines + ["  return 0;\n}"]))
        subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), src, "-o", exe],
                       check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out if line}
    for name, mirror in D.STRUCTS.items():
        assert [n for n, _ in mirror._fields_] == [n for n, _ in structs[name]]
        assert ctypes.sizeof(mirror) == got[(name, "sizeof")]
        for n, _ in mirror._fields_:
            assert getattr(mirror, n).offset == got[(name, n)], (name, n)


# ---- tree attention --------------------------------------------------------

def tree_args(**kw):
    a = M.PagedAttentionArgs()
    a.dtype, a.num_seqs, a.num_q_heads, a.num_kv_heads, a.head_dim, a.page_size = M.DTYPE_F16, 2, 32, 8, 128, 16
    a.num_pages, a.max_pages_per_seq, a.max_q_len, a.max_seq_len = 1024, 64, 40, 1024
    a.q = a.key_pool = a.value_pool = a.block_tables = a.seq_lens = a.cu_q_lens = a.out = FAKE
    a.q_stride_head = a.out_stride_head = 80 * 128
    a.q_stride_token = a.out_stride_token = 128
    t = D.DraftTrees(FAKE, 2)
    for k, v in kw.items():
        setattr(t if hasattr(t, k) else a, k, v)
    return a, t


def status(name, *args):
    lib = D.load_library()
    refs = [ctypes.byref(x) if isinstance(x, ctypes.Structure) else x for x in args]
    return getattr(lib, name)(*refs), lib.mvr_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(num_kv_heads=5), M.MVR_E_INVALID_ARGUMENT, "multiple of num_kv_heads"),
    (dict(head_dim=100), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=288), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(page_size=0), M.MVR_E_INVALID_ARGUMENT, "page_size"),
    (dict(num_pages=0), M.MVR_E_INVALID_ARGUMENT, "num_pages"),
    (dict(num_pages=1 << 31), M.MVR_E_UNSUPPORTED, "2^31 pages"),
    (dict(max_q_len=0), M.MVR_E_INVALID_ARGUMENT, "at least one token"),
    (dict(max_q_len=65), M.MVR_E_INVALID_ARGUMENT, "mask rows of 2 words"),
    (dict(max_q_len=2000), M.MVR_E_INVALID_ARGUMENT, "max_seq_len 1024 is smaller"),
    (dict(max_pages_per_seq=63), M.MVR_E_PAGES_UNCOVERED, "leaving 16 tokens uncovered"),
    (dict(total_q=81), M.MVR_E_INVALID_ARGUMENT, "total_q 81"),
    (dict(total_q=-1), M.MVR_E_INVALID_ARGUMENT, "total_q"),
    (dict(sum_seq_lens=5000), M.MVR_E_INVALID_ARGUMENT, "sum_seq_lens"),
    (dict(scale=-1.0), M.MVR_E_INVALID_ARGUMENT, "scale"),
    (dict(scale=float("nan")), M.MVR_E_INVALID_ARGUMENT, "scale"),
    (dict(q=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(q=FAKE + 8), M.MVR_E_INVALID_ARGUMENT, "16-byte aligned"),
    (dict(q_stride_token=132), M.MVR_E_INVALID_ARGUMENT, "strides"),
    (dict(cu_q_lens=None), M.MVR_E_INVALID_ARGUMENT, "required when num_seqs > 1"),
    (dict(masks=None), M.MVR_E_INVALID_ARGUMENT, "masks is null"),
    (dict(masks=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(mask_words=1), M.MVR_E_INVALID_ARGUMENT, "mask rows"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 20), M.MVR_E_INVALID_ARGUMENT, "256-byte aligned"),
])
def test_tree_refusals(change, code, text):
    rc, message = status("mvr_paged_attention_tree", *tree_args(**change))
    assert rc == code and text in message, message
    if "workspace" not in change:
        assert D.load_library().mvr_paged_attention_tree_workspace_size(*map(ctypes.byref, tree_args(**change))) == 0


def test_tree_null_structs():
    a, t = tree_args()
    assert status("mvr_paged_attention_tree", None, t)[0] == M.MVR_E_INVALID_ARGUMENT
    assert status("mvr_paged_attention_tree", a, None)[0] == M.MVR_E_INVALID_ARGUMENT


def test_tree_validate():
    a, t = tree_args(total_q=60)
    bt = np.arange(128, dtype=np.int32).reshape(2, 64)
    sl, cu = np.array([100, 1024], np.int32), np.array([0, 0, 40], np.int32)
    masks = np.full((60, 2), -1, np.int32)
    check = lambda **kw: D.validate_tree(a, t, **{**dict(  # noqa: E731
        block_tables_host=bt, seq_lens_host=sl, cu_q_lens_host=cu, masks_host=masks), **kw})
    check()  # an empty request is legal
    for kw, code, text in (
            (dict(cu_q_lens_host=np.array([1, 2, 3])), M.MVR_E_INVALID_ARGUMENT, "cu_q_lens[0]"),
            (dict(cu_q_lens_host=np.array([0, 40, 39])), M.MVR_E_INVALID_ARGUMENT, "q_len -1"),
            (dict(cu_q_lens_host=np.array([0, 0, 41])), M.MVR_E_INVALID_ARGUMENT, "q_len 41"),
            (dict(cu_q_lens_host=np.array([0, 40, 61])), M.MVR_E_INVALID_ARGUMENT, "exceeds total_q"),
            (dict(seq_lens_host=np.array([100, 1025])), M.MVR_E_INVALID_ARGUMENT, "seq_len 1025"),
            (dict(seq_lens_host=np.array([100, 39])), M.MVR_E_LENGTH_MISMATCH, "expected at least 40"),
            (dict(block_tables_host=np.where(bt == 127, 1024, bt)), M.MVR_E_PAGE_ID, "id 1024"),
            (dict(block_tables_host=np.where(bt == 64, -1, bt)), M.MVR_E_PAGE_ID, "id -1"),
            (dict(masks_host=np.zeros((60, 2), np.int32)), M.MVR_E_INVALID_ARGUMENT, "does not see itself")):
        with pytest.raises(M.MvrError) as e:
            check(**kw)
        assert e.value.code == code and text in e.value.message, e.value.message
    check(block_tables_host=np.where(bt < 64, -1, bt))  # an empty request reads no page
    # Starts that descend again: refused before a mask row behind the table's end (here, zeros) is read.
    masks[10:] = 0
    a.total_q = 10
    with pytest.raises(M.MvrError) as e:
        check(cu_q_lens_host=np.array([0, 40, 5]), masks_host=masks[:10])
    assert "q_len -35" in e.value.message


def test_tree_workspace_follows_the_hints():
    """Bounded by the splits, none for batches that fill the device, and no table makes the plan fail."""
    lib = D.load_library()
    size = lambda **kw: lib.mvr_paged_attention_tree_workspace_size(*map(ctypes.byref, tree_args(**kw)))  # noqa: E731
    assert size(max_seq_len=64, max_q_len=4) == 0
    long = dict(max_seq_len=1 << 20, max_pages_per_seq=1 << 16, num_pages=1 << 20)
    assert 0 < size(**long) < 1 << 30
    assert size(num_seqs=4096, max_q_len=8) == 0
    for lens, cu in (([1024, 1], [0, 40, 41]), ([0, 0], [0, 0, 0]), ([-5, 1 << 30], [0, -1, 7]), ([5, 5], [0, 40, 80])):
        sl, cu = np.array(lens, np.int32), np.array(cu, np.int32)
        assert size(seq_lens_host=sl.ctypes.data, cu_q_lens_host=cu.ctypes.data) >= 0


def test_tree_masks():
    cu = np.array([0, 4, 4, 6])
    masks = D.tree_masks([-1, 0, 0, 2, -1, -1], cu)
    assert masks.shape == (6, 1) and masks[:, 0].tolist() == [1, 3, 5, 13, 1, 2]
    chain = D.tree_masks(np.arange(70) - 1, np.array([0, 70])).view(np.uint32)
    assert chain.shape == (70, 3) and chain[69].tolist() == [2 ** 32 - 1, 2 ** 32 - 1, 63]
    with pytest.raises(M.MvrError, match="does not come before"):
        D.tree_masks([0], np.array([0, 1]))
    with pytest.raises(M.MvrError, match="cannot hold"):
        D.tree_masks([-1] * 33, np.array([0, 33]), mask_words=1)


# ---- norm, rotation, append ------------------------------------------------

def append_args(**kw):
    a = M.RopeAppendArgs()
    a.dtype, a.rope_type, a.num_seqs, a.num_q_heads, a.num_kv_heads, a.head_dim = M.DTYPE_F16, 0, 2, 8, 2, 64
    a.page_size, a.num_pages, a.max_pages_per_seq, a.total_q, a.max_seq_len, a.rope_len = 16, 64, 8, 10, 128, 128
    for name in ("q", "k", "v", "cos_table", "sin_table", "block_tables", "seq_lens", "cu_q_lens", "q_out", "key_pool",
                 "value_pool"):
        setattr(a, name, FAKE)
    for name in ("q", "k", "v", "q_out"):
        setattr(a, name + "_stride_head", 640)
        setattr(a, name + "_stride_token", 64)
    n = D.HeadNorms(FAKE, FAKE, 1e-6, FAKE)
    for k, v in kw.items():
        setattr(n if hasattr(n, k) else a, k, v)
    return a, n


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=5), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(rope_type=2), M.MVR_E_UNSUPPORTED, "rope_type"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(num_q_heads=7), M.MVR_E_INVALID_ARGUMENT, "multiple of num_kv_heads"),
    (dict(head_dim=60), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=520), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(total_q=0), M.MVR_E_INVALID_ARGUMENT, "empty"),
    (dict(max_seq_len=0), M.MVR_E_INVALID_ARGUMENT, "max_seq_len"),
    (dict(rope_len=0), M.MVR_E_INVALID_ARGUMENT, "rope_len"),
    (dict(rope_len=100, positions=None), M.MVR_E_INVALID_ARGUMENT, "100 positions"),
    (dict(max_pages_per_seq=7), M.MVR_E_PAGES_UNCOVERED, "cannot hold"),
    (dict(seq_lens=None), M.MVR_E_INVALID_ARGUMENT, "required when num_seqs > 1"),
    (dict(value_pool=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(eps=-1e-6), M.MVR_E_INVALID_ARGUMENT, "eps"),
    (dict(eps=float("nan")), M.MVR_E_INVALID_ARGUMENT, "eps"),
    (dict(eps=float("inf")), M.MVR_E_INVALID_ARGUMENT, "eps"),
    (dict(k_weight=FAKE + 4), M.MVR_E_INVALID_ARGUMENT, "aligned"),
    (dict(k_stride_token=66), M.MVR_E_INVALID_ARGUMENT, "strides"),
    (dict(total_q=1 << 26), M.MVR_E_UNSUPPORTED, "more than one call takes"),
])
def test_append_refusals(change, code, text):
    rc, message = status("mvr_norm_rope_append", *append_args(**change))
    assert rc == code and text in message, message


def test_append_validate():
    a, n = append_args()
    bt = np.arange(16, dtype=np.int32).reshape(2, 8)
    ok = dict(block_tables_host=bt, seq_lens_host=np.array([7, 40]), cu_q_lens_host=np.array([0, 0, 9]),
              positions_host=np.arange(10), page_writable_host=np.ones(64))
    D.validate_norm_rope_append(a, n, **ok)
    shared = bt.copy()
    shared[1, 2] = 0
    for kw, code, text in (
            (dict(cu_q_lens_host=np.array([0, 5, 11])), M.MVR_E_INVALID_ARGUMENT, "total_q"),
            (dict(cu_q_lens_host=np.array([0, 5, 4])), M.MVR_E_INVALID_ARGUMENT, "decreases"),
            (dict(cu_q_lens_host=np.array([0, 10, 5]), positions_host=np.full(10, -1)), M.MVR_E_INVALID_ARGUMENT, "decreases"),
            (dict(seq_lens_host=np.array([7, 129])), M.MVR_E_INVALID_ARGUMENT, "129"),
            (dict(seq_lens_host=np.array([7, 8])), M.MVR_E_LENGTH_MISMATCH, "after appending 9"),
            (dict(positions_host=np.full(10, 128)), M.MVR_E_INVALID_ARGUMENT, "position 128"),
            (dict(block_tables_host=bt + 60), M.MVR_E_PAGE_ID, "outside a pool"),
            (dict(page_writable_host=np.arange(64) != 10), M.MVR_E_READ_ONLY_PAGE, "cannot mutate written physical page 10"),
            (dict(block_tables_host=shared, cu_q_lens_host=np.array([0, 1, 10])), M.MVR_E_INVALID_ARGUMENT, "more than one")):
        with pytest.raises(M.MvrError) as e:
            D.validate_norm_rope_append(a, n, **{**ok, **kw})
        assert e.value.code == code and text in e.value.message, e.value.message


# ---- compaction and copies -------------------------------------------------

def compact_args(**kw):
    a = D.CompactDraftsArgs()
    a.dtype, a.num_layers, a.num_seqs, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages = M.DTYPE_F16, 2, 2, 2, 64, 4, 64
    a.max_pages_per_seq, a.max_seq_len, a.max_accepted = 8, 32, 4
    for name in ("key_pool", "value_pool", "block_tables", "seq_lens", "cu_q_lens", "accepted", "accepted_lens"):
        setattr(a, name, FAKE)
    a.new_seq_lens = 2 * FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(num_layers=0), M.MVR_E_INVALID_ARGUMENT, "num_layers"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(head_dim=0), M.MVR_E_INVALID_ARGUMENT, "geometry"),
    (dict(head_dim=1 << 30), M.MVR_E_UNSUPPORTED, "2^31 elements"),
    (dict(max_accepted=0), M.MVR_E_INVALID_ARGUMENT, "max_accepted"),
    (dict(max_seq_len=0), M.MVR_E_INVALID_ARGUMENT, "max_seq_len"),
    (dict(max_pages_per_seq=7), M.MVR_E_PAGES_UNCOVERED, "cannot hold"),
    (dict(key_pool=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(accepted=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(key_pool=FAKE + 1), M.MVR_E_INVALID_ARGUMENT, "aligned"),
    (dict(new_seq_lens=FAKE + 4), M.MVR_E_INVALID_ARGUMENT, "overlap"),
    *((dict({table: 2 * FAKE + 4}), M.MVR_E_INVALID_ARGUMENT, "overlap")
      for table in ("seq_lens", "cu_q_lens", "accepted", "accepted_lens", "block_tables")),
    (dict(num_layers=1 << 20, num_seqs=1 << 20, new_seq_lens=None), M.MVR_E_UNSUPPORTED, "more layers"),
])
def test_compact_refusals(change, code, text):
    rc, message = status("mvr_compact_drafts", compact_args(**change))
    assert rc == code and text in message, message


def test_compact_validate():
    a = compact_args()
    bt = np.arange(32, dtype=np.int32).reshape(2, 2, 8)
    ok = dict(block_tables_host=bt, seq_lens_host=np.array([12, 9]), cu_q_lens_host=np.array([0, 5, 9]),
              accepted_host=np.array([[0, 2, 4, 9], [1, 3, -1, -1]]), accepted_lens_host=np.array([3, 2]))
    D.validate_compact_drafts(a, **ok)
    same = bt.copy()
    same[1] = bt[0]
    for kw, code, text in (
            (dict(accepted_lens_host=np.array([4, 2])), M.MVR_E_INVALID_ARGUMENT, "draft 9"),
            (dict(accepted_lens_host=np.array([5, 2])), M.MVR_E_INVALID_ARGUMENT, "more than it has"),
            (dict(accepted_lens_host=np.array([-1, 2])), M.MVR_E_INVALID_ARGUMENT, "more than it has"),
            (dict(accepted_host=np.array([[0, 2, 2, 0], [1, 3, 0, 0]])), M.MVR_E_INVALID_ARGUMENT, "ascend"),
            (dict(seq_lens_host=np.array([4, 9])), M.MVR_E_LENGTH_MISMATCH, "expected at least 5"),
            (dict(seq_lens_host=np.array([33, 9])), M.MVR_E_INVALID_ARGUMENT, "seq_len 33"),
            (dict(cu_q_lens_host=np.array([0, 5, 4])), M.MVR_E_INVALID_ARGUMENT, "decreases"),
            (dict(block_tables_host=bt + 60), M.MVR_E_PAGE_ID, "outside a pool"),
            (dict(block_tables_host=same), M.MVR_E_INVALID_ARGUMENT, "more than one request or layer")):
        with pytest.raises(M.MvrError) as e:
            D.validate_compact_drafts(a, **{**ok, **kw})
        assert e.value.code == code and text in e.value.message, e.value.message


def copy_args(**kw):
    a = D.CopyPagesArgs()
    a.dtype, a.num_copies, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages = M.DTYPE_F16, 3, 2, 64, 4, 64
    a.key_pool = a.value_pool = a.src_pages = a.dst_pages = FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(num_copies=-1), M.MVR_E_INVALID_ARGUMENT, "num_copies"),
    (dict(page_size=0), M.MVR_E_INVALID_ARGUMENT, "geometry"),
    (dict(src_pages=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(value_pool=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(num_copies=1 << 30, page_size=1 << 10), M.MVR_E_UNSUPPORTED, "more than one call takes"),
    (dict(num_copies=1 << 23), M.MVR_E_UNSUPPORTED, "more than one call takes"),  # (2^24 blocks of 256 threads)
])
def test_copy_refusals(change, code, text):
    rc, message = status("mvr_copy_pages", copy_args(**change))
    assert rc == code and text in message, message


def test_copy_of_nothing_launches_nothing():
    assert status("mvr_copy_pages", copy_args(num_copies=0, src_pages=None, dst_pages=None))[0] == M.MVR_OK


def test_copy_validate():
    a = copy_args()
    D.validate_copy_pages(a, np.array([1, 1, 2]), np.array([3, 4, 5]), np.array([0, 4, 2]))
    for lists, code, text in (
            (([1, 1, 64], [3, 4, 5]), M.MVR_E_PAGE_ID, "source page 64"),
            (([1, 1, 2], [3, -1, 5]), M.MVR_E_PAGE_ID, "destination page -1"),
            (([1, 1, 2], [3, 4, 3]), M.MVR_E_INVALID_ARGUMENT, "twice a destination"),
            (([1, 1, 2], [3, 2, 5]), M.MVR_E_INVALID_ARGUMENT, "a source"),
            (([1, 1, 2], [3, 4, 5], [0, 5, 2]), M.MVR_E_INVALID_ARGUMENT, "5 tokens")):
        with pytest.raises(M.MvrError) as e:
            D.validate_copy_pages(a, *map(np.array, lists))
        assert e.value.code == code and text in e.value.message, e.value.message


# ---- what the Python binding itself refuses ----------------------------------

def test_python_refusals():
    torch = pytest.importorskip("torch")
    pool = torch.zeros((4, 1, 2, 16, 64), dtype=torch.float16)
    q = torch.zeros((4, 3, 64), dtype=torch.float16)
    table, lens, cu = (torch.zeros(s, dtype=torch.int32) for s in ((1, 4), (1,), (2,)))
    masks = torch.zeros((3, 1), dtype=torch.int32)
    kw = dict(max_q_len=3, max_seq_len=20)

    def tree(**changed):
        t = {**dict(q=q, key_pool=pool, value_pool=pool, block_tables=table, seq_lens=lens, cu_q_lens=cu, masks=masks,
                    out=q), **changed}
        with pytest.raises(M.MvrError) as e:
            D.make_tree_call(**t, **kw)
        return e.value.message

    assert "must be on a GPU" in tree()
    assert "one dtype" in tree(out=q.float())
    assert "head_dim" in tree(q=q[..., :32], out=q[..., :32])
    assert "masks" in tree(masks=masks[:2])
    assert "masks" in tree(masks=masks.long())
    assert "seq_lens" in tree(seq_lens=lens.repeat(2))
    assert "cu_q_lens" in tree(cu_q_lens=cu[:1])
    assert "block_tables" in tree(block_tables=table.long())
    assert "contiguous" in tree(key_pool=pool.transpose(2, 3), value_pool=pool.transpose(2, 3))
    with pytest.raises(M.MvrError, match="shape"):
        D.make_copy_pages_call(pool, pool, table[0], table[0, :2])
    with pytest.raises(M.MvrError, match="accepted"):
        D.make_compact_drafts_call(pool, pool, table, lens, cu, table.repeat(2, 1), lens, max_seq_len=20)
    with pytest.raises(M.MvrError, match="one dtype"):
        D.make_norm_rope_append_call(q, q[:2], q[:2], torch.zeros(64), None, q[0], q[0], table, lens, cu, pool, pool, q,
                                     eps=0.0, max_seq_len=20)
