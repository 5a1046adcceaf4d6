"""CPU-side checks of the calls on scores: the library exports what include/mvr_score.h declares, the bindings agree with
it, the host checks refuse bad arguments and tables before any launch, planning is bounded."""
import contextlib
import ctypes
import os
import re
import subprocess
import tempfile
import time

import numpy as np
import pytest

import mvr_attn as M
import mvr_draft as D
import mvr_score as S
import test_rust_binding as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mvr_score.h")
RUST = os.path.join(ROOT, "mini-vllm-rs_amd", "rust", "mvr_score.rs")
FAKE = 1 << 20  # an aligned address: these calls never launch


# ---- header and bindings ---------------------------------------------------

@pytest.fixture()
def score_header(monkeypatch):
    """The parsers of the other header's test on this one."""
    monkeypatch.setattr(R, "HEADER", HEADER)
    monkeypatch.setattr(R, "RUST", RUST)


RUST_NAMES = {"mvr_score_rules": "MvrScoreRules", "mvr_key_weights": "MvrKeyWeights",
              "mvr_select_tokens_args": "MvrSelectTokensArgs", "mvr_move_tokens_args": "MvrMoveTokensArgs",
              "mvr_paged_attention_args": "MvrPagedAttentionArgs"}
TYPES = {**R.C_TO_RUST, "int32_t*": "*mut i32", "const float*": "*const f32", "float*": "*mut f32"}


def test_library_exports_every_declared_symbol(score_header):
    declared = set(R.c_functions())
    assert declared == set(S.EXPORTED_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", M.library_path()], capture_output=True, text=True, check=True)
    assert declared <= set(re.findall(r"\bT (mvr_[a-z0-9_]+)$", out.stdout, flags=re.M))
    lib = S.load_library()
    assert all(getattr(lib, name).argtypes for name in declared)


def test_rust_source_matches_the_header(score_header):
    structs, rust = R.c_structs(), R.rust_structs()
    assert set(structs) == set(S.STRUCTS)
    for name, fields in structs.items():
        assert [(n, TYPES[t]) for n, t in fields] == rust[RUST_NAMES[name]], name
    functions, rust = R.c_functions(), R.rust_functions()
    assert set(rust) == set(functions)
    for name, (ret, args) in functions.items():
        want = [TYPES.get(t) or "*const " + RUST_NAMES[t[len("const "):-1]] for t in args]
        assert (TYPES[ret], want) == rust[name], name


@pytest.mark.skipif(subprocess.run(["which", "gcc"], capture_output=True).returncode != 0, reason="no gcc")
def test_ctypes_mirror_has_the_c_layout(score_header):
    structs = R.c_structs()
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "mvr_score.h"', "int main(void) {"]
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
    for name, mirror in S.STRUCTS.items():
        assert [n for n, _ in mirror._fields_] == [n for n, _ in structs[name]]
        assert ctypes.sizeof(mirror) == got[(name, "sizeof")]
        for n, _ in mirror._fields_:
            assert getattr(mirror, n).offset == got[(name, n)], (name, n)


def status(name, *args):
    lib = S.load_library()
    refs = [ctypes.byref(x) if isinstance(x, ctypes.Structure) else x for x in args]
    return getattr(lib, name)(*refs), lib.mvr_last_error().decode()


def set_fields(blocks, changes):
    for k, v in changes.items():
        setattr(next(b for b in blocks if hasattr(b, k)), k, v)
    return blocks


# ---- attention -------------------------------------------------------------

def scored_args(**kw):
    a = M.PagedAttentionArgs()
    a.dtype, a.num_seqs, a.num_q_heads, a.num_kv_heads, a.head_dim, a.page_size = M.DTYPE_F16, 2, 32, 8, 128, 16
    a.num_pages, a.max_pages_per_seq, a.max_q_len, a.max_seq_len = 1024, 64, 40, 1024
    a.q = a.key_pool = a.value_pool = a.block_tables = a.seq_lens = a.cu_q_lens = a.out = FAKE
    a.q_stride_head = a.out_stride_head = 80 * 128
    a.q_stride_token = a.out_stride_token = 128
    return set_fields((a, S.ScoreRules(lse=FAKE, lse_stride_head=80)), kw)


ATTENTION = [
    (dict(dtype=2), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(num_kv_heads=5), M.MVR_E_INVALID_ARGUMENT, "multiple of num_kv_heads"),
    (dict(head_dim=100), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(head_dim=288), M.MVR_E_UNSUPPORTED, "head_dim"),
    (dict(page_size=0), M.MVR_E_INVALID_ARGUMENT, "page_size"),
    (dict(num_pages=0), M.MVR_E_INVALID_ARGUMENT, "num_pages"),
    (dict(num_pages=1 << 31), M.MVR_E_UNSUPPORTED, "2^31 pages"),
    (dict(max_q_len=0), M.MVR_E_INVALID_ARGUMENT, "at least one token"),
    (dict(max_q_len=2000), M.MVR_E_INVALID_ARGUMENT, "max_seq_len 1024 is smaller"),
    (dict(max_pages_per_seq=63), M.MVR_E_PAGES_UNCOVERED, "leaving 16 tokens uncovered"),
    (dict(max_seq_len=2 ** 31 - 100, max_pages_per_seq=2 ** 28), M.MVR_E_UNSUPPORTED, "too close to 2^31"),
    (dict(total_q=81), M.MVR_E_INVALID_ARGUMENT, "total_q 81"),
    (dict(total_q=-1), M.MVR_E_INVALID_ARGUMENT, "total_q"),
    (dict(scale=-1.0), M.MVR_E_INVALID_ARGUMENT, "scale"),
    (dict(scale=float("nan")), M.MVR_E_INVALID_ARGUMENT, "scale"),
    (dict(q=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(q=FAKE + 8), M.MVR_E_INVALID_ARGUMENT, "16-byte aligned"),
    (dict(q_stride_token=132), M.MVR_E_INVALID_ARGUMENT, "strides"),
    (dict(cu_q_lens=None), M.MVR_E_INVALID_ARGUMENT, "required when num_seqs > 1"),
    (dict(num_seqs=1, cu_q_lens=None, total_q=7), M.MVR_E_INVALID_ARGUMENT, "smaller than max_q_len"),
    (dict(num_seqs=1 << 24, max_q_len=40), M.MVR_E_UNSUPPORTED, "more than one call takes"),
    (dict(cap=-1.0), M.MVR_E_INVALID_ARGUMENT, "cap"),
    (dict(cap=float("nan")), M.MVR_E_INVALID_ARGUMENT, "cap"),
    (dict(cap=float("inf")), M.MVR_E_INVALID_ARGUMENT, "cap"),
    (dict(cap=1e-35), M.MVR_E_UNSUPPORTED, "cap"),
    (dict(cap=1e35), M.MVR_E_UNSUPPORTED, "cap"),
    (dict(window=-1), M.MVR_E_INVALID_ARGUMENT, "window"),
    (dict(slopes=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(first_keys=FAKE + 1), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(prefix_lens=FAKE + 3), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(lse=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(total_q=80, lse_stride_head=79), M.MVR_E_INVALID_ARGUMENT, "lse_stride_head 79"),
]


@pytest.mark.parametrize("change,code,text", ATTENTION + [
    (dict(value_pool=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(out=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 20), M.MVR_E_INVALID_ARGUMENT, "256-byte aligned"),
])
def test_attention_refusals(change, code, text):
    rc, message = status("mvr_paged_attention_scored", *scored_args(**change))
    assert rc == code and text in message, message
    if "workspace" not in change:
        assert S.load_library().mvr_paged_attention_scored_workspace_size(*map(ctypes.byref, scored_args(**change))) == 0


def test_null_structs():
    a, r = scored_args()
    w = S.KeyWeights(FAKE, 1.0, None)
    for name, args in (("mvr_paged_attention_scored", (None, r)), ("mvr_paged_attention_scored", (a, None)),
                       ("mvr_attention_weights", (None, r, w)), ("mvr_attention_weights", (a, None, w)),
                       ("mvr_attention_weights", (a, r, None)), ("mvr_select_tokens", (None,)), ("mvr_move_tokens", (None,))):
        assert status(name, *args)[0] == M.MVR_E_INVALID_ARGUMENT


VALIDATE = [
    (dict(cu_q_lens_host=np.array([1, 2, 3])), M.MVR_E_INVALID_ARGUMENT, "cu_q_lens[0]"),
    (dict(cu_q_lens_host=np.array([0, 40, 39])), M.MVR_E_INVALID_ARGUMENT, "q_len -1"),
    (dict(cu_q_lens_host=np.array([0, 0, 41])), M.MVR_E_INVALID_ARGUMENT, "q_len 41"),
    (dict(cu_q_lens_host=np.array([0, 40, 61])), M.MVR_E_INVALID_ARGUMENT, "exceeds total_q"),
    (dict(seq_lens_host=np.array([100, 1025])), M.MVR_E_INVALID_ARGUMENT, "seq_len 1025"),
    (dict(seq_lens_host=np.array([100, 39])), M.MVR_E_LENGTH_MISMATCH, "expected at least 40"),
    (dict(first_keys_host=np.full(60, -1)), M.MVR_E_INVALID_ARGUMENT, "first key -1"),
    (dict(prefix_lens_host=np.array([0, -2])), M.MVR_E_INVALID_ARGUMENT, "prefix of -2"),
    (dict(slopes_host=np.full(32, np.inf)), M.MVR_E_INVALID_ARGUMENT, "slope of head 0"),
]


def whole_tables():
    bt = np.arange(128, dtype=np.int32).reshape(2, 64)
    return bt, dict(block_tables_host=bt, seq_lens_host=np.array([100, 1024]), cu_q_lens_host=np.array([0, 0, 40]),
                    first_keys_host=np.zeros(60), prefix_lens_host=np.array([0, 5000]), slopes_host=np.ones(32))


def test_attention_validate():
    a, r = scored_args(total_q=60)
    bt, ok = whole_tables()
    S.validate_scored(a, r, **ok)  # an empty request is legal
    S.validate_scored(a, r)
    S.validate_scored(a, r, **{**ok, "block_tables_host": np.where(bt < 64, -1, bt)})  # it reads no page
    for kw, code, text in VALIDATE + [(dict(block_tables_host=np.where(bt == 127, 1024, bt)), M.MVR_E_PAGE_ID, "id 1024"),
                                      (dict(block_tables_host=np.where(bt == 64, -1, bt)), M.MVR_E_PAGE_ID, "id -1")]:
        with pytest.raises(M.MvrError) as e:
            S.validate_scored(a, r, **{**ok, **kw})
        assert e.value.code == code and text in e.value.message, e.value.message


def test_validate_leaves_out_what_only_the_device_knows():
    """One request whose tables are on the device alone: its bounds are not taken for its lengths."""
    bt = np.array([[5, 1 << 20]], np.int32)  # (one page is used, the other entry never written)
    sizes = dict(num_seqs=1, total_q=20, max_seq_len=32, max_pages_per_seq=2, max_q_len=20)
    one = dict(seq_lens_host=np.array([3]))
    for validate, args in ((S.validate_scored, scored_args(**sizes)), (S.validate_weights, weights_args(**sizes))):
        validate(*args, block_tables_host=bt)
        validate(*args, block_tables_host=bt, **one)
        validate(*args, block_tables_host=bt, **one, cu_q_lens_host=np.array([0, 1]))
        with pytest.raises(M.MvrError) as e:
            validate(*args, block_tables_host=bt, seq_lens_host=np.array([20]))
        assert e.value.code == M.MVR_E_PAGE_ID
    with pytest.raises(M.MvrError) as e:  # without tables the bounds are the lengths
        S.validate_weights(*weights_args(**sizes, seq_lens=None, cu_q_lens=None), block_tables_host=bt)
    assert e.value.code == M.MVR_E_PAGE_ID


def test_workspace_of_mixed_batches():
    """By the tokens that are there, not by the longest request in every place."""
    lens, cu = np.full(64, 2000, np.int32), np.concatenate([[0], np.cumsum([1] * 63 + [2000])]).astype(np.int32)
    a, r = scored_args(num_seqs=64, num_q_heads=7, num_kv_heads=1, max_q_len=2000, max_seq_len=2000, max_pages_per_seq=125,
                       total_q=int(cu[-1]), seq_lens_host=lens.ctypes.data, cu_q_lens_host=cu.ctypes.data, q_stride_head=1 << 20)
    assert S.load_library().mvr_paged_attention_scored_workspace_size(ctypes.byref(a), ctypes.byref(r)) < 256 << 20


def test_workspace_follows_the_hints():
    """Bounded by the splits, none for batches that fill the device, and no table makes the plan fail."""
    lib = S.load_library()
    size = lambda **kw: lib.mvr_paged_attention_scored_workspace_size(*map(ctypes.byref, scored_args(**kw)))  # noqa: E731
    assert size(max_seq_len=64, max_q_len=4) == 0
    long = dict(max_seq_len=1 << 20, max_pages_per_seq=1 << 16, num_pages=1 << 20, max_q_len=1, num_seqs=2)
    assert 0 < size(**long) < 1 << 30
    assert size(**long, window=64) == 0  # two units of keys
    assert size(num_seqs=4096, max_q_len=8) == 0
    for lens, cu in (([1024, 1], [0, 40, 41]), ([0, 0], [0, 0, 0]), ([-5, 1 << 30], [0, -1, 7]), ([5, 5], [0, 40, 80]),
                     ([2 ** 31 - 1] * 2, [-2 ** 31, 2 ** 31 - 1, -2 ** 31])):
        sl, cu = np.array(lens, np.int32), np.array(cu, np.int32)
        assert size(seq_lens_host=sl.ctypes.data, cu_q_lens_host=cu.ctypes.data) >= 0


def test_planning_reads_the_tables_once_per_tile_size():
    """Host time of a plan, paid for each layer: a few us for hundreds of unequal requests, some ns for each more."""
    lib = S.load_library()

    def seconds(n, most):
        rng = np.random.default_rng(n)
        q = rng.integers(1, most + 1, n).astype(np.int32)
        seq, cu = (rng.integers(1, 4000, n) + q).astype(np.int32), np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        a, r = scored_args(num_seqs=n, max_q_len=most, max_seq_len=4100, max_pages_per_seq=257,
                           seq_lens_host=seq.ctypes.data, cu_q_lens_host=cu.ctypes.data)
        refs, best = (ctypes.byref(a), ctypes.byref(r)), 1.0
        for _ in range(30):
            start = time.perf_counter()
            for _ in range(20):
                lib.mvr_paged_attention_scored_workspace_size(*refs)
            best = min(best, (time.perf_counter() - start) / 20)
        return best * 1e6

    small, large = seconds(200, 3), seconds(4000, 3)
    print(f"[plan cost] 200 requests {small:.1f} us, {(large - small) / 3.8:.1f} ns for each more")
    assert small < 25 and (large - small) / 3800 < 0.05
    assert seconds(200, 40) < 60


# ---- weights ---------------------------------------------------------------

def weights_args(**kw):
    a, r = scored_args()
    a.value_pool = a.out = None  # not used
    return set_fields((a, r, S.KeyWeights(FAKE, 1.0, None)), kw)


@pytest.mark.parametrize("change,code,text", ATTENTION + [
    (dict(lse=None), M.MVR_E_INVALID_ARGUMENT, "log-sum-exps"),
    (dict(weights=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(weights=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(fresh_from=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "4-byte aligned"),
    (dict(decay=-0.1), M.MVR_E_INVALID_ARGUMENT, "decay"),
    (dict(decay=float("nan")), M.MVR_E_INVALID_ARGUMENT, "decay"),
    (dict(decay=float("inf")), M.MVR_E_INVALID_ARGUMENT, "decay"),
    (dict(num_seqs=1 << 14, max_q_len=1, max_seq_len=1 << 20, max_pages_per_seq=1 << 16), M.MVR_E_UNSUPPORTED, "one call"),
])
def test_weights_refusals(change, code, text):
    rc, message = status("mvr_attention_weights", *weights_args(**change))
    assert rc == code and text in message, message


def test_weights_validate():
    a, r, w = weights_args(total_q=60)
    bt, ok = whole_tables()
    ok["fresh_from_host"] = np.array([0, 2 ** 31 - 1])
    S.validate_weights(a, r, w, **ok)
    S.validate_weights(a, r, w, **{**ok, "block_tables_host": np.where(bt < 64, 70, bt)})  # an empty request has no weights
    both = dict(cu_q_lens_host=np.array([0, 1, 40]), block_tables_host=np.where(bt == 64, 3, bt))
    for kw, code, text in VALIDATE + [(dict(fresh_from_host=np.array([0, -1])), M.MVR_E_INVALID_ARGUMENT, "fresh_from -1"),
                                      (both, M.MVR_E_INVALID_ARGUMENT, "page 3 holds the weights of more than one")]:
        with pytest.raises(M.MvrError) as e:
            S.validate_weights(a, r, w, **{**ok, **kw})
        assert e.value.code == code and text in e.value.message, e.value.message


# ---- selection and moves ---------------------------------------------------

def select_args(**kw):
    a = S.SelectTokensArgs(num_layers=2, num_seqs=2, num_kv_heads=2, page_size=4, num_pages=64, max_pages_per_seq=8,
                           max_seq_len=32, max_moves=16, recent=2, first=1)
    for i, name in enumerate(("weights", "positions", "block_tables", "seq_lens", "next_positions", "kept_lens", "keep_lens",
                              "moves", "num_moves", "new_seq_lens")):
        setattr(a, name, FAKE * (i + 1))
    return set_fields((a,), kw)[0]


@pytest.mark.parametrize("change,code,text", [
    (dict(num_layers=0), M.MVR_E_INVALID_ARGUMENT, "num_layers"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(num_kv_heads=0), M.MVR_E_INVALID_ARGUMENT, "geometry"),
    (dict(page_size=0), M.MVR_E_INVALID_ARGUMENT, "geometry"),
    (dict(num_pages=1 << 31), M.MVR_E_UNSUPPORTED, "2^31 pages"),
    (dict(num_pages=1 << 30, page_size=1 << 20), M.MVR_E_UNSUPPORTED, "2^40"),
    (dict(max_seq_len=0), M.MVR_E_INVALID_ARGUMENT, "max_seq_len"),
    (dict(max_seq_len=2 ** 31 - 1), M.MVR_E_UNSUPPORTED, "2^31"),
    (dict(max_pages_per_seq=7), M.MVR_E_PAGES_UNCOVERED, "cannot hold"),
    (dict(max_moves=0), M.MVR_E_INVALID_ARGUMENT, "max_moves"),
    (dict(recent=-1), M.MVR_E_INVALID_ARGUMENT, "recent"),
    (dict(first=-1), M.MVR_E_INVALID_ARGUMENT, "recent and first"),
    (dict(weights=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(positions=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(keep_lens=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(num_moves=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(weights=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "aligned"),
    (dict(moves=FAKE * 8 + 4), M.MVR_E_INVALID_ARGUMENT, "8-byte aligned"),
    (dict(positions=FAKE + 4), M.MVR_E_INVALID_ARGUMENT, "overlaps a table or the weights"),
    *((dict(new_seq_lens=FAKE * k + 4), M.MVR_E_INVALID_ARGUMENT, "overlap") for k in (2, 3, 4, 5, 6, 7, 8, 9)),
    (dict(num_layers=1 << 16, num_seqs=1 << 16), M.MVR_E_UNSUPPORTED, "more layers"),
])
def test_select_refusals(change, code, text):
    rc, message = status("mvr_select_tokens", select_args(**change))
    assert rc == code and text in message, message


def test_select_validate():
    a = select_args()
    bt = np.arange(32, dtype=np.int32).reshape(2, 2, 8)
    ok = dict(block_tables_host=bt, seq_lens_host=np.array([32, 9]), next_positions_host=np.array([50, 9]),
              kept_lens_host=np.array([16, 0]), keep_lens_host=np.array([16, 40]))
    S.validate_select(a, **ok)
    same = bt.copy()
    same[1] = bt[0]
    for kw, code, text in (
            (dict(seq_lens_host=np.array([33, 9])), M.MVR_E_INVALID_ARGUMENT, "seq_len 33"),
            (dict(seq_lens_host=np.array([-1, 9])), M.MVR_E_INVALID_ARGUMENT, "seq_len -1"),
            (dict(next_positions_host=np.array([50, 8])), M.MVR_E_LENGTH_MISMATCH, "next position 8"),
            (dict(kept_lens_host=np.array([33, 0])), M.MVR_E_LENGTH_MISMATCH, "kept_len 33"),
            (dict(kept_lens_host=np.array([-1, 0])), M.MVR_E_LENGTH_MISMATCH, "kept_len -1"),
            (dict(keep_lens_host=np.array([-1, 0])), M.MVR_E_INVALID_ARGUMENT, "keep_len -1"),
            (dict(keep_lens_host=np.array([2, 40])), M.MVR_E_INVALID_ARGUMENT, "fewer than the first 1 and the last 2"),
            (dict(block_tables_host=bt + 60), M.MVR_E_PAGE_ID, "outside a pool"),
            (dict(block_tables_host=same), M.MVR_E_INVALID_ARGUMENT, "more than one request or layer")):
        with pytest.raises(M.MvrError) as e:
            S.validate_select(a, **{**ok, **kw})
        assert e.value.code == code and text in e.value.message, e.value.message
    with pytest.raises(M.MvrError, match="more than max_moves 15"):
        S.validate_select(select_args(max_moves=15), **ok)


def move_args(**kw):
    a = S.MoveTokensArgs(dtype=M.DTYPE_F16, num_layers=1, num_seqs=2, num_kv_heads=2, head_dim=64, page_size=4, num_pages=64,
                         max_pages_per_seq=4, max_moves=3)
    for name in ("key_pool", "value_pool", "weights", "positions", "block_tables", "moves", "num_moves"):
        setattr(a, name, FAKE)
    return set_fields((a,), kw)[0]


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), M.MVR_E_UNSUPPORTED, "not F32"),
    (dict(num_layers=0), M.MVR_E_INVALID_ARGUMENT, "num_layers"),
    (dict(num_seqs=0), M.MVR_E_INVALID_ARGUMENT, "at least one request"),
    (dict(head_dim=0), M.MVR_E_INVALID_ARGUMENT, "geometry"),
    (dict(head_dim=1 << 30), M.MVR_E_UNSUPPORTED, "2^31 elements"),
    (dict(num_pages=1 << 31), M.MVR_E_UNSUPPORTED, "2^31 pages"),
    (dict(max_pages_per_seq=0), M.MVR_E_INVALID_ARGUMENT, "max_pages_per_seq"),
    (dict(max_moves=0), M.MVR_E_INVALID_ARGUMENT, "max_moves"),
    (dict(key_pool=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(moves=None), M.MVR_E_INVALID_ARGUMENT, "null"),
    (dict(moves=FAKE + 4), M.MVR_E_INVALID_ARGUMENT, "8-byte aligned"),
    (dict(key_pool=FAKE + 1), M.MVR_E_INVALID_ARGUMENT, "aligned"),
    (dict(positions=FAKE + 2), M.MVR_E_INVALID_ARGUMENT, "aligned"),
    (dict(num_layers=1 << 16, num_seqs=1 << 16), M.MVR_E_UNSUPPORTED, "more layers"),
])
def test_move_refusals(change, code, text):
    rc, message = status("mvr_move_tokens", move_args(**change))
    assert rc == code and text in message, message


def test_move_validate():
    a = move_args()
    bt = np.arange(8, dtype=np.int32).reshape(2, 4)
    moves = np.zeros((1, 2, 2, 3, 2), np.int32)
    moves[0, :, :, 0], moves[0, :, :, 1] = (12, 1), (15, 0)
    counts = np.array([2, 0, 2, 1])
    S.validate_move(a, bt, moves, counts)

    def broken(code, text, moves=moves, counts=counts, bt=bt):
        with pytest.raises(M.MvrError) as e:
            S.validate_move(a, bt, moves, counts)
        assert e.value.code == code and text in e.value.message, e.value.message

    def changed(move):
        x = moves.copy()
        x[0, 1, 0, 1] = move
        return x

    broken(M.MVR_E_INVALID_ARGUMENT, "4 moves", counts=np.array([2, 0, 2, 4]))
    broken(M.MVR_E_INVALID_ARGUMENT, "slot 16", moves=changed((16, 0)))
    broken(M.MVR_E_INVALID_ARGUMENT, "slot -1", moves=changed((15, -1)))
    broken(M.MVR_E_INVALID_ARGUMENT, "to slot 1 twice", moves=changed((15, 1)))
    broken(M.MVR_E_INVALID_ARGUMENT, "both to and from slot 1", moves=changed((1, 0)))
    broken(M.MVR_E_PAGE_ID, "outside a pool", bt=bt + 60)


# ---- the Python binding ------------------------------------------------------

def test_short_host_tables_are_refused():
    def refused(f, *args, **tables):
        with pytest.raises(M.MvrError, match="must hold"):
            f(*args, **tables)

    _, ok = whole_tables()
    a, r = scored_args(total_q=60)
    for name in ok:  # (first keys: of the requests' 40 tokens)
        refused(S.validate_scored, a, r, **{**ok, name: np.asarray(ok[name]).reshape(-1)[:39 if "first" in name else -1]})
    refused(S.validate_weights, *weights_args(total_q=60), fresh_from_host=np.zeros(1))
    refused(S.validate_select, select_args(), keep_lens_host=np.zeros(1))
    refused(S.validate_select, select_args(), block_tables_host=np.zeros(31))
    refused(S.validate_move, move_args(), moves_host=np.zeros(23))


def tensors(tokens=0):
    torch = pytest.importorskip("torch")
    pool = torch.zeros((4, 1, 2, 16, 64), dtype=torch.float16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(q=pool.new_zeros((4, tokens, 64)), key_pool=pool, value_pool=pool.clone(), block_tables=i32(3, 2),
                seq_lens=i32(3), cu_q_lens=i32(4))


def test_calls_on_no_rows_launch_nothing(monkeypatch):
    torch = pytest.importorskip("torch")
    for module in (D, S):
        monkeypatch.setattr(module, "_same_device", lambda *t: torch.device("cuda", 0))
        monkeypatch.setattr(module, "_scope", lambda device, stream: contextlib.nullcontext())
    monkeypatch.setattr(M, "_stream_handle", lambda stream: 0)
    t = tensors()
    out, lse = S.paged_attention_scored(**t, max_q_len=8, max_seq_len=20, cap=5.0, slopes=torch.ones(4))
    assert out.shape == t["q"].shape and lse.shape == (4, 0)
    weights = torch.full((4, 2, 16), 3.0)
    value_pool = t.pop("value_pool")
    assert S.attention_weights(lse=lse, weights=weights, **t, max_q_len=8, max_seq_len=20) is weights
    assert bool((weights == 3).all())
    with pytest.raises(M.MvrError, match="first_keys"):  # the tensors are checked all the same
        S.paged_attention_scored(value_pool=value_pool, **t, max_q_len=8, max_seq_len=20,
                                 first_keys=torch.zeros(2, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    t = tensors(3)
    with pytest.raises(M.MvrError, match="must be on a GPU"):
        S.paged_attention_scored(**t, max_q_len=3, max_seq_len=20)
    weights, positions = torch.zeros((4, 2, 16)), torch.zeros((4, 2, 16), dtype=torch.int32)
    lens = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(M.MvrError, match="must be on a GPU"):
        S.select_tokens(weights, positions, t["block_tables"], lens, None, None, lens, recent=0, max_seq_len=20, max_moves=4)
    moves, counts = torch.zeros((1, 3, 2, 4, 2), dtype=torch.int32), torch.zeros((1, 3, 2), dtype=torch.int32)
    with pytest.raises(M.MvrError, match="must be on a GPU"):
        S.move_tokens(t["key_pool"], t["value_pool"], weights, positions, t["block_tables"], moves, counts)
    with pytest.raises(M.MvrError, match="moves"):
        S.move_tokens(t["key_pool"], t["value_pool"], weights, positions, t["block_tables"], moves[:, :2], counts)
