"""What planning a tree call costs the host, paid for each layer: two passes over the batch's length tables and look-ups,
not a pass for each tile size, target and part length that the planner tries.  Measured on the sizing call, and on the call
itself with the whole and with half of the workspace that it asks for, where most of the splits tried do not fit (without a
GPU, where its launch fails; with one the addresses of these calls would be read)."""
import ctypes
import os
import time

import numpy as np
import pytest

import mvr_attn as M
import mvr_draft as D

LIB = M.library_path()
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="build the library first")
FAKE = 1 << 32


def call(n, lo, hi, nodes, hq, hkv, d):
    """A call of n requests of 1..nodes drafts on lo..hi tokens."""
    rng = np.random.default_rng(n)
    q = rng.integers(1, nodes + 1, n).astype(np.int32)
    seq = (rng.integers(lo, hi + 1, n) + q).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    a = M.PagedAttentionArgs()
    a.dtype, a.num_seqs, a.num_q_heads, a.num_kv_heads, a.head_dim = M.DTYPE_F16, n, hq, hkv, d
    a.page_size, a.num_pages, a.max_pages_per_seq = 16, 1 << 20, -(-int(seq.max()) // 16)
    a.max_q_len, a.max_seq_len, a.sum_seq_lens = int(q.max()), int(seq.max()), int(seq.sum())
    a.q = a.key_pool = a.value_pool = a.block_tables = a.seq_lens = a.cu_q_lens = a.out = FAKE
    a.q_stride_head, a.q_stride_token, a.out_stride_head, a.out_stride_token = 1 << 20, d, 1 << 20, d
    a.seq_lens_host, a.cu_q_lens_host = seq.ctypes.data, cu.ctypes.data
    a._keep = seq, cu
    return a, D.DraftTrees(FAKE, (nodes + 31) // 32)


def seconds(function, a, t):
    refs = ctypes.byref(a), ctypes.byref(t)
    best = 1.0
    for _ in range(30):
        start = time.perf_counter()
        for _ in range(20):
            function(*refs)
        best = min(best, (time.perf_counter() - start) / 20)
    return best


def test_planning_reads_the_tables_twice():
    size = D.load_library().mvr_paged_attention_tree_workspace_size
    shape = (100, 8000, 8, 14, 2, 64)
    per_request = (seconds(size, *call(4000, *shape)) - seconds(size, *call(500, *shape))) / 3500 * 1e9
    print(f"[plan cost] {per_request:.2f} ns per request of a tree call")
    # Both passes with their checks take about 7 ns a request (a pass of checks alone 2).
    assert per_request < 15


@pytest.mark.parametrize("n,shape", [(200, (100, 500, 8, 14, 2, 64)), (200, (1, 4000, 16, 8, 1, 64)),
                                     (128, (1, 4000, 16, 14, 2, 64))])
def test_planning_a_few_hundred_unequal_requests(n, shape):
    """Some 5 us, whatever the lengths; 30 to 50 where every trial walks the requests again."""
    size = D.load_library().mvr_paged_attention_tree_workspace_size
    took = seconds(size, *call(n, *shape)) * 1e6
    print(f"[plan cost] {n} requests {shape}: {took:.1f} us")
    assert took < 15


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the launch of this call has to fail")
@pytest.mark.parametrize("n,shape", [(200, (1, 4000, 16, 8, 1, 64)), (128, (1, 4000, 16, 14, 2, 64))])
def test_planning_within_a_workspace(n, shape):
    """The bytes that the sizing call names, or half of them, rule most splits out; finding that out costs no walk over the
    requests for each."""
    lib = D.load_library()
    a, t = call(n, *shape)
    need = lib.mvr_paged_attention_tree_workspace_size(ctypes.byref(a), ctypes.byref(t))
    assert need > 0
    a.workspace = FAKE
    took = []
    for size in (0, need, need // 2):  # (0: nothing to try; the launch that fails is most of it)
        a.workspace_bytes = size
        took.append(seconds(lib.mvr_paged_attention_tree, a, t) * 1e6)
    print(f"[plan cost] {n} requests {shape}: {took[1] - took[0]:.1f} and {took[2] - took[0]:.1f} us more with the whole "
          "and with half of the workspace")
    assert max(took) - took[0] < 30
