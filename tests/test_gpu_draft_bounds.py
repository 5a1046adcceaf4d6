"""mvr_paged_attention_tree at the edges of its contract: device tables with more drafts than max_q_len, infinities in a
draft's K row, tensors without rows.  By the planner's own plans and, in child processes (a process reads the overrides
once), in every row tile with the keys whole and in parts."""
import copy
import math
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_draft as D  # noqa: E402
from draft_reference import Batch, check_attention  # noqa: E402

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    D.load_library()


@pytest.mark.parametrize("dtype,page", [(F16, 16), (F16, 5), (F32, 16), (F32, 24)])
def test_drafts_above_the_bound_are_left_out(dtype, page):
    """A request with 75 drafts in the device's table and 33 in the call's bounds: its first 33 rows are computed as those
    of a request of 33 drafts, the others stay as they are, and so does whatever lies behind the last request."""
    bound = 33
    b = Batch(80, dtype, 8, 2, 64, page, [1500, 2400, 0, 40], [20, 75, 1, 3], "random", tail=4)
    t = b.device()
    t["masks"] = t["masks"][:, :2].contiguous()
    t["q"][:, int(b.cu[-1]):] = math.nan
    out = torch.full_like(t["q"], 7.0)
    for hints in ({}, dict(seq_lens_host=b.seq_lens, cu_q_lens_host=b.cu)):
        out.fill_(7.0)
        D.paged_attention_tree(**t, out=out, max_q_len=bound, max_seq_len=b.max_len, **hints)
        torch.cuda.synchronize()
        computed = np.concatenate([np.arange(lo, lo + min(n, bound)) for lo, n in zip(b.cu[:-1], b.q_lens)])
        same = copy.copy(b)
        same.q_lens = np.minimum(b.q_lens, bound).astype(np.int32)
        same.cached = b.seq_lens - same.q_lens
        same.cu = np.concatenate([[0], np.cumsum(same.q_lens)]).astype(np.int32)
        same.queries, same.bits = b.queries[:, computed], b.bits[computed]
        check_attention(out[:, computed], same)
        rest = np.setdiff1d(np.arange(out.shape[1]), computed)
        assert len(rest) == 75 - bound + 4 and bool((out[:, rest] == 7.0).all())


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("nodes", [6, 40])
def test_infinities_in_the_keys_of_drafts(dtype, page, nodes):
    """A score of plus infinity makes a row NaN, one of minus infinity leaves its key out; rows that do not see the draft
    are as without it."""
    for value in (math.inf, -math.inf):
        b = Batch(nodes, dtype, 8, 2, 128, page, [37, 0], [nodes, nodes], "tree")
        for request, slot in ((0, 2), (1, nodes - 1)):
            at = int(b.cached[request]) + slot
            b.key_pool[int(b.table[request, at // page]), 0, :, at % page, 3] = value
        got = D.paged_attention_tree(**b.device(), max_q_len=b.max_q, max_seq_len=b.max_len, seq_lens_host=b.seq_lens,
                                     cu_q_lens_host=b.cu)
        torch.cuda.synchronize()
        check_attention(got, b, note=str(value))
        for request, slot in ((0, 2), (1, nodes - 1)):
            rows = slice(int(b.cu[request]), int(b.cu[request + 1]))
            seen = torch.from_numpy(b.bits[rows, slot])
            up = (b.queries[:, rows, 3] * value) > 0  # [heads, rows]
            finite = torch.isfinite(got[:, rows].cpu())
            assert bool((finite.all(-1) == ~(seen & up)).all()) and bool((finite.any(-1) == finite.all(-1)).all())


def test_tensors_without_rows():
    b = Batch(81, F16, 4, 2, 64, 16, [20, 0], [0, 0], "tree")
    t = b.device()
    pools = t["key_pool"].clone(), t["value_pool"].clone()
    q, masks = t["q"][:, :0], t["masks"][:0]
    got = D.paged_attention_tree(**{**t, "q": q, "masks": masks}, max_q_len=1, max_seq_len=b.max_len)
    kv, cos = t["q"][:2, :0], torch.zeros((32, 32), dtype=F16, device="cuda")
    t.pop("q"), t.pop("masks")
    turned = D.norm_rope_append(q, kv, kv, None, None, cos, cos, eps=0.0, max_seq_len=b.max_len, **t)
    torch.cuda.synchronize()
    assert got.shape == turned.shape == (4, 0, 64)
    assert torch.equal(t["key_pool"], pools[0]) and torch.equal(t["value_pool"], pools[1])


@pytest.mark.parametrize("units", ["1", "7", str(1 << 20)])  # of 64 keys in a part
@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_every_plan(rows, units):
    env = dict(os.environ, MVR_DRAFT_TILE_ROWS=str(rows), MVR_DRAFT_PART_UNITS=units, PYTHONPATH=os.pathsep.join(
        [os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], env=env, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=110)
    print(r.stdout[-3000:], flush=True)
    assert r.returncode == 0, r.stdout[-3000:]
    assert "ran every case" in r.stdout


if __name__ == "__main__":
    for case in ((F16, 16), (F16, 5), (F32, 16), (F32, 24)):
        print("bound", *case, flush=True)
        test_drafts_above_the_bound_are_left_out(*case)
    for dtype_ in (F16, F32):
        for page_, nodes_ in ((16, 6), (5, 40)):
            print("infinities", dtype_, page_, nodes_, flush=True)
            test_infinities_in_the_keys_of_drafts(dtype_, page_, nodes_)
    print("ran every case", flush=True)
