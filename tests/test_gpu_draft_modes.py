"""The drafted-tree calls in the checked mode and with trace ranges on (flags that a process reads once, hence the child
processes), and from two threads at a time."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_draft as D  # noqa: E402
from draft_reference import Batch, check_attention  # noqa: E402

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def skip_without_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    D.load_library()


def step():
    """Arguments of a small step: append, attention, compaction, copy."""
    b = Batch(70, torch.float16, 8, 2, 64, 16, [37, 300], [9, 5], "tree", spare=4)
    t = b.device()
    gen = torch.Generator().manual_seed(71)
    normal = lambda *shape: torch.randn(shape, generator=gen).half().cuda()  # noqa: E731
    ints = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    used = set(b.table[0, :3]) | set(b.table[1, :20])
    free = [p for p in range(b.num_pages) if p not in used]
    return b, {
        "append": dict(q=normal(8, 14, 64), k=normal(2, 14, 64), v=normal(2, 14, 64), q_weight=normal(64),
                       k_weight=normal(64), cos_table=normal(512, 32), sin_table=normal(512, 32),
                       positions=ints(*range(14)), eps=1e-6, max_seq_len=b.max_len,
                       **{k: t[k] for k in ("block_tables", "seq_lens", "cu_q_lens", "key_pool", "value_pool")}),
        "attention": dict(t, max_q_len=b.max_q, max_seq_len=b.max_len),
        "compact": dict(accepted=ints(0, 2, 5, 1, 4, 0).view(2, 3), accepted_lens=ints(3, 2), max_seq_len=b.max_len,
                        **{k: t[k] for k in ("block_tables", "seq_lens", "cu_q_lens", "key_pool", "value_pool")}),
        "copy": dict(src_pages=ints(int(b.table[0, 0])), dst_pages=ints(free[0]), tokens=ints(7),
                     key_pool=t["key_pool"], value_pool=t["value_pool"]),
    }


CALLS = {"append": D.norm_rope_append, "attention": D.paged_attention_tree, "compact": D.compact_drafts,
         "copy": D.copy_pages}


def run_step():
    b, args = step()
    outs = {}
    for name, f in CALLS.items():
        got = f(**args[name])
        torch.cuda.synchronize()
        if got is not None:
            outs[name] = got.cpu().numpy()
    outs["key_pool"], outs["value_pool"] = (args["copy"][k].cpu().numpy() for k in ("key_pool", "value_pool"))
    return outs


BROKEN = {  # a call, what breaks it, and the status it gets in the checked mode
    "page outside the pool": ("attention", lambda a: a["block_tables"][1].fill_(10 ** 6), M.MVR_E_PAGE_ID),
    "length above its bound": ("attention", lambda a: a["seq_lens"].fill_(10 ** 6), M.MVR_E_INVALID_ARGUMENT),
    "descending starts": ("attention", lambda a: a["cu_q_lens"][1].fill_(99), M.MVR_E_INVALID_ARGUMENT),
    "position outside the tables": ("append", lambda a: a["positions"].fill_(512), M.MVR_E_INVALID_ARGUMENT),
    "page of two requests": ("append", lambda a: a["block_tables"].fill_(1), M.MVR_E_INVALID_ARGUMENT),
    "descending path": ("compact", lambda a: a["accepted"].fill_(2), M.MVR_E_INVALID_ARGUMENT),
    "more accepted than drafted": ("compact", lambda a: a["accepted_lens"].fill_(4), M.MVR_E_INVALID_ARGUMENT),
    "copy onto itself": ("copy", lambda a: a["dst_pages"].copy_(a["src_pages"]), M.MVR_E_INVALID_ARGUMENT),
    "copy to no page": ("copy", lambda a: a["dst_pages"].fill_(-1), M.MVR_E_PAGE_ID),
}


def child(out_path):
    outs = run_step()
    for name, (call, spoil, _) in BROKEN.items():
        _, args = step()
        spoil(args[call])
        code = 0
        try:
            CALLS[call](**args[call])
        except M.MvrError as e:
            code = e.code
        torch.cuda.synchronize()
        outs[name] = np.array(code)
        print(name, code, flush=True)
    np.savez(out_path, **outs)


def test_checked_mode_and_trace_ranges(tmp_path):
    """Valid calls give the same bits as without; broken tables are reported and nothing is launched on them."""
    skip_without_gpu()
    path = str(tmp_path / "child.npz")
    env = dict(os.environ, MVR_ATTN_CHECKED="true", MVR_ENABLE_ROCTX="true", PYTHONPATH=os.pathsep.join(
        [os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__), path], env=env, capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    got, want = np.load(path), run_step()
    for name, x in want.items():
        assert got[name].tobytes() == x.tobytes(), name
    for name, (_, _, code) in BROKEN.items():
        assert int(got[name]) == code, (name, int(got[name]), code)


def test_two_threads():
    """Calls from two threads on streams of their own, at once: every result is its own batch's, and an error's message
    stays with the thread that made it."""
    skip_without_gpu()
    batches = [Batch(72 + i, torch.float16, 8, 2, 128, 16, [1500 + 900 * i, 40], [20, 7 + i], "tree") for i in range(2)]
    tensors, failures = [b.device() for b in batches], []
    outs = [[torch.empty_like(t["q"]) for _ in range(20)] for t in tensors]
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(i):
        b, t, stream = batches[i], tensors[i], torch.cuda.Stream()
        try:
            start.wait(30)
            for out in outs[i]:
                D.paged_attention_tree(**t, out=out, max_q_len=b.max_q, max_seq_len=b.max_len, stream=stream,
                                       seq_lens_host=b.seq_lens, cu_q_lens_host=b.cu)
                with pytest.raises(M.MvrError, match=f"mask rows of 1 words cannot hold max_q_len {33 + i}"):
                    D.paged_attention_tree(**t, out=out, max_q_len=33 + i, max_seq_len=b.max_len, stream=stream)
            stream.synchronize()
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join(60)
    assert not failures, failures
    for b, t, results in zip(batches, tensors, outs):
        check_attention(results[0], b)
        assert all(torch.equal(r, results[0]) for r in results[1:])


if __name__ == "__main__":
    child(sys.argv[1])
