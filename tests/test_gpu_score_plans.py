"""Every plan of the scored attention kernels: the planner's overrides, which a process reads once, fix the row tile and the
split of the keys in child processes that run the cases of test_gpu_score_attention.py, whatever the planner would take."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, F32 = torch.float16, torch.float32
UNSPLIT = str(1 << 20)


def cases():
    import test_gpu_score_attention as A
    from score_reference import Batch

    def shape(dtype, d, page, rules):
        """From one row to several of the largest tiles, keys from one unit to several parts."""
        A.check(Batch(d + page, dtype, 6, 2, d, page, [401, 64], [45, 33], **rules))

    for d in (32, 64, 96, 128, 160, 192, 224, 256):
        for dtype in (F16, F32):
            for rules in A.RULES:
                yield f"{dtype} {d} {rules}", lambda a=(dtype, d, 16, rules): A.test_every_head_dim_and_rule(*a)
            for page in (16, 24, 5):
                for rules in (dict(cap=30.0), dict(slopes=True, window=150), dict(prefix=[300, 20])):
                    yield f"{dtype} {d} page {page} {rules}", lambda a=(dtype, d, page, rules): shape(*a)
    for dtype in (F16, F32):
        for page in (1, 2, 4, 8, 12, 48, 100):
            yield f"{dtype} page {page}", lambda a=(dtype, page): A.test_page_sizes(*a)
        for cached in (0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 1000):
            yield f"{dtype} {cached} cached", lambda a=(dtype, cached): A.test_context_lengths(*a)
        for what in (float("inf"), float("nan")):
            for new in (1, 6, 80):
                yield f"{dtype} {new} {what}", lambda a=(dtype, new, what): A.test_values_that_are_not_finite(*a)
        for new in (1, 17, 65, 130):
            yield f"{dtype} {new} new", lambda a=(dtype, 8, 2, 128, new): A.test_new_tokens(*a)
    for window in (1, 16, 65, 200):
        yield f"window {window}", lambda a=(window, 90): A.test_windows(*a)
    for cap in (1e-3, 5.0, 1e6):
        yield f"cap {cap}", lambda a=cap: A.test_caps(a)
    for q in ([1] * 70 + [200], [1, 0, 1, 90, 0, 1, 1, 0, 1, 1], [0] * 64 + [129]):
        yield f"mixed {len(q)}", lambda a=(4, q): A.test_mixed_batches(*a)
    for f in (A.test_mixed_batch_of_thousands, A.test_mixed_graph_replays, A.test_scale_and_far_keys, A.test_rows_that_see_nothing, A.test_empty_requests_and_padded_rows,
              A.test_lse_is_not_wanted, A.test_strides, A.test_split_keys_and_workspaces, A.test_stale_hints,
              A.test_lengths_above_their_bounds_are_clamped, A.test_one_request_without_tables, A.test_pools_past_32_bits,
              A.test_many_requests, A.test_graph_replays, A.test_streams_and_repeats):
        yield f.__name__, f


@pytest.mark.parametrize("units", ["1", "3", UNSPLIT])  # of 64 keys in a part
@pytest.mark.parametrize("rows,waves", [(16, 4), (64, 4), (128, 4), (128, 8)])
def test_plans(rows, waves, units):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    env = dict(os.environ, MVR_SCORE_TILE_ROWS=str(rows), MVR_SCORE_TILE_WAVES=str(waves), MVR_SCORE_PART_UNITS=units,
               PYTHONPATH=os.pathsep.join([os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"),
                                           os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], env=env, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=110)
    print(r.stdout[-3000:], flush=True)
    assert r.returncode == 0, r.stdout[-3000:]
    assert "ran every case" in r.stdout


if __name__ == "__main__":
    for name, f in cases():
        print(name, flush=True)
        f()
    print("ran every case", flush=True)
