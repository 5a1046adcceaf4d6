"""Every plan of the tree attention kernels: the planner's overrides, which a process reads once, fix the row tile and the
split of the keys in child processes that run the cases of test_gpu_draft_attention.py, whatever the planner would take."""
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
    import test_gpu_draft_attention as A
    from draft_reference import Batch, check_attention

    def shape(dtype, d, page):
        """Trees from one row to several of the largest tiles, keys from one unit to several parts."""
        for masks, cached, nodes in (("random", [0, 13, 250], [7, 1, 12]), ("tree", [401, 64], [45, 33])):
            check_attention(A.run(b := Batch(d + page, dtype, 6, 2, d, page, cached, nodes, masks)), b)

    for d in (32, 64, 96, 128, 160, 192, 224, 256):
        for dtype in (F16, F32):
            for page in (16, 24, 5):
                yield f"{dtype} {d} page {page}", lambda a=(dtype, d, page): shape(*a)
    for dtype in (F16, F32):
        for page in (1, 2, 4, 8, 12, 48, 100):
            yield f"{dtype} page {page}", lambda a=(dtype, page): A.test_page_sizes(*a)
        for cached in (0, 1, 15, 16, 17, 31, 33, 63, 64, 65):
            yield f"{dtype} drafts from {cached}", lambda a=(dtype, cached): A.test_where_the_drafts_begin(*a)
        for page, nodes in ((16, 10), (24, 40), (5, 70)):
            yield f"{dtype} non-finite {page} {nodes}", \
                lambda a=(dtype, page, nodes): A.test_non_finite_drafts_reach_only_the_rows_that_see_them(*a)
        yield f"{dtype} slots behind", lambda a=dtype: A.test_slots_behind_the_sequences_may_hold_anything(a)
        yield f"{dtype} large scores", lambda a=dtype: A.test_large_scores(a)
        yield f"{dtype} strides", lambda a=dtype: A.test_strides(a)
    for f in (A.test_no_host_tables, A.test_rows_that_see_nothing_are_zero,
              A.test_mask_bits_behind_the_drafts_count_for_nothing, A.test_rows_behind_the_last_request_stay,
              A.test_bad_page_ids_read_inside_the_pool, A.test_lengths_above_the_bounds_are_clamped,
              A.test_pool_offsets_past_32_bits, A.test_thousands_of_empty_requests,
              A.test_same_bits_each_time):
        yield f.__name__, f
    if os.environ["MVR_DRAFT_PART_UNITS"] != UNSPLIT:
        yield "replayed", A.test_graph_replayed_for_other_lengths  # (its point is the workspace)


@pytest.mark.parametrize("units", ["1", "3", UNSPLIT])  # of 64 keys in a part
@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_plans(rows, units):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    env = dict(os.environ, MVR_DRAFT_TILE_ROWS=str(rows), MVR_DRAFT_PART_UNITS=units, PYTHONPATH=os.pathsep.join(
        [os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
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
