"""Every plan of the scored attention kernels, as test_gpu_score_plans.py runs them, on the cases of tables at the ends of
their types, of values that are not finite, of scores on both sides of a cap and of prompts among thousands of requests."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, F32 = torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")
UNSPLIT = str(1 << 20)


def cases():
    import test_gpu_score_bounds as B
    import test_gpu_score_mixed as X
    import test_gpu_score_nonfinite as N
    import test_gpu_score_precision as P

    for dtype in (F16, F32):
        for window in (0, 2 ** 31 - 1):
            for q in ([5, 3, 5, 7, 2], [45, 40, 5, 70, 60]):
                yield f"{dtype} ranges {window}", lambda a=(dtype, q, window): B.test_row_ranges_at_the_ends_of_32_bits(*a)
        for q in ([1, 1, 1], [60, 90, 1]):
            yield f"{dtype} length 0", lambda a=(dtype, q, 0): B.test_requests_of_length_0_with_query_tokens(*a)
        for new in (1, 8, 80):
            for cap in (300.0, 1e5):
                yield f"{dtype} {new} beside {cap}", lambda a=(dtype, cap, new): P.test_small_scores_beside_one_past_the_cap(*a)
        for new in (1, 6, 80):
            for what, dims in ((INF, 5), (-INF, 5), (NAN, 5), (NAN, slice(None))):
                yield f"{dtype} {new} {what} keys", lambda a=(dtype, new, what, dims, 30.0): N.test_keys_under_a_cap(*a)
            for what in (INF, NAN):
                yield f"{dtype} {new} {what} values", lambda a=(dtype, new, what): N.test_values_amid_a_long_context(*a)
    yield "thousands", lambda: X.test_one_prompt_among_thousands(F16, 2100)


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
