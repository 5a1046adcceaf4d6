"""Batches of thousands of requests among which few are prompts: as many row tiles as the tokens there are take, not as the
longest request would take in every place."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402
from score_reference import Batch, check_attention  # noqa: E402
from test_gpu_score_attention import run  # noqa: E402
from test_gpu_score_weights import check as check_weights  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


@pytest.mark.parametrize("at", [0, 2100, 4199])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_one_prompt_among_thousands(dtype, at):
    """Row tiles of 16: 4.2 million padded, 5,200 packed."""
    rng = np.random.default_rng(at)
    q = np.ones(4200, np.int64)
    q[at] = 501
    b = Batch(41, dtype, 32, 1, 32, 4, rng.integers(0, 6, len(q)), q, tail=2)
    t = b.device()
    out, lse = torch.full_like(t["q"], 7.0), torch.full(t["q"].shape[:2], 7.0, device="cuda")
    for hints in (True, False):
        check_attention(*run(b, dict(t, out=out, lse=lse), hints=hints), b)
    assert bool((out[:, int(b.cu[-1]):] == 7).all()) and bool((lse[:, int(b.cu[-1]):] == 7).all())
    check_weights(b, 0.5)
