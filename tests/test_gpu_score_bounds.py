"""Calls on scores whose device tables hold numbers at the ends of their type: nothing is read outside a block table's row,
and what the tables still say is computed."""
import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402
from test_gpu_score_evict import Cache, check as check_selection  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


@pytest.mark.parametrize("kept", [1 << 20, 2 ** 31 - 4096, 2 ** 31 - 2, 2 ** 31 - 1])
@pytest.mark.parametrize("lens,keep,page", [([300, 70], 400, 16), ([300, 70], [100, 40], 5), ([20000], 4000, 16), ([20000], 20000, 5)])
def test_kept_lengths_above_the_request(kept, lens, keep, page):
    """All positions are known, whether the request is cut, or too long for LDS, or neither."""
    c = Cache(21, lens, keep, hkv=1, page=page, kept=lens, past=50, recent=8)
    t = c.device()
    t["kept_lens"].fill_(kept)
    check_selection(c, t)
