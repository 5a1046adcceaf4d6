"""Kernel variants that only large calls of selection and weights take: a selection's small blocks, and those for requests
around what LDS holds; weights whose wavefronts have keys of their own and go through many row tiles."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402
from score_reference import Batch  # noqa: E402
from test_gpu_score_evict import Cache, check as check_selection  # noqa: E402
from test_gpu_score_weights import check as check_weights  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


def compute_units():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("values", ["spread", "equal", "odd"])
def test_selections_of_many_blocks(values, page):
    """More blocks than two to a CU, of requests that four blocks to a CU hold in LDS."""
    lens = [300, 1, 64, 257, 0, 128, 33, 299, 2, 150, 65, 200, 7, 255, 256, 90, 31]
    keep = [100, 1, 63, 200, 5, 20, 32, 8, 1, 200, 64, 199, 9, 1, 255, 45, 0]
    layers = -(-(2 * compute_units() + 1) // (len(lens) * 8)) + 1
    check_selection(Cache(51, lens, keep, layers=layers, hkv=8, page=page, recent=1, values=values))


@pytest.mark.parametrize("page", [16, 5])
def test_selections_of_many_blocks_cut_again(page):
    lens = [140, 129, 200, 128, 131] * 14
    check_selection(Cache(52, lens, 128, layers=1, hkv=8, page=page, kept=[128, 128, 150, 128, 128] * 14, past=777, recent=16,
                          first=4, values="odd"))


@pytest.mark.parametrize("n", [8127, 8128, 8129, 17407, 17408, 17409])
@pytest.mark.parametrize("page", [16, 5])
def test_selections_around_what_lds_holds(page, n):
    """In few blocks, and in many of which one is as long."""
    check_selection(Cache(n, [n], n // 3, page=page, recent=100, values="odd"))
    lens = [n] + [40] * (2 * compute_units() // 2)
    check_selection(Cache(n, lens, [n // 3] + [30] * (len(lens) - 1), page=page, recent=10, values="spread"))


@pytest.mark.parametrize("rules", [dict(), dict(cap=50.0), dict(cap=3.0, slopes=True, window=700), dict(prefix=[4000, 100, 9000, 0]),
                                   dict(first_keys=np.arange(0, 4200, 13))], ids=["plain", "cap", "window", "prefix", "documents"])
@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(F16, 28, 4, 128, 16), (F32, 12, 4, 64, 24), (F16, 16, 16, 64, 5)])
def test_weights_of_many_rows_and_keys(dtype, hq, hkv, d, page, rules):
    """Over 32 rows, and key units that give every SIMD a wavefront: none of them share keys."""
    cached, q = [6000, 3500, 6100, 5000], [33, 70, 1, 40]
    assert hkv * len(q) * -(-6101 // 64) >= 4 * compute_units() and hq // hkv * max(q) > 32
    check_weights(Batch(53, dtype, hq, hkv, d, page, cached, q, **rules), 0.5)
