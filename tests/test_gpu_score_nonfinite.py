"""Infinities and NaN in keys under a cap, and in values in the middle of a long context, where the kernels look at no mask."""
import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402
from score_reference import Batch, check_attention, within  # noqa: E402
from test_gpu_score_attention import run  # noqa: E402
from test_gpu_score_weights import inputs  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


def spoil(batch, keys, what, pool, dims=slice(None)):
    for key in keys:
        getattr(batch, pool)[batch.table[0, key // batch.page], 0, :, key % batch.page, dims] = what


@pytest.mark.parametrize("cap", [2.0, 30.0, 1e6])
@pytest.mark.parametrize("what,dims", [(INF, 5), (-INF, 5), (NAN, 5), (NAN, slice(None))])
@pytest.mark.parametrize("new", [1, 6, 80])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_keys_under_a_cap(dtype, new, what, dims, cap):
    """An infinite score is the cap or minus it, a NaN reaches the rows that see its key; others, and slots past the last
    token, nobody."""
    rules = dict(first_keys=[30, 350, 3, 351, 352, 0], cap=cap)
    b = Batch(61, dtype, 8, 2, 64, 16, [350], [new], **rules)
    spoil(b, [0, 2, 100, 349 + new // 2], what, "key_pool", dims)
    last = 350 + new
    b.key_pool[b.table[0, (last - 1) // 16], 0, :, (last - 1) % 16 + 1:] = NAN
    check_attention(*run(b), b)
    clean = Batch(61, dtype, 8, 2, 64, 16, [350], [new], **rules)
    lse, t = inputs(clean)  # of finite scores
    want, tol = b.key_weights(lse)
    t["key_pool"].copy_(b.key_pool)
    S.attention_weights(**t, **b.rules())
    within(t["weights"].cpu(), want, tol)


@pytest.mark.parametrize("what", [INF, -INF, NAN])
@pytest.mark.parametrize("new", [1, 9, 80])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_values_amid_a_long_context(dtype, new, what):
    """In the spoiled elements the rows that see the key are not finite; everything else is what it is without them."""
    for rules in (dict(), dict(cap=30.0, slopes=True), dict(first_keys=[0, 900, 0, 640, 901])):
        b = Batch(62, dtype, 8, 2, 64, 16, [1500, 300], [new, 2], **rules)
        b.slopes = None if b.slopes is None else b.slopes * 1e-3
        want, tol, want_lse, lse_tol = b.attention()
        spoil(b, [300, 700], what, "value_pool", slice(8, 24))
        out, lse = run(b)
        within(lse, want_lse, lse_tol, "lse")
        seen = b.visible(0)[:, 700]
        hit = torch.zeros(want.shape, dtype=torch.bool)
        hit[:, :new, 8:24] = (seen | b.visible(0)[:, 300])[None, :, None]
        assert not bool(torch.isfinite(out.cpu()[hit]).any())
        within(out.cpu()[~hit], want[~hit], tol[~hit], "out")
