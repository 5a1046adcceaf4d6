"""Calls on scores whose device tables hold numbers at the ends of their type: nothing is read outside a block table's row,
and what the tables still say is computed."""
import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402
from score_reference import Batch, check_attention  # noqa: E402
from test_gpu_score_attention import run  # noqa: E402
from test_gpu_score_evict import Cache, check as check_selection  # noqa: E402
from test_gpu_score_weights import check as check_weights  # noqa: E402

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


def broken(dtype, cached, q, **rules):
    """Requests shorter than their queries among whole ones, first keys and prefixes at the ends of their type."""
    ends = dict(first_keys=[2 ** 31 - 1, 0, -2 ** 31, 1, 2 ** 31 - 1, -5], prefix=[-2 ** 31, 2 ** 31 - 1, 1, -1, 0])
    return Batch(22, dtype, 16, 2, 64, 16, cached, q, **{**ends, **rules})


@pytest.mark.parametrize("window", [0, 1, 2 ** 31 - 1])
@pytest.mark.parametrize("q", [[5, 3, 5, 7, 2], [45, 40, 5, 70, 60]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_row_ranges_at_the_ends_of_32_bits(dtype, q, window):
    """Slots below 0 see no key, or a prefix; no difference of a slot and a table's number wraps."""
    for cached in ([-3, 60, -4, 90, -1], [-1, 200, 3, 0, 20]):
        b = broken(dtype, cached, q, window=window)
        check_attention(*run(b, hints=False), b, note=str(cached))
        check_weights(b, 0.5, note=str(cached))
        no_prefix = broken(dtype, cached, q, window=window, prefix=None)
        check_attention(*run(no_prefix, hints=False), no_prefix, note=str(cached))
        check_weights(no_prefix, 0.5, note=str(cached))


@pytest.mark.parametrize("seq_len", [0, -7, -2 ** 31])
@pytest.mark.parametrize("q", [[1, 1, 1], [3, 2, 70], [60, 90, 1]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_requests_of_length_0_with_query_tokens(dtype, q, seq_len):
    """A padded slot of a batch: its rows see nothing, which is an output of 0 and a log-sum-exp of -infinity; nobody's
    weights change for it."""
    for rules in (dict(cap=20.0), dict(prefix=[9, 2000, 5]), dict(slopes=True, window=40)):
        b = Batch(23, dtype, 16, 2, 64, 16, [100, -q[1], 2000], q, **rules)
        t = b.device()
        t["seq_lens"][1] = seq_len
        out, lse = torch.full_like(t["q"], 7.0), torch.full(t["q"].shape[:2], 7.0, device="cuda")
        check_attention(*run(b, dict(t, out=out, lse=lse), hints=False), b, note=str(rules))
        rows = slice(q[0], q[0] + q[1])
        assert not out[:, rows].any() and bool((lse[:, rows] == -float("inf")).all())
        check_weights(b, 0.5, note=str(rules))
