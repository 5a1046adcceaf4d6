"""How exact the calls on scores are where a step of the kernels mixes small scores and large ones."""
import math

import pytest

torch = pytest.importorskip("torch")

import mvr_score as S  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


@pytest.mark.parametrize("new", [1, 8, 80])
@pytest.mark.parametrize("cap", [300.0, 1e4, 1e5])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_small_scores_beside_one_past_the_cap(dtype, cap, new):
    """One key at minus twice the cap, which counts nothing, among scores up to 1, which are as exact as without it.

    A query holds one number and a key another, so products and their sums are exact; a capped score is off by 2^-22 of
    itself, at most 1: the polynomial and its coefficients; its distance to the running maximum, at most 16 log2 units, by
    2^-24 of it, 2^-20.5 of a probability, whose exponential adds 2^-22; the sums of n terms n 2^-24."""
    n, d, group = 70 + new, 64, 8
    gen = torch.Generator().manual_seed(int(cap) + new)
    scores = (torch.rand(n, generator=gen, dtype=torch.float64) * 2 - 1).to(dtype)
    scores[33] = -2 * cap
    q, keys = torch.zeros((group, new, d), dtype=dtype), torch.zeros((n, d), dtype=dtype)
    q[..., 5], keys[:, 5] = 8.0, scores / 8
    scores = keys[:, 5].double() * 8
    capped = cap * torch.tanh(scores / cap)
    pool = torch.zeros((8, 1, 1, 32, d), dtype=dtype)
    pool.view(-1, d)[:n] = keys
    values = torch.randn(pool.shape, generator=gen).to(dtype)
    seen = torch.arange(n) <= torch.arange(n - new, n)[:, None]
    x = capped.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[:, None])
    table = torch.arange(8, dtype=torch.int32)[None].cuda()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    args = (table, ints(n), ints(0, new))
    rules = dict(max_q_len=new, max_seq_len=n, scale=1.0, cap=cap)
    out, got = S.paged_attention_scored(q.cuda(), pool.cuda(), values.cuda(), *args, **rules)
    tol = 2.0 ** -22 + 2.0 ** -20.5 + 2.0 ** -22 + n * 2.0 ** -24
    off = (got.cpu().double() - lse).abs() - 2.0 ** -22 * lse.abs()
    assert float(off.max()) <= tol, f"lse: {float(off.max()) / tol:.3g} times the tolerance"
    want = p @ values.view(-1, d)[:n].double()
    size = p @ values.view(-1, d)[:n].double().abs()
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24  # (F16: of the probabilities, and of the output)
    off = (out.cpu().double() - want).abs() / (2 * tol * size + u * (size + want.abs()) + 2.0 ** -24)
    assert float(off.max()) <= 1, f"out: {float(off.max()):.3g} times the tolerance"
    weights = S.attention_weights(q.cuda(), lse.float().expand(group, -1).contiguous().cuda(), pool.cuda(),
                                  torch.zeros((8, 1, 32)).cuda(), *args, decay=0.0, **rules).cpu().view(-1)[:n].double()
    want = group * p.sum(0)
    off = (weights - want).abs() / (want * (tol + 2.0 ** -22 * float(lse.abs().max()) + group * new * 2.0 ** -24) + 1e-30)
    assert float(off.max()) <= 1, f"weights: {float(off.max()):.3g} times the tolerance"
