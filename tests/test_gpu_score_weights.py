"""mvr_attention_weights on the GPU against sums of probabilities in 64 bits: every head dimension and dtype, rows from one
to hundreds, ragged lengths and pages, decays, fresh slots, rows that see nothing, values that are not finite."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_score as S  # noqa: E402
from score_reference import Batch, within  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


def inputs(b):
    """The log-sum-exps in 32 bits, and the call's positional tensors."""
    lse = b.attention()[2].float()
    t = b.device()
    return lse, dict(q=t["q"], lse=lse.cuda(), key_pool=t["key_pool"], weights=b.weights.cuda(),
                     block_tables=t["block_tables"], seq_lens=t["seq_lens"], cu_q_lens=t["cu_q_lens"])


def check(b, decay=1.0, fresh=None, note=""):
    lse, t = inputs(b)
    want, tol = b.key_weights(lse, decay, fresh)
    if fresh is not None:
        t["fresh_from"] = torch.tensor(fresh, dtype=torch.int32, device="cuda")
    S.attention_weights(**t, **b.rules(), decay=decay)
    torch.cuda.synchronize()
    got = t["weights"].cpu()
    same = tol == 0  # slots of no request, or left alone
    assert torch.equal(got[same].view(torch.int32), want[same].float().view(torch.int32)), note
    return within(got, want, tol, note)


RULES = [dict(), dict(cap=3.0), dict(cap=50.0, slopes=True), dict(window=20), dict(prefix=[6, 1, 155]),
         dict(first_keys=[0, 0, 5, 5, 5, 9, 9, 140, 140, 0, 160, 161, 150]),
         dict(cap=4.0, slopes=True, window=33, first_keys=[0, 3, 3, 12, 150, 151, 0], prefix=[7, 0, 500])]


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_head_dim_and_rule(dtype, d, page):
    for k, rules in enumerate(RULES):
        check(Batch(d + page, dtype, 6, 2, d, page, [0, 13, 150], [7, 1, 12], **rules), note=str(rules))


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 24, 48, 100])
def test_page_sizes(page):
    for dtype in (F16, F32):
        check(Batch(page, dtype, 8, 2, 128, page, [1, 77, 130, 15], [3, 9, 1, 17], cap=30.0))


@pytest.mark.parametrize("new", [1, 2, 3, 5, 8, 16, 17, 33, 64, 130, 300])
@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (F16, 14, 2, 64), (F32, 6, 2, 128), (F32, 3, 3, 32)])
def test_new_tokens(dtype, hq, hkv, d, new):
    for rules in (dict(), dict(cap=20.0, window=70), dict(slopes=True, prefix=[100, 9])):
        check(Batch(new, dtype, hq, hkv, d, 16, [45, 200], [new, max(1, new // 3)], **rules), note=str(rules))


@pytest.mark.parametrize("cached", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 256, 257, 3000])
def test_context_lengths(cached):
    for dtype in (F16, F32):
        check(Batch(cached, dtype, 4, 2, 64, 16, [cached, 3], [1, 2], cap=30.0))


@pytest.mark.parametrize("decay", [0.0, 0.25, 1.0, 2.0])
def test_decay_and_fresh_slots(decay):
    for dtype in (F16, F32):
        check(b := Batch(3, dtype, 8, 2, 64, 16, [100, 20, 5], [1, 7, 3]), decay)
        check(b, decay, fresh=[0, 20, 1000])
        check(b, decay, fresh=[101, 3, 7])
        check(Batch(3, dtype, 8, 2, 64, 16, [100, 200, 5], [1, 7, 3], window=9), decay)


def test_what_was_there_is_not_read():
    """NaN in fresh slots, in every slot with a decay of 0, past the last token and in other pages: none comes back."""
    b = Batch(4, F16, 8, 2, 64, 16, [100], [3])
    lse, t = inputs(b)
    n = int(b.seq_lens[0])
    for decay in (1.0, 0.0):
        b.weights[:] = float("nan")
        if decay:
            for j in range(n - 3):
                b.weights[b.table[0, j // 16], :, j % 16] = 0.5
        t["weights"].copy_(b.weights)
        want, tol = b.key_weights(lse, decay)
        S.attention_weights(**t, **b.rules(), decay=decay)
        ids = b.ids(0)
        flat = lambda x: x.cpu()[ids].permute(1, 0, 2).reshape(2, -1)  # noqa: E731
        within(flat(t["weights"])[:, :n], flat(want)[:, :n], flat(tol)[:, :n])
        assert bool(flat(t["weights"])[:, n:].isnan().all())


def test_the_sum_of_all_weights_is_the_number_of_rows():
    """Of a fresh prompt, by the log-sum-exps that the attention call gives."""
    for dtype in (F16, F32):
        b = Batch(6, dtype, 8, 2, 128, 16, [0, 0], [300, 77], cap=20.0, slopes=True)
        t = b.device()
        out, lse = S.paged_attention_scored(**t, **b.rules())
        weights = torch.zeros_like(b.weights).cuda()
        S.attention_weights(t["q"], lse, t["key_pool"], weights, t["block_tables"], t["seq_lens"], t["cu_q_lens"], **b.rules())
        per_head = weights.double().sum((0, 2)).cpu()
        # A row's weights add up to 1 but for 32-bit scores on both sides: 2^-24 of (64 + 128) products of about 10 each.
        assert bool(((per_head - 4 * 377).abs() <= 4 * 377 * 2.0 ** -24 * 192 * 10).all()), per_head


def test_the_last_tokens_of_a_prompt():
    """q, lse, first keys and starts of the last 5 tokens alone; all the prompt's slots are fresh."""
    b = Batch(8, F16, 8, 2, 64, 16, [0, 0], [90, 40], first_keys=np.arange(130) // 30)
    last = Batch(8, F16, 8, 2, 64, 16, [85, 35], [5, 5])
    pick = np.concatenate([np.arange(85, 90), np.arange(125, 130)])
    last.queries, last.first_keys, last.key_pool, last.table = b.queries[:, pick], b.first_keys[pick], b.key_pool, b.table
    check(last, fresh=[0, 0])


def test_rows_that_see_nothing_and_keys_that_nobody_sees():
    for dtype in (F16, F32):
        check(Batch(9, dtype, 8, 2, 64, 16, [40, 2000], [5, 3], first_keys=[0, 10 ** 6, 2, 10 ** 6, 2 ** 31 - 1]), 0.5)
        check(Batch(9, dtype, 8, 2, 64, 16, [40, 2000], [5, 3], first_keys=[10 ** 6]), 0.5)


def test_requests_without_tokens_are_left_alone():
    b = Batch(10, F16, 8, 2, 64, 16, [50, 60, 70], [0, 2, 0], tail=4)
    check(b, 0.5)
    empty = Batch(10, F16, 8, 2, 64, 16, [50, 60], [0, 0])
    lse, t = inputs(empty)
    S.attention_weights(**t, **empty.rules(), decay=0.5)
    assert torch.equal(t["weights"].cpu(), empty.weights)


@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_keys_that_are_not_finite(what):
    """In keys that some rows do not see, and past the last token: only their own weights are touched by them."""
    for dtype in (F16, F32):
        b = Batch(11, dtype, 8, 2, 64, 16, [60], [6], window=24)
        lse, t = inputs(b)
        clean, tol = b.key_weights(lse)
        for key in (0, 20, 64):
            b.key_pool[b.table[0, key // 16], 0, :, key % 16] = what
        b.key_pool[b.table[0, 65 // 16], 0, :, 2:] = what
        t["key_pool"].copy_(b.key_pool)
        S.attention_weights(**t, **b.rules())
        got = t["weights"].cpu()
        seen = torch.ones_like(clean, dtype=torch.bool)
        seen[b.table[0, 64 // 16], :, 64 % 16] = False
        within(got[seen], clean[seen], tol[seen])


def test_graph_replays_and_streams():
    b = Batch(12, F16, 8, 2, 128, 16, [900, 33], [1, 20], cap=30.0)
    lse, t = inputs(b)
    call = S.make_weights_call(*t.values(), **b.rules(), decay=0.5)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    stream = torch.cuda.Stream()
    for k in range(4):
        t["weights"].copy_(b.weights * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        replayed = t["weights"].clone()
        t["weights"].copy_(b.weights * (k + 1))
        stream.wait_stream(torch.cuda.current_stream())
        S.attention_weights(**t, **b.rules(), decay=0.5, stream=stream)
        stream.synchronize()
        assert torch.equal(replayed, t["weights"])


def test_refuses_tensors_that_do_not_fit():
    b = Batch(13, F16, 8, 2, 64, 16, [20], [2])
    lse, t = inputs(b)
    for name, bad in (("weights", t["weights"][:-1]), ("weights", t["weights"].half()), ("weights", None), ("lse", None),
                      ("decay", -1.0), ("decay", float("inf")), ("q", t["q"].float()), ("weights", t["weights"].cpu()),
                      ("fresh_from", torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(M.MvrError):
            S.attention_weights(**{**t, **b.rules(), name: bad})
