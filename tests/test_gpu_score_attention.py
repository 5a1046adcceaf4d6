"""mvr_paged_attention_scored on the GPU against softmax attention in 64 bits, at the sizes and rules where it can go
wrong: caps below and far above the scores, windows of one key, documents, prefixes, rows that see nothing, one token to
thousands, pages that end inside a chunk, every head dimension and dtype, split and unsplit keys, strides, stale hints,
values that are not finite, graphs, streams."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_score as S  # noqa: E402
from score_reference import Batch, check_attention  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


def run(batch, t=None, hints=True, **kw):
    t = t or batch.device()
    if hints:
        kw = dict(dict(seq_lens_host=batch.seq_lens, cu_q_lens_host=batch.cu, sum_seq_lens=int(batch.seq_lens.sum())), **kw)
    got = S.paged_attention_scored(**t, **{**batch.rules(), **kw})
    torch.cuda.synchronize()
    return got


def check(batch, note="", scale=None, **kw):
    check_attention(*run(batch, **(dict(kw, scale=scale) if scale else kw)), batch, scale=scale, note=note)


RULES = {  # of requests of up to 150 + 12 tokens
    "plain": dict(),
    "cap": dict(cap=3.0),
    "wide cap": dict(cap=50.0),
    "slopes": dict(slopes=True),
    "window": dict(window=20),
    "documents": dict(first_keys=[0, 0, 5, 5, 5, 9, 9, 140, 140, 0, 160, 161, 150]),
    "prefix": dict(prefix=[6, 1, 155]),
    "all": dict(cap=4.0, slopes=True, window=33, first_keys=[0, 3, 3, 12, 150, 151, 0], prefix=[7, 0, 500]),
}


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_head_dim_and_rule(dtype, d, page, rules):
    check(Batch(d + page, dtype, 6, 2, d, page, [0, 13, 150], [7, 1, 12], **RULES[rules]))


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 16, 24, 32, 48, 100])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_page_sizes(dtype, page):
    for q in ([3, 9, 1, 17], [1, 1, 1, 1], [130, 2, 70, 33]):
        check(Batch(page, dtype, 8, 2, 128, page, [1, 77, 130, 15], q, cap=30.0, slopes=True, window=90))


@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 130, 257, 600])
@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (F16, 14, 2, 64), (F32, 6, 2, 128), (F16, 3, 3, 128)])
def test_new_tokens(dtype, hq, hkv, d, new):
    """Rows per KV head from 1 to thousands: every row tile."""
    rng = np.random.default_rng(new)
    for rules in (dict(), dict(cap=20.0, window=70), dict(slopes=True, prefix=[100, 9]),
                  dict(first_keys=rng.integers(0, 45 + new, new + max(1, new // 3)))):
        check(Batch(new, dtype, hq, hkv, d, 16, [45, 200], [new, max(1, new // 3)], **rules), note=str(sorted(rules)))


@pytest.mark.parametrize("cached", [0, 1, 14, 15, 16, 17, 30, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_context_lengths(dtype, cached):
    check(Batch(cached, dtype, 4, 2, 64, 16, [cached], [1], cap=30.0))
    check(Batch(cached, dtype, 4, 2, 64, 16, [cached, 3], [70, 1], slopes=True))


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 65, 200, 1 << 30, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 90])
def test_windows(window, new):
    for dtype in (F16, F32):
        check(Batch(window % 1000, dtype, 8, 2, 128, 16, [300, 5], [new, 1], window=window))


@pytest.mark.parametrize("cap", [1e-3, 0.5, 5.0, 1e6])
def test_caps(cap):
    """From caps that flatten every score to ones that no score comes near."""
    for dtype in (F16, F32):
        check(Batch(7, dtype, 8, 2, 128, 16, [300, 5], [1, 60], cap=cap, q_std=6.0))


def test_scale_and_far_keys():
    b = Batch(8, F32, 4, 1, 64, 16, [200], [3], slopes=True, cap=2.0)
    check(b, scale=0.31)
    # Slopes over a long context: far keys count nothing, and distances are exact.
    check(Batch(9, F16, 4, 1, 64, 16, [70000], [2], slopes=True))


def test_rows_that_see_nothing():
    """A first key past the row's slot: output 0 and log-sum-exp -infinity, also where every row of a call is so, and
    where the keys are split."""
    for dtype in (F16, F32):
        for cached, new in (([40, 2000], [5, 3]), ([10, 300], [100, 90])):
            tokens = sum(new)
            some = Batch(3, dtype, 8, 2, 128, 16, cached, new, first_keys=[0, 10 ** 6, 2, 10 ** 6, 2 ** 31 - 1])
            out, lse = run(some)
            check_attention(out, lse, some)
            assert bool((lse[:, 1] == -float("inf")).all()) and not out[:, 1].any()
            none = Batch(3, dtype, 8, 2, 128, 16, cached, new, first_keys=[10 ** 6])
            out, lse = run(none)
            assert not out.any() and bool((lse == -float("inf")).all()) and lse.shape[1] == tokens


def test_empty_requests_and_padded_rows():
    """Requests without tokens, also all of them, and rows behind the last request left as they are."""
    for dtype in (F16, F32):
        for q in ([0, 4, 0, 0, 1, 0], [0, 90, 0, 2, 0, 0], [0] * 6):
            b = Batch(5, dtype, 8, 2, 64, 16, [30, 100, 2, 0, 700, 9], q, cap=30.0, tail=3)
            t = b.device()
            out, lse = torch.full_like(t["q"], 7.0), torch.full(t["q"].shape[:2], 7.0, device="cuda")
            got = run(b, dict(t, out=out, lse=lse))
            if sum(q):
                check_attention(*got, b)
            assert bool((out[:, int(b.cu[-1]):] == 7).all()) and bool((lse[:, int(b.cu[-1]):] == 7).all())


def spoil(batch, keys, what, pool):
    for key in keys:
        getattr(batch, pool)[batch.table[0, key // batch.page], 0, :, key % batch.page] = what


@pytest.mark.parametrize("what", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("new", [1, 6, 80])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_values_that_are_not_finite(dtype, new, what):
    """In keys and values that some rows do not see they reach the other rows only; in places that no row sees, and in
    slots past the last token, nobody."""
    rules = dict(window=24, first_keys=[30, 60, 3, 61, 62, 0])
    for pool in ("key_pool", "value_pool"):
        b = Batch(11, dtype, 8, 2, 64, 16, [60], [new], **rules)
        spoil(b, [0, 2, 45, 59 + new // 2], what, pool)
        last = 60 + new
        getattr(b, pool)[b.table[0, (last - 1) // 16], 0, :, (last - 1) % 16 + 1:] = what
        check(b, note=pool)


def test_lse_is_not_wanted():
    b = Batch(2, F16, 8, 2, 128, 16, [100, 40], [1, 30])
    t = b.device()
    out = torch.empty_like(t["q"])
    S.make_scored_call(*t.values(), out, None, **b.rules())()
    torch.cuda.synchronize()
    check_attention(out, None, b)


def test_strides():
    """Token-major queries and outputs, heads cut from a wider tensor, an lse with a longer row."""
    for dtype in (F16, F32):
        for q in ([2, 5], [70, 3]):
            b = Batch(13, dtype, 8, 2, 128, 16, [70, 300], q, cap=30.0, slopes=True)
            t = b.device()
            wide = torch.randn(b.tokens, 12, 128).to(dtype).cuda()
            wide[:, 2:10] = t["q"].transpose(0, 1)
            out = torch.zeros_like(wide)
            lse = torch.zeros(8, b.tokens + 5, device="cuda")
            run(b, dict(t, q=wide[:, 2:10].transpose(0, 1), out=out[:, 2:10].transpose(0, 1), lse=lse[:, :b.tokens]))
            check_attention(out[:, 2:10].transpose(0, 1), lse[:, :b.tokens], b)
            assert not out[:, :2].any() and not out[:, 10:].any() and not lse[:, b.tokens:].any()


def test_split_keys_and_workspaces():
    """Long contexts of few rows in as many parts as their workspace allows, down to none, and without hints."""
    for dtype in (F16, F32):
        for rules in (dict(cap=30.0), dict(slopes=True, window=3000), dict(first_keys=[4000, 0, 6000])):
            b = Batch(17, dtype, 4, 1, 128, 16, [7000], [3], **rules)
            want = run(b)
            check_attention(*want, b, note=str(rules))
            for workspace in (256, 1 << 14, 1 << 18, 1 << 26):
                got = run(b, workspace=torch.full((workspace,), 255, dtype=torch.uint8, device="cuda"))
                check_attention(*got, b, note=f"{rules} {workspace}")
            check_attention(*run(b, hints=False), b, note="no hints")


def test_stale_hints():
    """Host tables of other lengths cost speed, not results."""
    for q in ([1, 1, 1], [40, 1, 90]):
        b = Batch(19, F16, 8, 2, 128, 16, [900, 20, 3000], q, cap=50.0)
        for seq, cu in ((b.seq_lens // 7 + 1, b.cu), (b.seq_lens * 0, b.cu * 0), (b.seq_lens * 3, b.cu * 3)):
            check_attention(*run(b, seq_lens_host=seq.astype(np.int32), cu_q_lens_host=cu.astype(np.int32), sum_seq_lens=0), b)


def test_lengths_above_their_bounds_are_clamped():
    """A device length above max_seq_len and a q_len above max_q_len: nothing outside is read or written."""
    b = Batch(21, F16, 8, 2, 64, 16, [64, 64], [2, 2])
    t = b.device()
    t["seq_lens"][1] = 10 ** 6
    t["cu_q_lens"] += torch.tensor([0, 0, 1000], dtype=torch.int32, device="cuda")
    out, lse = run(b, t, hints=False)
    check_attention(out[:, :2], lse[:, :2], Batch1(b))
    assert bool(torch.isfinite(out).all())


def Batch1(b):
    """The first request alone."""
    one = Batch(21, F16, 8, 2, 64, 16, [64, 64], [2, 2])
    one.q_lens, one.seq_lens, one.cu, one.queries = b.q_lens[:1], b.seq_lens[:1], b.cu[:2], b.queries[:, :2]
    return one


def test_one_request_without_tables():
    b = Batch(23, F32, 6, 2, 64, 16, [100], [4], cap=9.0)
    t = b.device()
    check_attention(*run(b, dict(t, seq_lens=None, cu_q_lens=None), hints=False), b)


def test_pools_past_32_bits():
    """Pages whose offsets pass 2^32 elements."""
    b = Batch(25, F16, 4, 2, 128, 16, [100, 40], [1, 40], cap=30.0)
    pages = (1 << 32) // (2 * 16 * 128) + 200
    t = b.device()
    for name in ("key_pool", "value_pool"):
        big = torch.empty((pages, 1, 2, 16, 128), dtype=F16, device="cuda")
        big[pages - b.num_pages:] = t[name]
        t[name] = big
    t["block_tables"] = t["block_tables"] + (pages - b.num_pages)
    check_attention(*run(b, t), b)


def test_many_requests():
    rng = np.random.default_rng(4)
    for dtype in (F16, F32):
        b = Batch(27, dtype, 8, 2, 64, 16, rng.integers(0, 400, 150), rng.integers(0, 5, 150), window=100, cap=20.0)
        check(b)


@pytest.mark.parametrize("q", [[1] * 70 + [200], [200] + [1] * 70, [1, 0, 1, 90, 0, 1, 1, 0, 1, 1], [1] * 30 + [33, 0, 0] + [2] * 40 + [64],
                               [0] * 63 + [128], [0] * 64 + [129], [5] + [0] * 200 + [64]])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_mixed_batches(group, q):
    """Prompts among single tokens and empty requests, where row tiles' places are packed by the tokens there are."""
    for dtype in (F16, F32):
        rng = np.random.default_rng(len(q) + group)
        b = Batch(31, dtype, 2 * group, 2, 64, 16, rng.integers(0, 300, len(q)), q, cap=20.0, tail=2)
        t = b.device()
        out, lse = torch.full_like(t["q"], 7.0), torch.full(t["q"].shape[:2], 7.0, device="cuda")
        check_attention(*run(b, dict(t, out=out, lse=lse)), b)
        assert bool((out[:, int(b.cu[-1]):] == 7).all()) and bool((lse[:, int(b.cu[-1]):] == 7).all())


def test_mixed_batch_of_thousands():
    rng = np.random.default_rng(8)
    for n in (4095, 4200):
        q = np.ones(n, np.int64)
        q[rng.integers(0, n, 3)] = 150
        q[rng.integers(0, n, 500)] = 0
        check(Batch(32, F16, 4, 1, 32, 4, rng.integers(0, 6, n), q))


def test_mixed_graph_replays():
    """A captured call whose prompt is another request's at each replay."""
    batches = [Batch(33, F16, 8, 2, 128, 16, [700] * 20, [1] * k + [150] + [1] * (19 - k), cap=30.0) for k in (3, 0, 19, 11)]
    t = batches[0].device()
    out, lse = torch.empty_like(t["q"]), torch.empty(t["q"].shape[:2], device="cuda")
    call = S.make_scored_call(*t.values(), out, lse, **batches[0].rules())
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    pages = t["block_tables"].shape[1]
    for b in batches + batches[::-1]:
        for name, x in b.device().items():
            if name == "block_tables":
                t[name][:, :min(pages, x.shape[1])] = x[:, :pages]
            else:
                t[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, lse, b)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_many_keys_far_below_one(dtype, new):
    """One key at e^18.75 of 200,000 others, which hold 0.14% of a row together and all of its output.

    F16 probabilities are off by 2^-25 at most where they are that small, the largest being 2^7 or more: 2^-32 of the sum
    for each key (2^-31, where both halves of one are cut); 2^-24 of the sum for each in 32 bits, of which the large key's
    own adds 2^-24 of the sum; then half a step of the output."""
    n, page, d = 200_000, 16, 32
    pages = n // page
    q = torch.zeros((2, new, d), dtype=dtype, device="cuda")
    q[..., 0] = 8.0
    keys = torch.zeros((pages, 1, 1, page, d), dtype=dtype, device="cuda")
    values = torch.ones_like(keys)
    keys[0, 0, 0, 0, 0], values[0, 0, 0, 0] = 18.75 / 8, 0.0
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = S.paged_attention_scored(q, keys, values, table, ints(n), ints(0, new), max_q_len=new, max_seq_len=n, scale=1.0)
    torch.cuda.synchronize()
    others = torch.arange(n - new, n, dtype=torch.float64) * np.exp(-18.75)
    want = (others / (1 + others))[None, :, None]
    u = 2.0 ** -11 if dtype == F16 else 2.0 ** -24
    tol = n * (2.0 ** -31 if dtype == F16 else 0) + want * (u + 2.0 ** -16) + 2.0 ** -24
    assert bool(((out.double().cpu() - want).abs() <= tol).all()), float(((out.double().cpu() - want).abs() / tol).max())
    within = (lse.double().cpu() - (18.75 + torch.log1p(others))).abs()
    assert float(within.max()) <= 2.0 ** -18


def test_graph_replays():
    """Captured calls, split and not, replayed with changed lengths and values between, with eager work in between."""
    for cached, q, rules in (([3000], [1], dict(cap=30.0)), ([200, 90], [70, 4], dict(slopes=True, window=50))):
        b = Batch(29, F16, 8, 2, 128, 16, cached, q, **rules)
        t = b.device()
        out, lse = torch.empty_like(t["q"]), torch.empty(t["q"].shape[:2], device="cuda")
        call = S.make_scored_call(*t.values(), out, lse, **b.rules())
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for k in range(4):
            b.queries = (b.queries * -0.9).to(F16)
            t["q"].copy_(b.queries)
            b.seq_lens = b.seq_lens - k
            t["seq_lens"].copy_(torch.from_numpy(b.seq_lens))
            out.fill_(9)
            graph.replay()
            torch.cuda.synchronize()
            check_attention(out, lse, b, note=f"replay {k}")
            eager = run(b, t)
            assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


def test_streams_and_repeats():
    """On a stream of its own, and the same bits every time."""
    b = Batch(31, F16, 8, 2, 128, 16, [2500, 40], [1, 6], cap=50.0)
    t = b.device()
    want = run(b, t)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        out, lse = S.paged_attention_scored(**t, **b.rules(), seq_lens_host=b.seq_lens, cu_q_lens_host=b.cu,
                                            sum_seq_lens=int(b.seq_lens.sum()), stream=stream)
        stream.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_refuses_tensors_that_do_not_fit():
    b = Batch(33, F16, 8, 2, 64, 16, [20], [2])
    t, rules = b.device(), b.rules()
    for name, bad in (("slopes", torch.ones(7, device="cuda")), ("first_keys", torch.zeros(3, dtype=torch.int32, device="cuda")),
                      ("prefix_lens", torch.zeros(2, dtype=torch.int32, device="cuda")), ("cap", -1.0), ("cap", float("nan")),
                      ("window", -1), ("slopes", torch.ones(8)), ("lse", torch.ones(8, 3, device="cuda")),
                      ("lse", torch.ones(8, 2, dtype=F16, device="cuda")), ("max_q_len", 0)):
        with pytest.raises(M.MvrError):
            S.paged_attention_scored(**t, **{**rules, name: bad})
