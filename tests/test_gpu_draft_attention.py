"""mvr_paged_attention_tree on the GPU against softmax attention in 64 bits, at the sizes and masks where it can go
wrong: trees of one token to hundreds, empty requests and rows, pages that end inside a chunk, every head dimension and
dtype, split and unsplit keys, strides, stale hints, values that are not finite, graphs, streams."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_draft as D  # noqa: E402
from draft_reference import Batch, check_attention  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    D.load_library()


def run(batch, t=None, hints=True, **kw):
    t = t or batch.device()
    out = t.pop("out", None)
    if hints:
        kw.setdefault("seq_lens_host", batch.seq_lens)
        kw.setdefault("cu_q_lens_host", batch.cu)
        kw.setdefault("sum_seq_lens", int(batch.seq_lens.sum()))
    got = D.paged_attention_tree(out=out, max_q_len=batch.max_q, max_seq_len=batch.max_len, **t, **kw)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_head_dim(dtype, d, page):
    check_attention(run(b := Batch(d + page, dtype, 6, 2, d, page, [0, 13, 150], [7, 1, 12])), b)


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 16, 24, 32, 48, 100])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_page_sizes(dtype, page):
    check_attention(run(b := Batch(page, dtype, 8, 2, 128, page, [1, 77, 130, 15], [3, 9, 1, 17])), b)


@pytest.mark.parametrize("nodes", [1, 2, 4, 5, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 96, 130, 257])
@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (F16, 14, 2, 64), (F32, 6, 2, 128)])
def test_tree_sizes(dtype, hq, hkv, d, nodes):
    """Grouped rows from 3 to over a thousand: every row tile, and mask rows of up to 9 words."""
    for masks in ("tree", "random"):
        check_attention(run(b := Batch(nodes, dtype, hq, hkv, d, 16, [45, 200], [nodes, max(1, nodes // 3)], masks)), b,
                        note=masks)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (64, 1), (1, 1), (10, 2), (24, 8)])
def test_head_layouts(dtype, hq, hkv):
    """A KV head for every query head, one for all of them, and groups between."""
    for nodes in ([3, 1], [40, 130]):
        check_attention(run(b := Batch(hq + hkv, dtype, hq, hkv, 64, 16, [70, 200], nodes, "tree")), b, note=str(nodes))


@pytest.mark.parametrize("dtype,cached,nodes", [(F16, [200_000, 3], [4, 2]), (F32, [70_001], [1]), (F16, [0, 900], [1100, 5]),
                                                (F16, [120_000], [90])])
def test_long(dtype, cached, nodes):
    """Contexts of more keys than the most parts of the shortest units hold, and masks of tens of words."""
    check_attention(run(b := Batch(sum(nodes), dtype, 4, 2, 64, 16, cached, nodes, "tree")), b)


@pytest.mark.parametrize("cached", [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_where_the_drafts_begin(dtype, cached):
    """The first draft anywhere in a chunk or key tile: every shift of the mask words."""
    for nodes in (1, 20, 40, 70):
        check_attention(run(b := Batch(cached + nodes, dtype, 4, 2, 64, 16, [cached], [nodes])), b, note=str(nodes))


@pytest.mark.parametrize("dtype,page", [(F16, 16), (F16, 24), (F32, 16), (F32, 5)])
@pytest.mark.parametrize("cached,nodes", [([3000], [8]), ([1500, 40, 2900], [20, 64, 3]), ([2048] * 4, [33] * 4)])
def test_split_keys(dtype, page, cached, nodes):
    """Long contexts over few heads: parts of the keys on several blocks.  Without a workspace, and with half of it,
    the same call runs with fewer parts."""
    b = Batch(sum(nodes), dtype, 8, 2, 128, page, cached, nodes, "tree")
    t = b.device()
    check_attention(run(b, dict(t)), b, note="whole workspace")
    a = D.make_tree_call(**t, out=torch.empty_like(t["q"]), max_q_len=b.max_q, max_seq_len=b.max_len,
                         seq_lens_host=b.seq_lens, cu_q_lens_host=b.cu, sum_seq_lens=int(b.seq_lens.sum()))
    need = a.args.workspace_bytes
    assert need > 0
    for size in (need // 2, 0):
        ws = torch.full((max(size, 1) + 4096,), 255, dtype=torch.uint8, device="cuda")
        got = run(b, dict(t), workspace=ws[:size] if size else ws[:0])
        check_attention(got, b, note=f"{size} bytes")
        assert bool((ws[size:] == 255).all()), "wrote behind its workspace"


def test_no_host_tables():
    b = Batch(3, F16, 8, 2, 128, 16, [700, 0, 30, 1900], [5, 0, 33, 12])
    check_attention(run(b, hints=False), b)


def test_one_request_without_tables():
    b = Batch(4, F16, 8, 2, 64, 16, [333], [9])
    t = b.device()
    t["seq_lens"] = t["cu_q_lens"] = None
    check_attention(run(b, t, hints=False), b)


@pytest.mark.parametrize("stale", ["short", "long", "other trees"])
def test_stale_hints_cost_no_rows(stale):
    """Host tables that are not the device's: longer or shorter contexts, other trees; every row is still computed."""
    b = Batch(5, F16, 8, 2, 128, 16, [900, 2500, 64, 1700], [12, 30, 1, 8])
    lens = {"short": b.q_lens + 1, "long": np.full(4, b.max_len, np.int32), "other trees": b.seq_lens}[stale]
    cu = np.array([0, 1, 2, 3, 4], np.int32) if stale == "other trees" else b.cu
    got = run(b, seq_lens_host=lens.astype(np.int32), cu_q_lens_host=cu, sum_seq_lens=int(lens.sum()))
    check_attention(got, b)


def test_stale_hints_that_plan_too_few_parts():
    """Hints of one long request where all are long: more parts than the workspace was planned for, so nothing is split
    and the blocks go on to the tiles that the grid has none for."""
    b = Batch(50, F16, 8, 2, 128, 16, [2500, 2400, 2300, 2600], [12, 30, 1, 8], "tree")
    lens = np.array([40, 40, 2301, 40], np.int32)
    a = D.make_tree_call(**b.device(), out=b.device()["q"], max_q_len=b.max_q, max_seq_len=b.max_len,
                         seq_lens_host=lens, cu_q_lens_host=b.cu, sum_seq_lens=int(lens.sum()))
    assert a.args.workspace_bytes > 0
    check_attention(run(b, seq_lens_host=lens, sum_seq_lens=int(lens.sum())), b)
    check_attention(run(b, hints=False, sum_seq_lens=int(b.seq_lens.sum())), b, note="the sum alone")


def test_thousands_of_empty_requests():
    """A padded batch of 3,000, three of them with drafts; over 2^16 row tiles in the grid of the merge."""
    q, cached = np.zeros(3000, np.int64), np.zeros(3000, np.int64)
    for s, n, c in ((5, 60, 1500), (1777, 3, 2000), (2999, 1, 700)):
        q[s], cached[s] = n, c
    b = Batch(51, F16, 16, 2, 64, 16, cached, q, "tree")
    check_attention(run(b), b)
    check_attention(run(b, hints=False), b)


def test_many_requests():
    """More requests than one scan holds, a third of them empty."""
    rng = np.random.default_rng(6)
    q = rng.integers(0, 7, 150)
    b = Batch(6, F16, 4, 2, 64, 16, rng.integers(0, 90, 150), q, "tree")
    check_attention(run(b), b)
    check_attention(run(b, hints=False), b)
    few = Batch(7, F16, 2, 1, 64, 16, [0] * 100 + [3000], [0] * 100 + [4], "tree")  # split: found behind empty ones
    check_attention(run(few), few)


@pytest.mark.parametrize("hkv", [1, 3, 8])
@pytest.mark.parametrize("requests", [63, 64, 65, 150])
def test_requests_of_all_lengths(requests, hkv):
    """More blocks than CUs, which start by length: every request is found once, empty ones, equal ones and those of the
    last, shorter batch of 64 among them."""
    rng = np.random.default_rng(requests)
    nodes = rng.choice([0, 1, 3, 9], requests)
    b = Batch(requests, F16, 4 * hkv, hkv, 32, 16, rng.choice([0, 1, 30, 64, 200, 700], requests), nodes, "tree", tail=3)
    for hints in (True, False):
        t = b.device()
        t["out"] = torch.full_like(t["q"], 7.0)
        check_attention(out := run(b, t, hints, workspace=torch.empty(0, dtype=torch.uint8, device="cuda")), b,
                        note=f"hints {hints}")
        assert bool((out[:, int(b.cu[-1]):] == 7.0).all())


def test_rows_that_see_nothing_are_zero():
    """Masks without a bit: with a cached prefix the rows see it, without one they see nothing."""
    for dtype in (F16, F32):
        b = Batch(8, dtype, 8, 2, 128, 16, [0, 20, 0], [70, 5, 3], "none")
        got = run(b)
        check_attention(got, b)
        lo, hi = b.cu[1], b.cu[2]
        assert bool((got[:, :lo] == 0).all()) and bool((got[:, hi:] == 0).all()) and bool((got[:, lo:hi] != 0).any())
        b.bits[3, :2] = True  # one row of the first request sees two drafts
        check_attention(run(b), b)


def test_mask_bits_behind_the_drafts_count_for_nothing():
    b = Batch(9, F16, 4, 2, 64, 16, [30, 7], [33, 5], "tree", words=4)
    got = run(b)
    q_len = np.repeat(b.q_lens, b.q_lens)
    b.bits |= np.arange(b.bits.shape[1])[None, :] >= q_len[:, None]
    assert torch.equal(run(b), got)
    check_attention(got, b)


def test_rows_behind_the_last_request_stay():
    """A padded batch: more rows in q and out than the requests have, an empty request last."""
    b = Batch(10, F16, 8, 2, 128, 16, [40, 2000, 9], [6, 9, 0], tail=13)
    t = b.device()
    t["q"][:, int(b.cu[-1]):] = math.nan
    t["out"] = torch.full_like(t["q"], 7.0)
    got = run(b, t)
    check_attention(got, b)
    assert bool((got[:, int(b.cu[-1]):] == 7.0).all())


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("nodes", [6, 40])
def test_non_finite_drafts_reach_only_the_rows_that_see_them(dtype, page, nodes):
    """A NaN or an infinity in the K or V row of a draft: rows whose mask leaves the draft out are untouched by it."""
    for what, value in (("key", math.nan), ("value", math.nan), ("value", math.inf), ("value", -math.inf)):
        b = Batch(nodes, dtype, 8, 2, 128, page, [37, 0], [nodes, nodes], "tree")
        for request, slot in ((0, 2), (1, nodes - 1)):
            at = int(b.cached[request]) + slot
            pool = b.key_pool if what == "key" else b.value_pool
            pool[int(b.table[request, at // page]), 0, :, at % page, 3] = value
        # a NaN score reaches every dim of the row
        got = run(b)
        want = b.attention()[0]
        for request, slot in ((0, 2), (1, nodes - 1)):
            seen = torch.from_numpy(b.bits[b.cu[request]:b.cu[request + 1], slot])
            rows = got[:, b.cu[request]:b.cu[request + 1]].cpu()
            assert bool(torch.isfinite(rows[:, ~seen]).all()), (what, value)
            hit = rows[:, seen] if what == "key" else rows[:, seen][..., 3]
            assert not bool(torch.isfinite(hit).any()), (what, value)
            if what == "value" and not math.isnan(value):
                assert bool((hit == value).all())
        finite = torch.isfinite(want)
        if what == "value":
            check_attention(got, b, note=f"{what} {value}")
        else:
            assert torch.equal(torch.isfinite(got.cpu())[finite], torch.ones_like(finite)[finite])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_slots_behind_the_sequences_may_hold_anything(dtype):
    b = Batch(12, dtype, 8, 2, 128, 16, [37, 9], [6, 20], "tree")
    plain = run(b)
    for s in range(2):
        n = int(b.seq_lens[s])
        for t in range(n, math.ceil(n / 16) * 16):
            for pool in (b.key_pool, b.value_pool):
                pool[int(b.table[s, t // 16]), 0, :, t % 16] = math.nan
    assert torch.equal(run(b), plain)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_large_scores(dtype):
    """Scores of thousands, of either sign: the running maximum carries them."""
    b = Batch(13, dtype, 4, 2, 64, 16, [1, 300], [5, 40], "tree", q_std=300.0)
    check_attention(run(b), b)
    b.key_pool[:] = b.key_pool.abs()
    b.queries[:] = -b.queries.abs()
    check_attention(run(b), b)


def test_scale():
    b = Batch(14, F16, 4, 2, 64, 16, [20, 300], [5, 40])
    check_attention(run(b, scale=0.3), b, scale=0.3)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides(dtype):
    """Token-major queries out of a wider row, and a head-major output with gaps."""
    b = Batch(15, dtype, 8, 2, 64, 16, [50, 700], [11, 3])
    t = b.device()
    tokens = t["q"].shape[1]
    wide = torch.full((tokens, 12, 64), math.nan, dtype=dtype, device="cuda")
    wide[:, 2:10] = t["q"].transpose(0, 1)
    t["q"] = wide[:, 2:10].transpose(0, 1)
    backing = torch.full((8, tokens + 5, 64), 3.0, dtype=dtype, device="cuda")
    t["out"] = backing[:, 2:2 + tokens]
    check_attention(run(b, t), b)
    assert bool((backing[:, :2] == 3.0).all()) and bool((backing[:, 2 + tokens:] == 3.0).all())


def test_equals_the_causal_call_on_a_chain():
    """A chain's masks are the causal ones: mvr_paged_attention gives the same attention."""
    b = Batch(16, F16, 8, 2, 128, 16, [200, 1500, 31], [5, 5, 5], "chain")
    t = b.device()
    got = run(b, dict(t))
    t.pop("masks")
    causal = M.paged_attention(**t, max_q_len=b.max_q, max_seq_len=b.max_len)
    check_attention(got, b)
    check_attention(causal, b)


def test_bad_page_ids_read_inside_the_pool():
    """An entry outside the pool reads the last page, whatever request it belongs to; the others are not touched."""
    b = Batch(17, F16, 8, 2, 64, 16, [100, 60, 33], [4, 9, 2], "tree")
    t = b.device()
    good = run(b, dict(t))
    bad = t["block_tables"].clone()
    bad[1, 0], bad[1, 2] = 2 ** 31 - 1, -5
    last = t["block_tables"].clone()
    last[1, 0] = last[1, 2] = b.num_pages - 1
    got = run(b, dict(t, block_tables=bad))
    assert torch.equal(got, run(b, dict(t, block_tables=last)))
    for s in (0, 2):
        assert torch.equal(got[:, b.cu[s]:b.cu[s + 1]], good[:, b.cu[s]:b.cu[s + 1]])


def test_lengths_above_the_bounds_are_clamped():
    """Device lengths above max_seq_len and max_q_len: clamped to what the host checked, nothing read past the tables."""
    b = Batch(18, F16, 4, 2, 64, 16, [60, 100], [4, 9], "random")
    t = b.device()
    lens = t["seq_lens"].clone()
    lens[1] = 10 ** 6
    got = run(b, dict(t, seq_lens=lens))
    assert torch.equal(got, run(b, dict(t)))  # the longest request is as long as max_seq_len


def test_pool_offsets_past_32_bits():
    """Pages whose elements lie past 2^31 and whose bytes lie past 2^32."""
    d, page, hkv = 128, 16, 8
    pages = (1 << 31) // (hkv * page * d) + 40
    b = Batch(19, F16, 32, hkv, d, page, [70, 20], [9, 3], "tree")
    t = b.device()
    far = [torch.empty((pages, 1, hkv, page, d), dtype=F16, device="cuda") for _ in range(2)]
    for big, small in zip(far, ("key_pool", "value_pool")):
        big[-b.num_pages:] = t[small]
    t.update(key_pool=far[0], value_pool=far[1], block_tables=t["block_tables"] + (pages - b.num_pages))
    check_attention(run(b, t), b)


@pytest.mark.parametrize("cached,nodes", [([2500, 60], [20, 7]), ([30], [64])])
def test_graph(cached, nodes):
    """Captured and replayed with new contents, eager calls between the replays; two graphs share one workspace."""
    batches = [Batch(20 + i, F16, 8, 2, 128, 16, cached, nodes, "tree") for i in range(3)]
    b = batches[0]
    t = b.device()
    outs = [torch.zeros_like(t["q"]) for _ in range(2)]
    calls = [D.make_tree_call(**t, out=outs[0], max_q_len=b.max_q, max_seq_len=b.max_len, seq_lens_host=b.seq_lens,
                              cu_q_lens_host=b.cu)]
    calls.append(D.make_tree_call(**t, out=outs[1], max_q_len=b.max_q, max_seq_len=b.max_len,
                                  workspace=calls[0].workspace, seq_lens_host=b.seq_lens, cu_q_lens_host=b.cu))
    graphs = []
    for c in calls:
        c()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c()
        graphs.append(g)
    for other in batches:
        new = other.device()
        for k in ("q", "key_pool", "value_pool", "block_tables", "masks"):
            t[k].copy_(new[k])
        for o in outs:
            o.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        eager = run(other, dict(new))
        for o in outs:
            assert torch.equal(o, eager)
        check_attention(outs[0], other)


def test_graph_replayed_for_other_lengths():
    """A graph captured for one batch, replayed with the tables of others within its bounds: longer and shorter
    contexts, other trees, empty requests."""
    hkv, d, width = 2, 128, 200
    pages = 4 * width
    first = Batch(60, F16, 8, hkv, d, 16, [2500, 60, 1200, 9], [20, 7, 1, 33], "tree", spare=pages)
    t = first.device()
    t["block_tables"] = torch.zeros((4, width), dtype=torch.int32, device="cuda")
    t["block_tables"][:, :first.table.shape[1]] = torch.from_numpy(first.table).cuda()
    tokens, max_q, max_len = 160, 40, 3000
    for k, shape in (("q", (8, tokens, d)), ("masks", (tokens, 2))):
        big = torch.zeros(shape, dtype=t[k].dtype, device="cuda")
        if k == "q":
            big[:, :t[k].shape[1]] = t[k]
        else:
            big[:t[k].shape[0], :t[k].shape[1]] = t[k]
        t[k] = big
    out = torch.zeros_like(t["q"])
    call = D.make_tree_call(**t, out=out, max_q_len=max_q, max_seq_len=max_len, seq_lens_host=first.seq_lens,
                            cu_q_lens_host=first.cu, sum_seq_lens=int(first.seq_lens.sum()))
    assert call.args.workspace_bytes > 0
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed, cached, q in ((61, [2900, 2900, 2900, 2900], [40, 40, 40, 40]), (62, [0, 5, 0, 1], [1, 1, 2, 3]),
                            (63, [100, 0, 2000, 700], [0, 40, 0, 12]), (60, first.cached, first.q_lens)):
        b = Batch(seed, F16, 8, hkv, d, 16, cached, q, "tree", words=2)
        new = b.device()
        t["key_pool"][:b.num_pages].copy_(new["key_pool"])
        t["value_pool"][:b.num_pages].copy_(new["value_pool"])
        t["q"][:, :b.queries.shape[1]].copy_(new["q"])
        t["masks"][:b.masks.shape[0]].copy_(new["masks"])
        t["block_tables"][:, :b.table.shape[1]].copy_(new["block_tables"])
        t["seq_lens"].copy_(new["seq_lens"])
        t["cu_q_lens"].copy_(new["cu_q_lens"])
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        check_attention(out[:, :b.queries.shape[1]], b, note=str(seed))
        assert bool((out[:, int(b.cu[-1]):] == 9.0).all())
        check_attention(run(b, dict(new)), b, note=f"eager {seed}")


def test_streams():
    """A call given another stream, and the call objects on the stream that is current."""
    b = Batch(23, F16, 8, 2, 128, 16, [2500, 60], [20, 7], "tree")
    want = run(b)
    side = torch.cuda.Stream()
    t = b.device()
    torch.cuda.synchronize()
    got = D.paged_attention_tree(**t, max_q_len=b.max_q, max_seq_len=b.max_len, stream=side, seq_lens_host=b.seq_lens,
                                 cu_q_lens_host=b.cu, sum_seq_lens=int(b.seq_lens.sum()))
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(t["q"])
    call = D.make_tree_call(**t, out=out, max_q_len=b.max_q, max_seq_len=b.max_len, seq_lens_host=b.seq_lens,
                            cu_q_lens_host=b.cu, sum_seq_lens=int(b.seq_lens.sum()))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    assert torch.equal(out, want)


def test_same_bits_each_time():
    b = Batch(24, F16, 8, 2, 128, 16, [2500, 60, 1111], [20, 7, 33], "tree")
    t = b.device()
    first = run(b, dict(t))
    for _ in range(5):
        assert torch.equal(run(b, dict(t)), first)


def test_workspace_of_a_call_is_refused_unaligned():
    b = Batch(25, F16, 8, 2, 128, 16, [2500], [20])
    t = b.device()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")[8:]
    with pytest.raises(M.MvrError, match="256-byte aligned"):
        run(b, t, workspace=ws)


def test_c_entry_point():
    """The C entry point itself, as a runner calls it."""
    b = Batch(26, F16, 8, 2, 128, 16, [100], [20], "tree")
    t = b.device()
    out = torch.empty_like(t["q"])
    c = D.make_tree_call(**t, out=out, max_q_len=b.max_q, max_seq_len=b.max_len)
    lib = D.load_library()
    c.args.stream = None
    assert lib.mvr_paged_attention_tree(ctypes.byref(c.args), ctypes.byref(c.extra)) == 0
    torch.cuda.synchronize()
    check_attention(out, b)
