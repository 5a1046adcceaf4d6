"""The cache side of drafted trees on the GPU: mvr_norm_rope_append against norm and rotation in 64 bits, the
compaction and the page copies bit for bit against plain indexing; and the four calls together as one step uses them."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_draft as D  # noqa: E402
from draft_reference import EPS, Batch, check_attention, random_tables  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    D.load_library()


# ---- norm, rotation, append ------------------------------------------------

class Append:
    """New rows of a batch, and what the append makes of them in 64 bits."""

    def __init__(self, seed, dtype, hq, hkv, d, page, cached, q, rope=D.ROPE_NEOX, eps=1e-5, norms="both",
                 positions=True, tail=0, rope_len=None, std=1.0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.page, self.rope, self.eps = dtype, hq, hkv, d, page, rope, eps
        self.q_lens, self.cached = np.array(q, np.int32), np.array(cached, np.int32)
        self.seq_lens = (self.cached + self.q_lens).astype(np.int32)
        self.cu = np.concatenate([[0], np.cumsum(self.q_lens)]).astype(np.int32)
        self.max_len = max(int(self.seq_lens.max()), 1)
        need = [math.ceil(n / page) for n in self.seq_lens]
        self.num_pages = max(sum(need), 1) + 2
        self.table = random_tables(rng, need, self.num_pages)
        tokens = max(int(self.cu[-1]) + tail, 1)
        normal = lambda shape, mean=0.0, s=1.0: (torch.randn(shape, generator=gen) * s + mean).to(dtype)  # noqa: E731
        self.q, self.k = normal((hq, tokens, d), s=std), normal((hkv, tokens, d), s=std)
        self.v = normal((hkv, tokens, d))
        self.q_weight = normal((d,), 1.0, 0.3) if norms in ("both", "q") else None
        self.k_weight = normal((d,), 1.0, 0.3) if norms in ("both", "k") else None
        self.key_pool = normal((self.num_pages, 1, hkv, page, d))
        self.value_pool = normal((self.num_pages, 1, hkv, page, d))
        self.rope_len = rope_len or self.max_len
        angle = np.arange(self.rope_len)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
        self.cos, self.sin = (torch.from_numpy(f(angle)).to(dtype) for f in (np.cos, np.sin))
        self.positions = rng.integers(0, self.rope_len, tokens).astype(np.int32) if positions else None

    def slots(self):
        """(request, slot) of every token of a request."""
        return [(b, int(self.cached[b]) + i) for b in range(len(self.q_lens)) for i in range(int(self.q_lens[b]))]

    def rotated(self, x, weight):
        """(rows, tolerance) in 64 bits.  Rounded: the result (half a step); before it the norm (D/8 + log2 D products
        and sums in the square sum, then a root, a quotient, three products) and the rotation (two products, a sum) in
        32 bits, relative to the two products' size."""
        rows = int(self.cu[-1])
        x = x[:, :rows].double()
        if weight is not None:
            x = x / ((x * x).mean(-1, keepdim=True) + self.eps).sqrt() * weight.double()
        pos = self.positions[:rows] if self.positions is not None else np.array([t for _, t in self.slots()], np.int64)
        c, s = self.cos[pos].double(), self.sin[pos].double()
        if self.rope == D.ROPE_NEOX:
            a, b = x[..., :self.d // 2], x[..., self.d // 2:]
        else:
            a, b = x[..., 0::2], x[..., 1::2]
        pair = [a * c - b * s, a * s + b * c]
        size = [(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()]
        join = (lambda z: torch.cat(z, -1)) if self.rope == D.ROPE_NEOX else (lambda z: torch.stack(z, -1).flatten(-2))
        y, m = join(pair), join(size)
        tiny = 2.0 ** -25 if self.dtype == F16 else 2.0 ** -149  # half a step below the normal range
        return y, EPS[self.dtype] * y.abs() + 2.0 ** -24 * (self.d / 8 + 20) * m + tiny

    def device(self):
        dev = lambda x: None if x is None else (torch.from_numpy(x) if isinstance(x, np.ndarray) else x).cuda()  # noqa: E731
        return dict(q=dev(self.q), k=dev(self.k), v=dev(self.v), q_weight=dev(self.q_weight), k_weight=dev(self.k_weight),
                    cos_table=dev(self.cos), sin_table=dev(self.sin), block_tables=dev(self.table),
                    seq_lens=dev(self.seq_lens), cu_q_lens=dev(self.cu), key_pool=dev(self.key_pool),
                    value_pool=dev(self.value_pool), positions=dev(self.positions))

    def kw(self):
        return dict(eps=self.eps, max_seq_len=self.max_len, rope_type=self.rope)

    def check(self, q_out, key_pool, value_pool, skip=()):
        rows = int(self.cu[-1])
        keep = torch.tensor([n not in skip for n in range(rows)])
        want, tol = self.rotated(self.q, self.q_weight)
        off = ((q_out[:, :rows].double().cpu() - want).abs() - tol)[:, keep]
        assert off.numel() == 0 or float(off.max()) <= 0, "queries"
        keys, key_tol = self.key_pool.double(), torch.zeros(self.key_pool.shape, dtype=torch.float64)
        values = self.value_pool.clone()
        want, tol = self.rotated(self.k, self.k_weight)
        for n, (b, t) in enumerate(self.slots()):
            if n in skip:
                continue
            at = (int(self.table[b, t // self.page]), 0, slice(None), t % self.page)
            keys[at], key_tol[at] = want[:, n], tol[:, n]
            values[at] = self.v[:, n]
        assert float(((key_pool.double().cpu() - keys).abs() - key_tol).max()) <= 0, "keys (untouched slots bit for bit)"
        assert torch.equal(value_pool.cpu(), values), "values"


def append(a, t=None, **kw):
    t = t or a.device()
    out = D.norm_rope_append(**t, **{**a.kw(), **kw})
    torch.cuda.synchronize()
    return out, t["key_pool"], t["value_pool"]


@pytest.mark.parametrize("rope", [D.ROPE_NEOX, D.ROPE_INTERLEAVED])
@pytest.mark.parametrize("d", [8, 16, 24, 40, 64, 80, 96, 128, 256, 264, 512])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_every_head_dim(dtype, d, rope):
    a = Append(d, dtype, 6, 2, d, 5, [0, 13, 40], [7, 1, 12], rope)
    a.check(*append(a))


@pytest.mark.parametrize("norms", ["both", "q", "k", "none"])
@pytest.mark.parametrize("positions", [True, False])
def test_append_norms_and_positions(norms, positions):
    for dtype in (F16, F32):
        a = Append(1, dtype, 8, 2, 64, 16, [0, 100], [1, 30], norms=norms, positions=positions)
        a.check(*append(a))


@pytest.mark.parametrize("requests", [1, 2, 62, 63, 64, 65, 130, 700, 4100])
def test_append_finds_the_request_of_a_token(requests):
    """Tables of one search round and of two, empty requests among them, first and last."""
    rng = np.random.default_rng(requests)
    q = rng.integers(0, 3, requests)
    q[requests // 2] = 2
    a = Append(requests, F16, 2, 1, 16, 4, rng.integers(0, 9, requests), q)
    a.check(*append(a))


def test_append_one_request_without_tables():
    a = Append(2, F16, 8, 2, 64, 16, [21], [9])
    t = a.device()
    t["seq_lens"] = t["cu_q_lens"] = None
    a.check(*append(a, t))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_in_place_from_a_packed_projection(dtype):
    """q, k and v as slices of one [tokens, (Hq + 2 Hkv) D] row, the queries rotated in place."""
    a = Append(3, dtype, 8, 2, 64, 16, [5, 60], [9, 33])
    t = a.device()
    packed = torch.cat([t["q"], t["k"], t["v"]]).transpose(0, 1).contiguous()
    heads = packed.transpose(0, 1)
    t.update(q=heads[:8], k=heads[8:10], v=heads[10:])
    out, keys, values = append(a, t, q_out=heads[:8])
    a.check(out, keys, values)
    assert torch.equal(packed[:, 8:].cpu(), torch.cat([a.k, a.v]).transpose(0, 1))


def test_append_padded_batch():
    """Rows behind the last request: neither read nor written."""
    a = Append(4, F16, 4, 2, 64, 16, [5, 0, 60], [9, 0, 3], tail=6)
    t = a.device()
    rows = int(a.cu[-1])
    for k in ("q", "k", "v"):
        t[k][:, rows:] = math.nan
    t["positions"][rows:] = 10 ** 9
    out = torch.full_like(t["q"], 5.0)
    a.check(*append(a, t, q_out=out))
    assert bool((out[:, rows:] == 5.0).all())


def test_append_leaves_out_what_lies_outside():
    """Positions outside the rotary tables and pages outside the pool: those rows alone are left out."""
    a = Append(5, F16, 4, 2, 64, 4, [4, 8], [5, 4])
    t = a.device()
    t["positions"][1], t["positions"][3] = -1, a.rope_len
    t["block_tables"][1, 2] = a.num_pages  # request 1: tokens 5 .. 8
    out = torch.full_like(t["q"], 5.0)
    a.check(*append(a, t, q_out=out), skip=(1, 3, 5, 6, 7, 8))
    assert bool((out[:, [1, 3, 5, 6, 7, 8]] == 5.0).all())


def test_append_extreme_rows():
    """Rows of zeros, tiny and huge values, eps 0; NaN stays in its row."""
    for dtype, std in ((F16, 1e-4), (F16, 300.0), (F32, 1e-15), (F32, 1e12)):
        a = Append(6, dtype, 4, 2, 64, 16, [5], [9], eps=0.0, std=std)
        a.check(*append(a))
    a = Append(7, F16, 4, 2, 64, 16, [5], [9], eps=1e-6)
    a.q[1, 2] = 0
    a.check(*append(a))
    a.q[1, 2, 5] = math.nan
    out = append(a)[0]
    bad = torch.isnan(out)
    assert bool(bad[1, 2].all()) and int(bad.sum()) == 64


def test_append_far_positions():
    a = Append(8, F32, 4, 2, 64, 16, [5], [9], rope_len=200000)
    a.positions[:] = np.arange(9) + 199991
    a.check(*append(a))


# ---- compaction ------------------------------------------------------------

def compact_case(seed, dtype, hkv, d, page, cached, q, counts, layers):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    q_lens, cached = np.array(q, np.int32), np.array(cached, np.int32)
    seq_lens = (cached + q_lens).astype(np.int32)
    need = [math.ceil(n / page) for n in seq_lens] * layers
    pages = max(sum(need), 1) + 2
    table = random_tables(rng, need, pages, width=max(max(need), 1)).reshape(layers, len(q), -1)
    most = max(max(counts), 1)
    accepted = np.full((len(q), most), -7, np.int32)  # entries behind a path are never looked at
    for b, n in enumerate(counts):
        accepted[b, :n] = np.sort(rng.permutation(q_lens[b])[:n])
    pools = [torch.randn((pages, 1, hkv, page, d), generator=gen).to(dtype) for _ in range(2)]
    return dict(pools=pools, table=table, seq_lens=seq_lens, cu=np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32),
                accepted=accepted, counts=np.array(counts, np.int32), page=page, first=cached)


def compact_expected(c):
    out = []
    for pool in c["pools"]:
        new = pool.clone()
        for layer in range(c["table"].shape[0]):
            for b, n in enumerate(c["counts"]):
                for j in range(n):
                    s, t = int(c["first"][b]) + int(c["accepted"][b, j]), int(c["first"][b]) + j
                    row = c["table"][layer, b]
                    new[int(row[t // c["page"]]), 0, :, t % c["page"]] = pool[int(row[s // c["page"]]), 0, :, s % c["page"]]
        out.append(new)
    return out


def run_compact(c, **kw):
    dev = [p.cuda() for p in c["pools"]]
    t = [torch.from_numpy(c[k]).cuda() for k in ("table", "seq_lens", "cu", "accepted", "counts")]
    lens = D.compact_drafts(*dev, *t, max_seq_len=max(int(c["seq_lens"].max()), 1), **kw)
    torch.cuda.synchronize()
    return dev, lens


@pytest.mark.parametrize("dtype,d,page", [(F16, 128, 16), (F32, 64, 16), (F16, 64, 5), (F16, 3, 7), (F32, 5, 1),
                                          (F16, 7, 2), (F32, 1030, 4), (F16, 5000, 3), (F32, 96, 24)])
@pytest.mark.parametrize("layers", [1, 3])
def test_compact(dtype, d, page, layers):
    """Rows of every vector width, shorter and longer than a batch of registers; paths of none, one, some and all."""
    c = compact_case(d + page, dtype, 2, d, page, [0, 13, 40, 9, 3], [7, 1, 12, 0, 70], [3, 1, 12, 0, 41], layers)
    dev, lens = run_compact(c)
    for got, want in zip(dev, compact_expected(c)):
        assert torch.equal(got.cpu(), want)
    assert torch.equal(lens.cpu(), torch.from_numpy(c["first"] + c["counts"]))


def test_compact_long_paths():
    """Paths of many batches, each of which overwrites sources of the ones before."""
    for dtype, d in ((F16, 128), (F32, 128), (F16, 8)):
        c = compact_case(1, dtype, 2, d, 16, [5, 100], [900, 333], [600, 332], 2)
        dev, _ = run_compact(c)
        for got, want in zip(dev, compact_expected(c)):
            assert torch.equal(got.cpu(), want)


def test_compact_broken_tables_write_nothing_outside():
    """Indices outside the drafts or out of order, counts and pages out of range: left out; the other requests are
    served."""
    c = compact_case(2, F16, 2, 64, 4, [8, 6, 5], [9, 6, 4], [4, 3, 2], 1)
    want = compact_expected({**c, "counts": np.array([0, 3, 0], np.int32)})
    c["accepted"][0] = [3, 99, -5, 3]    # 3 -> 0 is moved: nothing else ascends inside the drafts
    c["table"][0, 2, :] = [-1] * c["table"].shape[2]
    c["counts"][2] = 1000                # clamped to the 4 drafts, whose pages are outside
    dev, lens = run_compact(c)
    for got, new, pool in zip(dev, want, c["pools"]):
        t, s = 8, 11
        row = c["table"][0, 0]
        new[int(row[t // 4]), 0, :, t % 4] = pool[int(row[s // 4]), 0, :, s % 4]
        assert torch.equal(got.cpu(), new)
    assert lens.tolist() == [12, 9, 9]


def test_compact_pool_without_vector_alignment():
    """Pools that start two bytes off a 16-byte boundary."""
    c = compact_case(3, F16, 2, 64, 16, [5], [30], [11], 2)
    shape = c["pools"][0].shape
    backing = [torch.zeros(p.numel() + 8, dtype=F16, device="cuda") for p in c["pools"]]
    dev = [b[1:1 + p.numel()].view(shape).copy_(p) for b, p in zip(backing, c["pools"])]
    t = [torch.from_numpy(c[k]).cuda() for k in ("table", "seq_lens", "cu", "accepted", "counts")]
    D.compact_drafts(*dev, *t, max_seq_len=int(c["seq_lens"].max()))
    for got, want in zip(dev, compact_expected(c)):
        assert torch.equal(got.cpu(), want)


# ---- copies ----------------------------------------------------------------

@pytest.mark.parametrize("dtype,hkv,d,page", [(F16, 8, 128, 16), (F32, 2, 64, 5), (F16, 3, 3, 7), (F32, 1, 1, 1),
                                              (F16, 4, 256, 48), (F32, 2, 1030, 4)])
@pytest.mark.parametrize("partial", [False, True])
@pytest.mark.parametrize("copies", [0, 1, 37])
def test_copy(dtype, hkv, d, page, partial, copies):
    rng = np.random.default_rng(copies)
    pools = [torch.randn((2 * copies + 3, 1, hkv, page, d)).to(dtype) for _ in range(2)]
    order = rng.permutation(2 * copies + 3).astype(np.int32)
    src, dst = order[:copies].copy(), order[copies:2 * copies].copy()
    if copies > 2:
        src[1] = src[0]  # one page forked twice
    tokens = rng.integers(0, page + 1, copies).astype(np.int32) if partial else None
    dev = [p.cuda() for p in pools]
    D.copy_pages(*dev, torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(),
                 None if tokens is None else torch.from_numpy(tokens).cuda())
    for got, pool in zip(dev, pools):
        want = pool.clone()
        for i in range(copies):
            n = page if tokens is None else int(tokens[i])
            want[int(dst[i]), :, :, :n] = pool[int(src[i]), :, :, :n]
        assert torch.equal(got.cpu(), want)


def test_copy_leaves_out_pages_outside_the_pool():
    pools = [torch.randn((9, 1, 2, 4, 64)).half() for _ in range(2)]
    dev = [p.cuda() for p in pools]
    lists = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, -1, 2, 9, 4], [5, 6, -3, 7, 8], [4, 4, 4, 4, 99])]
    D.copy_pages(*dev, *lists)
    for got, want in zip(dev, pools):
        want[5], want[8] = want[0], want[4]
        assert torch.equal(got.cpu(), want)


# ---- streams, graphs, and the calls together ---------------------------------

def test_cache_calls_in_a_graph():
    """Append, compaction and copy captured together, replayed on new contents with eager calls in between."""
    cases = [Append(30 + i, F16, 4, 2, 64, 16, [20, 50], [9, 5]) for i in range(3)]
    a = cases[0]
    t = a.device()
    out = torch.zeros_like(t["q"])
    accepted = torch.tensor([[0, 3, 7], [1, 4, 0]], dtype=torch.int32).cuda()
    counts = torch.tensor([3, 2], dtype=torch.int32).cuda()
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    page = torch.tensor([int(a.table[0, 1])], dtype=torch.int32).cuda()
    spare = torch.tensor([sorted(set(range(a.num_pages)) - set(a.table.flatten().tolist()))[0]],
                         dtype=torch.int32).cuda()
    calls = [D.make_norm_rope_append_call(**t, q_out=out, **a.kw()),
             D.make_compact_drafts_call(t["key_pool"], t["value_pool"], t["block_tables"], t["seq_lens"],
                                        t["cu_q_lens"], accepted, counts, lens, max_seq_len=a.max_len),
             D.make_copy_pages_call(t["key_pool"], t["value_pool"], page, spare)]
    for c in calls:
        c()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in calls:
            c()
    for other in cases:
        new = other.device()
        for k in ("q", "k", "v", "q_weight", "k_weight", "key_pool", "value_pool"):
            t[k].copy_(new[k])
        eager = {k: t[k].clone() for k in ("key_pool", "value_pool")}
        g.replay()
        torch.cuda.synchronize()
        want = D.norm_rope_append(**{**t, **eager}, **a.kw())
        D.compact_drafts(eager["key_pool"], eager["value_pool"], t["block_tables"], t["seq_lens"], t["cu_q_lens"],
                         accepted, counts, max_seq_len=a.max_len)
        D.copy_pages(eager["key_pool"], eager["value_pool"], page, spare)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and lens.tolist() == [23, 52]
        assert all(torch.equal(t[k], eager[k]) for k in eager)


def test_cache_calls_on_another_stream():
    a = Append(33, F16, 4, 2, 64, 16, [20, 50], [9, 5])
    t = a.device()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = D.norm_rope_append(**t, **a.kw(), stream=side)
    side.synchronize()
    a.check(out, t["key_pool"], t["value_pool"])
    c = compact_case(4, F16, 2, 64, 16, [5], [30], [11], 2)
    dev, _ = run_compact(c, stream=side)
    for got, want in zip(dev, compact_expected(c)):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_step_of_a_drafted_tree(dtype):
    """Append, verify, compact, then a decode step on the compacted cache: the attention of the next token is that of a
    request that generated the accepted path token by token; a request forked before the step is not touched by it."""
    hq, hkv, d, page = 8, 2, 64, 16
    parents = [[-1, 0, 0, 1, 2, 4, 2, 5], [-1, 0, 1, 1, 2]]
    paths = [[0, 2, 4, 5], [0, 1, 3]]
    rng = np.random.default_rng(40)
    cached, q = [37, 20], [len(p) for p in parents]
    b = Batch(40, dtype, hq, hkv, d, page, cached, q, spare=12)
    cu, tokens = b.cu, int(b.cu[-1])
    masks = D.tree_masks(sum(parents, []), cu)
    b.bits = np.unpackbits(masks.view(np.uint8), axis=1, bitorder="little").astype(bool)
    depth = b.bits.sum(1) - 1
    positions = (np.repeat(cached, q) + depth).astype(np.int32)
    t = b.device()
    new = {k: torch.randn((h, tokens, d)).to(dtype).cuda() for k, h in (("q", hq), ("k", hkv), ("v", hkv))}
    angle = np.arange(128)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
    rope = [torch.from_numpy(f(angle)).to("cuda", dtype) for f in (np.cos, np.sin)]
    weights = [(torch.randn(d) * 0.2 + 1).to("cuda", dtype) for _ in range(2)]
    # The fork: request 0's last page is shared, so its copy gets a page of its own.
    free = sorted(set(range(b.num_pages)) - set(b.table[0, :math.ceil(45 / page)]) - set(b.table[1, :math.ceil(25 / page)]))
    last = int(b.table[0, 37 // page])
    D.copy_pages(t["key_pool"], t["value_pool"], torch.tensor([last], dtype=torch.int32).cuda(),
                 torch.tensor([free[0]], dtype=torch.int32).cuda(), torch.tensor([37 % page], dtype=torch.int32).cuda())
    before = [t[k].clone() for k in ("key_pool", "value_pool")]

    rotated = D.norm_rope_append(new["q"], new["k"], new["v"], *weights, *rope, t["block_tables"], t["seq_lens"],
                                 t["cu_q_lens"], t["key_pool"], t["value_pool"], eps=1e-6, max_seq_len=b.max_len,
                                 positions=torch.from_numpy(positions).cuda())
    t["q"] = rotated
    out = D.paged_attention_tree(**t, max_q_len=b.max_q, max_seq_len=b.max_len)
    torch.cuda.synchronize()
    b.queries, b.key_pool, b.value_pool = rotated.cpu(), t["key_pool"].cpu(), t["value_pool"].cpu()
    check_attention(out, b)

    accepted = torch.tensor([paths[0], paths[1] + [0]], dtype=torch.int32).cuda()
    lens = D.compact_drafts(t["key_pool"], t["value_pool"], t["block_tables"], t["seq_lens"], t["cu_q_lens"], accepted,
                            torch.tensor([4, 3], dtype=torch.int32).cuda(), max_seq_len=b.max_len)
    assert lens.tolist() == [41, 23]
    # The same requests, the path appended token by token at its own slots.
    linear = [p.clone() for p in before]
    for step in range(4):
        live = [s for s in range(2) if step < len(paths[s])]
        rows = [int(cu[s]) + paths[s][step] for s in live]
        args = [new[k][:, rows].contiguous() for k in ("q", "k", "v")]
        D.norm_rope_append(*args, *weights, *rope, t["block_tables"][live].contiguous(),
                           torch.tensor([cached[s] + step + 1 for s in live], dtype=torch.int32).cuda(),
                           torch.arange(len(live) + 1, dtype=torch.int32).cuda(), *linear, eps=1e-6,
                           max_seq_len=b.max_len)
    query = torch.randn((hq, 2, d)).to(dtype).cuda()
    ones = torch.arange(3, dtype=torch.int32).cuda()
    got = M.paged_attention(query, t["key_pool"], t["value_pool"], t["block_tables"], lens, ones, max_q_len=1,
                            max_seq_len=b.max_len)
    want = M.paged_attention(query, *linear, t["block_tables"], lens, ones, max_q_len=1, max_seq_len=b.max_len)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for pool, old in zip((t["key_pool"], t["value_pool"]), before):  # the fork's page is as it was
        assert torch.equal(pool[free[0]], old[free[0]])
