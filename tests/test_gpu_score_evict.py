"""mvr_select_tokens and mvr_move_tokens on the GPU against token-by-token forms: equal weights, infinities, NaN and zeros
of both signs, protected tokens, lengths from one token to long ones, odd pages, rows of any bytes, broken tables."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_score as S  # noqa: E402
from draft_reference import random_tables  # noqa: E402
from score_reference import select  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


class Cache:
    """Requests of some tokens in several layers, on the host."""

    def __init__(self, seed, lens, keep, layers=1, hkv=2, page=16, kept=None, past=0, recent=0, first=0, values="spread",
                 max_moves=None):
        rng = np.random.default_rng(seed)
        self.lens, self.keep = np.array(lens, np.int32), np.resize(np.array(keep, np.int32), len(lens))
        self.kept = np.zeros(len(lens), np.int32) if kept is None else np.resize(np.array(kept, np.int32), len(lens))
        self.next = (self.lens + past).astype(np.int32)
        self.recent, self.first, self.page, self.hkv, self.layers = recent, first, page, hkv, layers
        need = [-(-int(n) // page) for n in lens]
        self.pages = layers * sum(need) + 2
        table = random_tables(rng, need * layers, self.pages)
        self.table = table.reshape(layers, len(lens), -1)
        shape = (self.pages, hkv, page)
        if values == "spread":
            self.weights = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
        elif values == "equal":
            self.weights = np.full(shape, 0.25, np.float32)
        else:  # few values, odd ones among them
            self.weights = rng.choice(np.array([0.0, -0.0, 1.0, 1.0, 2.0, np.inf, -np.inf, np.nan, -3.0, 1e-42], np.float32), shape)
        self.positions = rng.permutation(np.arange(self.pages * hkv * page)).astype(np.int32).reshape(shape)
        for b, k in enumerate(self.kept):  # what was kept lies before what was appended since
            for layer in range(layers):
                for h in range(hkv):
                    slots = np.arange(k)
                    some = rng.permutation(int(k) + past)[:int(k)]
                    self.positions[self.table[layer, b, slots // page], h, slots % page] = some
        self.max_len = max(1, int(self.lens.max()))
        self.max_moves = max_moves or max(1, int(np.minimum(self.keep, self.lens - self.keep).max(initial=1)))

    def reference(self):
        return select(self.weights, self.positions, self.table, self.lens, self.next, self.kept, self.keep, self.recent,
                      self.first, self.max_moves)

    def device(self):
        up = lambda x: torch.from_numpy(x.copy()).cuda()  # noqa: E731
        return dict(weights=up(self.weights), positions=up(self.positions), block_tables=up(self.table),
                    seq_lens=up(self.lens), next_positions=up(self.next), kept_lens=up(self.kept), keep_lens=up(self.keep))

    def sizes(self):
        return dict(recent=self.recent, first=self.first, max_seq_len=self.max_len)


def check(c, t=None, **changed):
    t = {**(t or c.device()), **changed}
    rows = (c.layers, len(c.lens), c.hkv)
    moves = torch.full(rows + (c.max_moves, 2), -7, dtype=torch.int32, device="cuda")
    counts = torch.full(rows, -7, dtype=torch.int32, device="cuda")
    new = torch.full((len(c.lens),), -7, dtype=torch.int32, device="cuda")
    S.make_select_call(*t.values(), moves, counts, new, **c.sizes())()
    torch.cuda.synchronize()
    want, new_lens, positions = c.reference()
    assert new.cpu().numpy().tolist() == new_lens.tolist()
    assert np.array_equal(t["positions"].cpu().numpy(), positions)
    moves, counts = moves.cpu().numpy(), counts.cpu().numpy()
    for layer in range(c.layers):
        for b in range(len(c.lens)):
            for h in range(c.hkv):
                n, row = counts[layer, b, h], moves[layer, b, h]
                assert [tuple(x) for x in row[:n].tolist()] == want[layer][b][h], (layer, b, h)
                assert bool((row[n:] == -7).all())
    return want


@pytest.mark.parametrize("values", ["spread", "equal", "odd"])
@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 127, 128, 129, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 5000])
def test_lengths(n, values):
    for keep in sorted({1, max(1, n // 3), max(1, n - 1), n}):
        check(Cache(n + keep, [n], keep, values=values))


@pytest.mark.parametrize("values", ["spread", "odd"])
@pytest.mark.parametrize("page", [1, 3, 5, 16, 100])
def test_pages_layers_and_ragged_requests(page, values):
    check(Cache(page, [5, 700, 64, 1, 300], [10, 200, 63, 1, 17], layers=3, page=page, recent=4, first=2, values=values))


def test_protected_tokens():
    for values in ("spread", "equal", "odd"):
        check(Cache(1, [500, 90], [100, 40], recent=30, first=4, values=values))
        check(Cache(2, [500, 90], [100, 40], recent=96, first=4, values=values))
        check(Cache(3, [500, 90], [100, 40], recent=2 ** 31 - 1, values=values))  # all are: the lowest slots
        check(Cache(4, [516, 520], 500, kept=[500, 500], past=3000, recent=64, first=4, values=values))
        check(Cache(5, [516, 520], 500, kept=[516, 500], past=3000, recent=64, first=2000, values=values))


def test_caches_that_are_cut_again():
    for values in ("spread", "odd"):
        check(Cache(6, [1040, 1030, 1100], 1024, layers=4, kept=[1024, 1024, 1050], past=777, recent=128, values=values))


def test_long_rows():
    for n, keep in ((30000, 4000), (131072, 128), (131072, 130000)):
        check(Cache(n + keep, [n], keep, hkv=1, recent=32))


def test_requests_that_are_not_cut():
    """Shorter ones, ones whose moves might not fit, and ones that keep nothing."""
    check(Cache(7, [50, 60, 400, 0, 33], [50, 61, 200, 5, 0]))
    check(Cache(8, [400, 60], [200, 50], max_moves=150))
    check(Cache(9, [400, 60], [-5, 2 ** 31 - 1]))


def test_tables_left_out():
    """No next positions and no kept lengths: a cache that was never cut."""
    c = Cache(10, [300, 70], [100, 40], recent=10)
    check(c, next_positions=None, kept_lens=None)
    one = Cache(11, [300, 70], [100, 40])
    t = one.device()
    check(one, t, block_tables=t["block_tables"][0])


def test_pages_outside_the_pool_are_left_alone():
    """Their tokens rank last, and no position is written for them."""
    for bad in (-1, 10 ** 6, 2 ** 31 - 1):
        c = Cache(12, [300, 70], [100, 40], layers=2, recent=20)
        c.table[1, 0, 3] = bad
        c.table[0, 0, 18] = bad  # of protected tokens
        check(c)


def test_lengths_above_their_bound_are_clamped():
    c = Cache(13, [300, 70], [100, 40])
    t = c.device()
    t["seq_lens"][0] = 10 ** 6
    c.next[0] = 300
    check(c, t)


# ---- moves -------------------------------------------------------------------

def moved(pools, weights, positions, table, moves, counts, page):
    """numpy, move by move."""
    layers, batch, hkv = counts.shape
    for layer in range(layers):
        for b in range(batch):
            for h in range(hkv):
                for a, z in moves[layer, b, h, :max(0, min(counts[layer, b, h], moves.shape[3]))].tolist():
                    if not (0 <= a < table.shape[2] * page and 0 <= z < table.shape[2] * page):
                        continue
                    s, d = table[layer, b, a // page], table[layer, b, z // page]
                    if not (0 <= s < len(pools[0]) and 0 <= d < len(pools[0])):
                        continue
                    for p in pools:
                        p[d, 0, h, z % page] = p[s, 0, h, a % page]
                    for p in (weights, positions):
                        if p is not None:
                            p[d, h, z % page] = p[s, h, a % page]


def move_case(seed, dtype, d, page, lens, layers=1, hkv=2, most=None, offset=0):
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens] * layers
    pages = sum(need) + 2
    table = random_tables(rng, need, pages).reshape(layers, len(lens), -1)
    shape = (pages, 1, hkv, page, d)
    bits = rng.integers(0, 2 ** 16, (2, int(np.prod(shape)) + offset), dtype=np.uint16)
    if dtype == torch.float32:
        bits = bits.astype(np.uint32) << 7
    pools = [torch.from_numpy(x.view(np.float16 if dtype == torch.float16 else np.float32)).cuda()[offset:].view(shape) for x in bits]
    weights = rng.random((pages, hkv, page)).astype(np.float32)
    positions = rng.integers(0, 10 ** 6, (pages, hkv, page)).astype(np.int32)
    most = most or max(1, max(lens) // 2)
    moves = np.full((layers, len(lens), hkv, most, 2), -9, np.int32)
    counts = np.zeros((layers, len(lens), hkv), np.int32)
    for layer in range(layers):
        for b, n in enumerate(lens):
            for h in range(hkv):
                k = int(rng.integers(0, min(most, n // 2) + 1))
                moves[layer, b, h, :k] = rng.permutation(n)[:2 * k].reshape(k, 2)
                counts[layer, b, h] = k
    return pools, weights, positions, table, moves, counts


def check_moves(pools, weights, positions, table, moves, counts, page, pick=(True, True)):
    up = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    w, p = up(weights) if pick[0] else None, up(positions) if pick[1] else None
    # (A move that is refused or left out leaves the target as it was.)
    want = [x.cpu().contiguous().view(torch.int16 if x.dtype == torch.float16 else torch.int32).numpy().copy() for x in pools]
    S.move_tokens(*pools, w, p, up(table), up(moves), up(counts))
    torch.cuda.synchronize()
    moved(want, weights if pick[0] else None, positions if pick[1] else None, table, moves, counts, page)
    for got, x in zip(pools, want):
        assert np.array_equal(got.cpu().view(torch.int16 if got.dtype == torch.float16 else torch.int32).numpy(), x)
    if pick[0]:
        assert np.array_equal(w.cpu().numpy(), weights)
    if pick[1]:
        assert np.array_equal(p.cpu().numpy(), positions)


@pytest.mark.parametrize("d", [1, 3, 8, 40, 64, 96, 128, 256, 1000, 3000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_moves_of_any_row(dtype, d):
    check_moves(*move_case(d, dtype, d, 16, [60, 200, 1]), 16)


@pytest.mark.parametrize("page", [1, 5, 24])
def test_moves_in_layers(page):
    check_moves(*move_case(page, torch.float16, 128, page, [90, 33, 700, 2], layers=3, hkv=3), page)
    check_moves(*move_case(page, torch.float16, 64, page, [90, 33], layers=2), page, pick=(True, False))
    check_moves(*move_case(page, torch.float32, 64, page, [90, 33], layers=2), page, pick=(False, True))
    check_moves(*move_case(page, torch.float32, 64, page, [90, 33], layers=2), page, pick=(False, False))


def test_pools_that_are_aligned_to_elements_only():
    check_moves(*move_case(5, torch.float16, 64, 16, [90, 33], offset=3), 16)
    check_moves(*move_case(6, torch.float32, 64, 16, [90, 33], offset=1), 16)


def test_broken_moves_are_left_out():
    pools, weights, positions, table, moves, counts = move_case(7, torch.float16, 64, 16, [90, 64])
    moves[0, 0, 0, :5] = [[-1, 3], [5, -2], [10 ** 6, 7], [9, 2 ** 31 - 1], [11, 12]]
    counts[0, 0, 0] = 5
    counts[0, 0, 1] = -4
    moves[0, 1, 0] = np.arange(2 * moves.shape[3]).reshape(-1, 2)
    moves[0, 1, 0, 30:] = -1
    counts[0, 1, 0] = 10 ** 6
    table[0, 1, 1] = -1
    table[0, 1, 2] = 10 ** 6
    check_moves(pools, weights, positions, table, moves, counts, 16)


def test_graph_replays_of_a_cut():
    """Selection and moves in one graph, on other weights each time."""
    c = Cache(14, [900, 300], [256, 100], layers=2, recent=16)
    t = c.device()
    rng = np.random.default_rng(3)
    pools = [torch.from_numpy(rng.standard_normal((c.pages, 1, c.hkv, 16, 64)).astype(np.float16)).cuda() for _ in range(2)]
    rows = (c.layers, 2, c.hkv)
    moves, counts = torch.zeros(rows + (c.max_moves, 2), dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    calls = (S.make_select_call(*t.values(), moves, counts, None, **c.sizes()),
             S.make_move_call(*pools, t["weights"], t["positions"], t["block_tables"], moves, counts))
    for call in calls:
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            call()
    for k in range(4):
        fresh = torch.from_numpy(np.exp(rng.standard_normal(c.weights.shape)).astype(np.float32))
        results = []
        for go in (graph.replay, lambda: [call() for call in calls]):
            t["weights"].copy_(fresh)
            t["positions"].copy_(torch.from_numpy(c.positions))
            for x, seed in zip(pools, (1, 2)):
                x.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(x.shape).astype(np.float16)))
            go()
            torch.cuda.synchronize()
            results.append([x.clone() for x in (*pools, t["weights"], t["positions"], counts)])
        assert all(torch.equal(x, y) for x, y in zip(*results)), k


def test_refuses_tensors_that_do_not_fit():
    c = Cache(15, [90], [40])
    t = c.device()
    for name, bad in (("positions", t["positions"].float()), ("weights", t["weights"][..., :-1]), ("keep_lens", t["keep_lens"][:0]),
                      ("seq_lens", None), ("positions", None), ("block_tables", t["block_tables"].long()),
                      ("weights", t["weights"].cpu()), ("recent", -1), ("max_seq_len", 10 ** 4), ("max_moves", 0)):
        with pytest.raises(M.MvrError):
            S.select_tokens(**{**t, **c.sizes(), "max_moves": 50, name: bad})
