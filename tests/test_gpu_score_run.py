"""The calls on scores as a server uses them together: prompts and decode steps of requests whose caches are cut to a budget,
against a plain simulation in 64 bits; in the checked mode and with trace ranges on (flags that a process reads once, hence
the child processes); from two threads at a time."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_draft as D  # noqa: E402
import mvr_score as S  # noqa: E402
from score_reference import Batch, check_attention, within  # noqa: E402

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, F32 = torch.float16, torch.float32


def skip_without_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    S.load_library()


class Head:
    """The cache of one request and KV head: a row of each kept token, in any order."""

    def __init__(self):
        self.pos, self.k, self.v, self.w = [], [], [], []


@pytest.mark.parametrize("dtype", [F32, F16])
def test_generation_on_a_bounded_cache(dtype):
    """Two requests, prompts of 70 and 33 tokens, then 40 steps: append at the tokens' own positions, capped attention,
    weights, and a cut to 48 tokens whenever a cache holds 56.  Every step's outputs, weights and choices, per KV head."""
    skip_without_gpu()
    hq, hkv, d, page, budget, limit, cap, recent, first = 4, 2, 64, 8, 48, 56, 20.0, 8, 2
    layers, gen = 2, torch.Generator().manual_seed(5)
    normal = lambda *shape: torch.randn(shape, generator=gen).to(dtype)  # noqa: E731
    prompts, steps, width = [70, 33], 40, 12
    pages = layers * 2 * width + 1
    table = torch.from_numpy(np.random.default_rng(1).permutation(pages)[:layers * 2 * width].reshape(layers, 2, width).astype(np.int32)).cuda()
    pools = [torch.zeros((pages, 1, hkv, page, d), dtype=dtype, device="cuda") for _ in range(2)]
    weights = torch.full((pages, hkv, page), float("nan"), device="cuda")
    positions = torch.full((pages, hkv, page), -1, dtype=torch.int32, device="cuda")
    angle = torch.arange(200)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)[None]
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    heads = [[[Head() for _ in range(hkv)] for _ in range(2)] for _ in range(layers)]
    lens, kept, seen = [0, 0], [0, 0], [0, 0]
    # F16 keys are rounded where they are written: the simulation takes the cache's rows from there.
    for step in range(steps + 1):
        new = prompts if step == 0 else [1, 1]
        lens, seen = [a + b for a, b in zip(lens, new)], [a + b for a, b in zip(seen, new)]
        at = [p for s, n in zip(seen, new) for p in range(s - n, s)]
        cu, seq, tokens = [0, new[0], sum(new)], ints(lens), sum(new)
        sizes = dict(max_q_len=max(new), max_seq_len=width * page)
        for layer in range(layers):
            q, k, v = normal(hq, tokens, d) * 2, normal(hkv, tokens, d), normal(hkv, tokens, d)
            rows = D.norm_rope_append(q.cuda(), k.cuda(), v.cuda(), None, None, cos.cuda(), sin.cuda(), table[layer], seq,
                                      ints(cu), *pools, eps=0.0, max_seq_len=width * page, positions=ints(at))
            out, lse = S.paged_attention_scored(rows, *pools, table[layer], seq, ints(cu), cap=cap, **sizes)
            S.attention_weights(rows, lse, pools[0], weights, table[layer], seq, ints(cu), cap=cap, **sizes)
            torch.cuda.synchronize()
            host = [x.double().cpu() for x in (rows, out, lse, pools[0], pools[1], weights)]
            for b in range(2):
                for h in range(hkv):
                    c = heads[layer][b][h]
                    slots = torch.arange(lens[b])
                    ids = table[layer, b].cpu().long()[slots // page]
                    fresh = slots[lens[b] - new[b]:]
                    for j in fresh.tolist():
                        c.pos.append(seen[b] - lens[b] + j)
                        c.k.append(host[3][ids[j], 0, h, j % page])
                        c.v.append(host[4][ids[j], 0, h, j % page])
                        c.w.append(0.0)
                    key, value, pos = torch.stack(c.k), torch.stack(c.v), torch.tensor(c.pos)
                    group = slice(h * hq // hkv, (h + 1) * hq // hkv)
                    mine = host[0][group, cu[b]:cu[b + 1]]  # [G, q, D]
                    x = cap * torch.tanh(mine @ key.T / math.sqrt(d) / cap)
                    x = x.masked_fill(pos > torch.tensor(at[cu[b]:cu[b + 1]])[:, None], -math.inf)
                    # 32-bit scores of sizes up to cap, and F16 outputs and probabilities.
                    off = 2.0 ** -18 * cap + 2.0 ** -24 * (d + 8) * 40
                    u = 2.0 ** -10 if dtype == F16 else 2.0 ** -22
                    p = torch.softmax(x, -1)
                    within(out[group, cu[b]:cu[b + 1]], p @ value, (off + u) * (p @ value.abs()) + u, f"{step} {b} {h}")
                    got = p.sum((0, 1)).tolist()
                    c.w = [a + g for a, g in zip(c.w, got)]
                    # Weights of the slots, in the simulation's order.  (Positions are written as far as kept tokens go.)
                    where = {t: j for j, t in enumerate(positions[ids, h, slots % page][:kept[b]].tolist())}
                    for j in range(kept[b], lens[b]):
                        where[seen[b] - lens[b] + j] = j
                    order = torch.tensor([where[t] for t in c.pos])
                    mine_w = host[5][ids[order], h, order % page]
                    within(mine_w, torch.tensor(c.w).double(), torch.full((lens[b],), (step + 1) * 200 * 2.0 ** -18), f"{step}")
        if max(lens) < limit:
            continue
        keep = [budget if n >= limit else 2 ** 30 for n in lens]
        moves, counts, shorter = S.select_tokens(weights, positions, table, seq, ints(seen), ints(kept), ints(keep),
                                                 recent=recent, first=first, max_seq_len=width * page, max_moves=budget)
        S.move_tokens(*pools, weights, positions, table, moves, counts)
        torch.cuda.synchronize()
        lens = shorter.cpu().tolist()
        assert lens == [budget if n == budget else m for n, m in zip(keep, seq.cpu().tolist())]
        for layer in range(layers):
            for b in range(2):
                for h in range(hkv):
                    c = heads[layer][b][h]
                    if keep[b] == budget:
                        guarded = [t < first or t >= seen[b] - recent for t in c.pos]
                        rank = sorted(range(len(c.pos)), key=lambda i: (not guarded[i], -c.w[i]))
                        edge = c.w[rank[budget - 1]] - c.w[rank[budget]]
                        assert edge > 1e-3 * c.w[rank[budget]] / 1e2, "the test's own choice is too near to call"
                        stay = sorted(rank[:budget])
                        c.pos, c.k, c.v, c.w = ([x[i] for i in stay] for x in (c.pos, c.k, c.v, c.w))
                    slots = torch.arange(lens[b], device="cuda")
                    got = positions[table[layer, b].long()[slots // page], h, slots % page].cpu().tolist()
                    assert sorted(got) == sorted(c.pos), (step, layer, b, h)
        kept = lens


def step():
    """Arguments of a small step of each call."""
    b = Batch(70, F16, 8, 2, 64, 16, [37, 300], [9, 5], cap=20.0, slopes=True, prefix=[10, 4], first_keys=[3])
    t = b.device()
    lse = b.attention()[2].float().cuda()
    weights, positions = b.weights.cuda(), torch.zeros(b.weights.shape, dtype=torch.int32, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    moves = torch.zeros((1, 2, 2, 4, 2), dtype=torch.int32, device="cuda")
    moves[0, :, :, 0, 0], moves[0, :, :, 1, 0], moves[0, :, :, 1, 1] = 40, 33, 7
    tables = dict(block_tables=t["block_tables"], seq_lens=t["seq_lens"])
    return {
        "attention": dict(t, **b.rules()),
        "weights": dict({k: t[k] for k in ("q", "key_pool", "block_tables", "seq_lens", "cu_q_lens")}, lse=lse, weights=weights,
                        decay=0.5, **b.rules()),
        "select": dict(tables, weights=weights, positions=positions, next_positions=ints(50, 400), kept_lens=ints(0, 20),
                       keep_lens=ints(30, 400), recent=4, max_seq_len=b.max_len, max_moves=16),
        "move": dict(key_pool=t["key_pool"], value_pool=t["value_pool"], weights=weights, positions=positions,
                     block_tables=t["block_tables"], moves=moves, num_moves=ints(2, 2, 2, 2).view(1, 2, 2)),
    }


CALLS = {"attention": S.paged_attention_scored, "weights": S.attention_weights, "select": S.select_tokens,
         "move": S.move_tokens}


def run_step():
    args, outs = step(), {}
    for name, f in CALLS.items():
        got = f(**args[name])
        torch.cuda.synchronize()
        if name == "select":  # (moves behind the counts are not written)
            moves, counts, lens = (x.cpu().numpy() for x in got)
            moves[np.arange(moves.shape[3]) >= counts[..., None]] = 0
            got = (torch.from_numpy(x) for x in (moves, counts, lens))
        for i, x in enumerate(got if name in ("attention", "select") else [got] if got is not None else []):
            outs[f"{name} {i}"] = x.cpu().numpy()
    for k in ("key_pool", "value_pool", "weights", "positions"):
        outs[k] = args["move"][k].cpu().numpy()
    return outs


BROKEN = {  # a call, what breaks it, and the status it gets in the checked mode
    "page outside the pool": ("attention", lambda a: a["block_tables"][1].fill_(10 ** 6), M.MVR_E_PAGE_ID),
    "length above its bound": ("attention", lambda a: a["seq_lens"].fill_(10 ** 6), M.MVR_E_INVALID_ARGUMENT),
    "descending starts": ("attention", lambda a: a["cu_q_lens"][1].fill_(99), M.MVR_E_INVALID_ARGUMENT),
    "first key below 0": ("attention", lambda a: a["first_keys"].fill_(-1), M.MVR_E_INVALID_ARGUMENT),
    "infinite slope": ("attention", lambda a: a["slopes"].fill_(math.inf), M.MVR_E_INVALID_ARGUMENT),
    "prefix below 0": ("weights", lambda a: a["prefix_lens"].fill_(-1), M.MVR_E_INVALID_ARGUMENT),
    "page of two requests": ("weights", lambda a: a["block_tables"].fill_(1), M.MVR_E_INVALID_ARGUMENT),
    "next position before the tokens": ("select", lambda a: a["next_positions"].fill_(3), M.MVR_E_LENGTH_MISMATCH),
    "more moves than room": ("select", lambda a: a["keep_lens"].fill_(23), M.MVR_E_INVALID_ARGUMENT),
    "two moves to a slot": ("move", lambda a: a["moves"][..., 1].fill_(2), M.MVR_E_INVALID_ARGUMENT),
    "slot outside the pages": ("move", lambda a: a["moves"][0, 0, 0, 0].fill_(-3), M.MVR_E_INVALID_ARGUMENT),
}


def child(out_path):
    outs = run_step()
    for name, (call, spoil, _) in BROKEN.items():
        args = step()
        spoil(args[call])
        code = 0
        try:
            CALLS[call](**args[call])
        except M.MvrError as e:
            code = e.code
        torch.cuda.synchronize()
        outs[name] = np.array(code)
        print(name, code, flush=True)
    np.savez(out_path, **outs)


def test_checked_mode_and_trace_ranges(tmp_path):
    """Valid calls give the same bits as without; broken tables are reported and nothing is launched on them."""
    skip_without_gpu()
    path = str(tmp_path / "child.npz")
    env = dict(os.environ, MVR_ATTN_CHECKED="true", MVR_ENABLE_ROCTX="true", PYTHONPATH=os.pathsep.join(
        [os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__), path], env=env, capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    got, want = np.load(path), run_step()
    for name, x in want.items():
        assert got[name].tobytes() == x.tobytes(), name
    for name, (_, _, code) in BROKEN.items():
        assert int(got[name]) == code, (name, int(got[name]), code)


def test_two_threads():
    """Calls from two threads on streams of their own, at once: every result is its own batch's."""
    skip_without_gpu()
    batches = [Batch(72 + i, F16, 8, 2, 128, 16, [1500 + 900 * i, 40], [1, 7 + i], cap=30.0) for i in range(2)]
    tensors, failures = [b.device() for b in batches], []
    outs = [[torch.empty_like(t["q"]) for _ in range(20)] for t in tensors]
    lses = [[torch.empty(t["q"].shape[:2], device="cuda") for _ in range(20)] for t in tensors]
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            calls = [S.make_scored_call(*tensors[i].values(), out, lse, stream=stream, **batches[i].rules())
                     for out, lse in zip(outs[i], lses[i])]
            start.wait()
            for call in calls:
                call()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    for i, b in enumerate(batches):
        for out, lse in zip(outs[i], lses[i]):
            assert torch.equal(out, outs[i][0]) and torch.equal(lse, lses[i][0])
        check_attention(outs[i][0], lses[i][0], b)


if __name__ == "__main__":
    child(sys.argv[1])
