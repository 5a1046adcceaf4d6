"""The calls of a server that bounds its cache by the attention its tokens get, for timing and for comparing outputs.

Attention whose scores are capped by a tanh, sloped by the distance, or masked by a window, documents or a prefix, with
the log-sum-exp of every row (attend); the weight that each cached key has got from the queries, added to what it had
(weigh); the tokens of each layer, request and KV head that stay, by that weight, as a list of moves (select); and the
moves of their K and V rows, weights and positions to the slots that become free (move).

Head shapes are those of perf/cases.py, and its distributions: queries and keys N(0, 1.5^2) and N(0, 1), so that scores
after the 1/sqrt(head_dim) scale spread by about 1.5.  Gathered weights are spread log-normally, as attention's are.

Lengths, documents and prefixes belong to the case; the seed gives the values and the pages' order.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

SHAPES = {  # query heads, KV heads, head_dim
    "qwen2-0.5b": (14, 2, 64),
    "qwen2-7b": (28, 4, 128),
    "llama-3-8b": (32, 8, 128),
    "llama-3.2-1b": (32, 8, 64),
}
DTYPES = {"f16": torch.float16, "f32": torch.float32}
MAX_BYTES = 1.1e9    # K/V that the largest listed attention reads
MAX_FLOPS = 3.0e11   # and its products
MAX_GATHER = 1.2e9   # elements of K (or V) that the plain form gathers, padded to the longest request
MAX_SCORES = 1.2e9   # scores that it holds
MAX_TOKENS = 1.1e6   # tokens times KV heads over all layers, of the selections
MAX_MOVED = 1.2e8    # elements of the key pool in the moves


def _case(name, kind, model, dtype, **sizes):
    """kind: attend, weigh, select or move.  batch requests of lo..hi cached tokens, page tokens per page.
    attend, weigh: q_lo..q new tokens each; cap of the scores, slopes per head, window, documents of about that many
    tokens, a prefix of that share of a request's tokens; weigh: decay of what a key had.
    select, move: layers tables; keep tokens stay, the last `recent` and the first `first` of them in any case; steady: a
    cache that was cut before, and has grown by up to that many tokens since (0: a fresh prompt)."""
    c = dict(kind=kind, model=model, dtype=dtype, batch=1, lo=0, hi=0, page=16)
    if kind in ("attend", "weigh"):
        c.update(q=1, q_lo=0, cap=0.0, slopes=False, window=0, documents=0, prefix=0.0)
        if kind == "weigh":
            c.update(decay=1.0)
    else:
        c.update(layers=1, keep=0, recent=0, first=0, steady=0)
    c.update(sizes)
    if "q" in c:
        c["q_lo"] = c["q_lo"] or c["q"]
    return dict(name=name, **c) if name else c


def listed():
    return [
        # One chat with the smallest model, F32, capped scores: launches and latency.
        _case("attend f32 1x1 on 512", "attend", "qwen2-0.5b", "f32", lo=511, hi=511, cap=30.0),
        # A decode step of a server, chats of all lengths, scores that fall with the distance: bound by HBM.
        _case("attend f16 64x1 sloped", "attend", "llama-3-8b", "f16", batch=64, lo=300, hi=8192, slopes=True),
        # A layer with a window, at long contexts, capped.
        _case("attend f16 32x1 window", "attend", "llama-3-8b", "f16", batch=32, lo=16383, hi=16383, window=4096,
              cap=50.0),
        # A prefill step of four requests with capped scores: the products, the tanh and the exponential.
        _case("attend f16 4x256 capped", "attend", "qwen2-7b", "f16", batch=4, lo=2048, hi=2048, q=256, cap=50.0),
        # A long prompt of several documents that do not see each other.
        _case("attend f16 6000 documents", "attend", "llama-3-8b", "f16", q=6000, documents=1500),
        # F32 at odd sizes: prompts of which a prefix sees itself both ways, pages that end inside tiles.
        _case("attend f32 3x217 prefix", "attend", "qwen2-7b", "f32", batch=3, lo=300, hi=1001, q=217, q_lo=90,
              prefix=0.8, page=24),
        # The keys of a decode step get their share, chats of all lengths, F32.
        _case("weigh f32 16x1 ragged", "weigh", "llama-3.2-1b", "f32", batch=16, lo=200, hi=5000, page=24, decay=0.95),
        # Four prompts: what their last 32 tokens look at, capped scores.
        _case("weigh f16 4x32 on 6000", "weigh", "qwen2-7b", "f16", batch=4, lo=6000, hi=6000, q=32, cap=50.0),
        # One chat has grown a page beyond its budget, in 24 layers.
        _case("select 1 on 1040 24 layers", "select", "qwen2-0.5b", "f16", lo=1040, hi=1040, layers=24, keep=1024,
              recent=128, first=4, steady=16),
        # A batch of fresh prompts is cut, 8 layers.
        _case("select 16 ragged 8 layers", "select", "llama-3-8b", "f16", batch=16, lo=1500, hi=8000, layers=8,
              keep=1024, recent=64),
        # The same chat's rows.
        _case("move f16 1 on 1040 24 layers", "move", "qwen2-0.5b", "f16", lo=1040, hi=1040, layers=24, keep=1024,
              recent=128, first=4, steady=16),
        # The rows of fresh prompts, 4 layers.
        _case("move f16 8 on 3500 4 layers", "move", "llama-3-8b", "f16", batch=8, lo=3000, hi=3500, layers=4,
              keep=1024, recent=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "attend", "attend", "weigh", "weigh", "select", "move"])
        dtype = "f16" if rng.random() < 0.6 else "f32"
        s = dict(page=rng.choice([16, 16, 16, 32, 24, 8, 5]), batch=_log(rng, 1, 64))
        if kind in ("attend", "weigh"):
            s["q"] = 1 if rng.random() < 0.4 else _log(rng, 2, 1500 if kind == "attend" else 64)
            s["q_lo"] = s["q"] if rng.random() < 0.5 else rng.randint(1, s["q"])
            s["hi"] = _log(rng, 1, 16384)
            s["lo"] = s["hi"] if rng.random() < 0.4 else rng.randint(0, s["hi"])
            s["cap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
            s["slopes"] = rng.random() < 0.35
            s["window"] = _log(rng, 1, 5000) if rng.random() < 0.3 else 0
            mask = rng.random()
            if kind == "attend" and s["q"] > 64 and mask < 0.3:
                s["documents"] = _log(rng, 20, 2000)
            elif mask > 0.75:
                s["prefix"] = rng.choice([0.3, 0.9, 1.0])
            if kind == "weigh":
                s["decay"] = rng.choice([1.0, 1.0, 0.9])
        else:
            s["hi"] = _log(rng, 40, 20000)
            s["lo"] = s["hi"] if rng.random() < 0.4 else rng.randint(s["hi"] // 4, s["hi"])
            s["layers"] = rng.randint(1, 32)
            s["keep"] = rng.randint(max(8, s["lo"] // 8), max(8, s["lo"]))
            s["recent"] = rng.randint(0, s["keep"] // 2)
            s["first"] = rng.choice([0, 4])
            s["steady"] = rng.choice([0, 1, 16])
        c = _case("", kind, rng.choice(sorted(SHAPES)), dtype, **s)
        w = work(c)
        hq, hkv, d = SHAPES[c["model"]]
        _, n = _lengths(c)
        if kind in ("attend", "weigh"):
            fits = (len(n) * int(n.max()) * hkv * d <= MAX_GATHER and
                    len(n) * int(n.max()) * hq * c["q"] <= MAX_SCORES)
        else:
            tokens = sum(_tables(c)) * c["page"] * c["layers"] * hkv
            padded = len(n) * int(n.max()) * c["layers"] * hkv
            fits = padded <= 4 * MAX_TOKENS and tokens * (d if kind == "move" else 1) <= (
                MAX_MOVED if kind == "move" else MAX_TOKENS)
        if fits and w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS / (1 if dtype == "f16" else 8):
            return c


def _es(c):
    return 2 if c["dtype"] == "f16" else 4


def _lengths(c):
    """(new tokens, total tokens) per request."""
    rng = np.random.default_rng([c["batch"], c["lo"], c["hi"], c.get("q", 0), c.get("keep", 0)])
    cached = rng.integers(c["lo"], c["hi"], size=c["batch"], endpoint=True).astype(np.int32)
    cached[-1] = c["hi"]
    if "q" in c:
        q = rng.integers(c["q_lo"], c["q"], size=c["batch"], endpoint=True).astype(np.int32)
        q[-1] = c["q"]
        return q, (cached + q).astype(np.int32)
    if c["steady"]:  # requests at their budget, and grown since
        cached = c["keep"] + rng.integers(1, c["steady"], size=c["batch"], endpoint=True).astype(np.int32)
    return None, cached


def _tables(c):
    """Pages of every request, of one layer."""
    return [math.ceil(int(n) / c["page"]) for n in _lengths(c)[1]]


def _first_keys(c):
    """Per packed query token: where its document starts."""
    q, n = _lengths(c)
    rng = np.random.default_rng([c["batch"], c["hi"], c["q"], c["documents"]])
    out = []
    for new, total in zip(q.tolist(), n.tolist()):
        starts = [0]
        while starts[-1] < total:
            starts.append(starts[-1] + int(rng.integers(1, 2 * c["documents"])))
        starts = np.array(starts)
        at = np.arange(total - new, total)
        out.append(starts[np.searchsorted(starts, at, side="right") - 1])
    return np.concatenate(out).astype(np.int32)


def _prefix_lens(c):
    return np.maximum(1, (_lengths(c)[1] * c["prefix"]).astype(np.int32))


def _ranges(c):
    """Per packed query token: (request, position, first key seen, key past the last one seen)."""
    q, n = _lengths(c)
    b = np.repeat(np.arange(c["batch"]), q)
    start = np.concatenate([[0], np.cumsum(q)])[:-1]
    pos = (n - q)[b] + np.arange(int(q.sum())) - start[b]
    lo, hi = np.zeros_like(pos), pos + 1
    if c["documents"]:
        lo = np.maximum(lo, _first_keys(c))
    if c["window"]:
        lo = np.maximum(lo, pos - c["window"] + 1)
    if c["prefix"]:
        hi = np.maximum(hi, _prefix_lens(c)[b])
    return b, pos, lo, hi


def work(c):
    hq, hkv, d = SHAPES[c["model"]]
    _, n = _lengths(c)
    if c["kind"] == "select":  # weight and position of every token, the moves
        moves = _moves_expected(c) * c["layers"] * hkv
        return {"bytes": int(n.sum()) * c["layers"] * hkv * 8 + moves * 8 + 4 * c["layers"] * sum(_tables(c)), "flops": 0}
    if c["kind"] == "move":
        return {"bytes": _moves_expected(c) * c["layers"] * hkv * (2 * (2 * d * _es(c) + 8) + 8), "flops": 0}
    b, _, lo, hi = _ranges(c)
    first, last = np.full(c["batch"], 1 << 30), np.zeros(c["batch"], int)
    np.minimum.at(first, b, lo)
    np.maximum.at(last, b, hi)
    keys = int(np.maximum(last - first, 0).sum())
    pairs = int(np.maximum(hi - lo, 0).sum())
    row = hkv * d * _es(c)
    if c["kind"] == "attend":
        return {"bytes": keys * row * 2 + len(b) * hq * (d * _es(c) * 2 + 4) + 4 * (keys // c["page"]),
                "flops": 4 * hq * d * pairs}
    touched = keys if c["decay"] == 1.0 else int(n.sum())
    return {"bytes": keys * row + touched * hkv * 8 + len(b) * hq * (d * _es(c) + 4) + 4 * (keys // c["page"]),
            "flops": 2 * hq * d * pairs}


def _moves_expected(c):
    """Moves of one layer and head over all requests: of the tokens that stay beside the protected ones, as many as lie
    past the new length where weights do not go by slots."""
    total = 0
    for n in _lengths(c)[1].tolist():
        if n > c["keep"]:
            total += int((n - c["keep"]) * (c["keep"] - c["recent"]) / n) + min(c["recent"], n - c["keep"])
    return total


def _inputs(c, seed):
    """Host tables and device values of a case."""
    hq, hkv, d = SHAPES[c["model"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std, mean=0.0, dtype=DTYPES[c["dtype"]]):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)

    need, layers = _tables(c), c.get("layers", 1)
    pages = layers * sum(need)
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.zeros((layers, c["batch"], max(need)), np.int32)
    used = 0
    for layer in range(layers):
        for b in range(c["batch"]):
            table[layer, b, :need[b]] = order[used:used + need[b]]
            used += need[b]
    q_lens, seq_lens = _lengths(c)
    t = dict(seq_lens=seq_lens)
    pool = (pages, 1, hkv, c["page"], d)
    if c["kind"] in ("attend", "weigh"):
        tokens = int(q_lens.sum())
        t.update(table=table[0], q_lens=q_lens, cu=np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32),
                 q=normal((hq, tokens, d), 1.5), key_pool=normal(pool, 1.0))
        if c["slopes"]:
            t["slopes"] = 2.0 ** (-8.0 * np.arange(1, hq + 1, dtype=np.float32) / hq)
        if c["documents"]:
            t["first_keys"] = _first_keys(c)
        if c["prefix"]:
            t["prefix_lens"] = _prefix_lens(c)
        if c["kind"] == "attend":
            t["value_pool"] = normal(pool, 1.0)
        else:
            t["weights"] = normal((pages, hkv, c["page"]), 2.0, dtype=torch.float32).exp_()
        return t
    weights = normal((pages, hkv, c["page"]), 2.0, dtype=torch.float32).exp_()
    grown = seq_lens - c["keep"] if c["steady"] else seq_lens  # tokens since the cache was last cut
    kept = seq_lens - grown
    rng = np.random.default_rng(seed + 1)
    past = (rng.integers(0, 3000, size=c["batch"]) if c["steady"] else np.zeros(c["batch"])).astype(np.int32)
    # Positions of the tokens that stayed then: some of those before the grown ones, in any order.
    positions = torch.full((pages, hkv, c["page"]), -1, dtype=torch.int32, device="cuda")
    if c["steady"]:
        for b in range(c["batch"]):
            span = int(kept[b] + past[b])
            some = torch.rand((layers, hkv, span), device="cuda", generator=gen).argsort(-1)[..., :int(kept[b])].int()
            slot = torch.arange(int(kept[b]), device="cuda")
            ids = torch.from_numpy(table[:, b]).cuda().long()[:, slot // c["page"]]
            positions[ids, :, slot % c["page"]] = some.transpose(1, 2)
    t.update(table=table, weights=weights, positions=positions, kept_lens=kept.astype(np.int32),
             keep_lens=np.full(c["batch"], c["keep"], np.int32), next_positions=(seq_lens + past).astype(np.int32))
    if c["kind"] == "move":
        t.update(key_pool=normal(pool, 1.0), value_pool=normal(pool, 1.0))
    return t


def prepare(c, seed):
    t = _inputs(c, seed)
    s = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in t.items()}
    _, hkv, _ = SHAPES[c["model"]]
    s["case"] = c
    s["max_len"] = int(t["seq_lens"].max())
    if c["kind"] in ("attend", "weigh"):  # what the scheduler that built the tables has on the host
        s.update(max_q=int(t["q_lens"].max()), host_seq_lens=t["seq_lens"], host_cu=t["cu"])
        s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
        if c["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
        else:  # what the attention call on these queries gave
            s["lse"].copy_(_row_lse(s))
        return s
    most = max(1, int(np.minimum(t["keep_lens"], t["seq_lens"] - t["keep_lens"]).max()))
    rows = (c["layers"], c["batch"], hkv)
    s["moves"] = torch.zeros(rows + (most, 2), dtype=torch.int32, device="cuda")
    s["num_moves"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s["new_lens"] = torch.zeros(c["batch"], dtype=torch.int32, device="cuda")
    if c["kind"] == "move":
        _select(s)
    return s


# ---- the framework's calls -------------------------------------------------

def _own_call(s):
    """The call of one layer (or step), its argument block and workspace made once and kept, as a runner keeps them."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-vllm-rs_amd"))
    import mvr_score as S

    c = s["case"]
    if c["kind"] in ("attend", "weigh"):
        rules = dict(cap=c["cap"], slopes=s.get("slopes"), window=c["window"], first_keys=s.get("first_keys"),
                     prefix_lens=s.get("prefix_lens"), max_q_len=s["max_q"], max_seq_len=s["max_len"],
                     seq_lens_host=s["host_seq_lens"], cu_q_lens_host=s["host_cu"])
    if c["kind"] == "attend":
        a = S.make_scored_call(s["q"], s["key_pool"], s["value_pool"], s["table"], s["seq_lens"], s["cu"], s["out"],
                               s["lse"], **rules)
        return a, dict(out=s["out"], lse=s["lse"])
    if c["kind"] == "weigh":
        a = S.make_weights_call(s["q"], s["lse"], s["key_pool"], s["weights"], s["table"], s["seq_lens"], s["cu"],
                                decay=c["decay"], **rules)
        return a, dict(weights=s["weights"])
    if c["kind"] == "select":
        a = S.make_select_call(s["weights"], s["positions"], s["table"], s["seq_lens"], s["next_positions"],
                               s["kept_lens"], s["keep_lens"], s["moves"], s["num_moves"], s["new_lens"],
                               recent=c["recent"], first=c["first"], max_seq_len=s["max_len"])
        return a, {k: s[k] for k in ("moves", "num_moves", "new_lens", "positions")}
    a = S.make_move_call(s["key_pool"], s["value_pool"], s["weights"], s["positions"], s["table"], s["moves"],
                         s["num_moves"])
    return a, {k: s[k] for k in ("key_pool", "value_pool", "weights", "positions")}


# ---- plain forms -----------------------------------------------------------

def _token_index(s):
    """(request, index within the request) of every packed token."""
    t = torch.arange(s["q"].shape[1], device="cuda")
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return b, t - s["cu"].long()[b]


def _gather(s, pool):
    """[B, Hkv, longest, D] of a pool in 32 bits."""
    batch, hkv, d = s["table"].shape[0], pool.shape[2], pool.shape[4]
    x = pool[s["table"].long(), 0].float()  # [B, pages, Hkv, P, D]
    return x.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :s["max_len"]]


def _scores(s):
    """Scores [B, Hkv, G, longest query, longest] of what each query sees, -inf elsewhere."""
    c, q = s["case"], s["q"]
    hq, tokens, d = q.shape
    hkv = s["key_pool"].shape[2]
    batch, qm, length = s["table"].shape[0], s["max_q"], s["max_len"]
    cu, n = s["cu"].long(), s["seq_lens"].long()
    index = (cu[:-1, None] + torch.arange(qm, device="cuda")).clamp(max=tokens - 1)  # [B, qm]
    rows = q[:, index].float().view(hkv, hq // hkv, batch, qm, d).permute(2, 0, 1, 3, 4)
    rows = rows.reshape(batch, hkv, hq // hkv * qm, d)
    x = rows @ _gather(s, s["key_pool"]).transpose(-1, -2).contiguous()
    x = x.mul_(1.0 / math.sqrt(d)).view(batch, hkv, hq // hkv, qm, length)
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    key = torch.arange(length, device="cuda")
    pos = (n - (cu[1:] - cu[:-1]))[:, None] + torch.arange(qm, device="cuda")  # [B, qm]
    if c["slopes"]:
        away = (key - pos[..., None]).abs().float()  # [B, qm, L]
        x.addcmul_(s["slopes"].view(1, hkv, -1, 1, 1), away[:, None, None], value=-1.0)
    last = pos + 1
    if c["prefix"]:
        last = torch.maximum(last, torch.minimum(s["prefix_lens"].long(), n)[:, None])
    seen = key < last[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    if c["documents"]:
        seen &= key >= s["first_keys"].long()[index][..., None]
    return x.masked_fill_(~seen[:, None, None], -math.inf)


def _unpack(s, x):
    """[B, Hkv, G, longest query, ...] to the packed [Hq, tokens, ...]."""
    b, i = _token_index(s)
    return x.flatten(1, 2)[b, :, i].transpose(0, 1)


def _row_lse(s):
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    return _unpack(s, (x.sub_(top).exp_().sum(-1).log() + top[..., 0]))


def _attend(s):
    x = _scores(s)
    batch, hkv, group, qm, length = x.shape
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total)).view(batch, hkv, group * qm, length)
    o = (p @ _gather(s, s["value_pool"])).view(batch, hkv, group, qm, -1)
    s["out"].copy_(_unpack(s, o))
    s["lse"].copy_(_unpack(s, (total.log() + top)[..., 0]))
    return dict(out=s["out"], lse=s["lse"])


def _weigh(s):
    c, pool, page = s["case"], s["weights"], s["key_pool"].shape[3]
    cu, n = s["cu"].long(), s["seq_lens"].long()
    batch, qm, length = s["table"].shape[0], s["max_q"], s["max_len"]
    x = _scores(s)
    index = (cu[:-1, None] + torch.arange(qm, device="cuda")).clamp(max=s["q"].shape[1] - 1)
    real = torch.arange(qm, device="cuda") < (cu[1:] - cu[:-1])[:, None]  # [B, qm]
    lse = s["lse"][:, index].view(x.shape[1], x.shape[2], batch, qm).permute(2, 0, 1, 3)
    lse = torch.where(real[:, None, None], lse, math.inf)  # rows past a request's last count nothing
    got = x.sub_(lse[..., None]).exp_().sum((2, 3))  # [B, Hkv, L]
    key = torch.arange(length, device="cuda")
    b, slot = torch.nonzero(key < n[:, None], as_tuple=True)
    pages = s["table"].long()[b, slot // page]
    had = pool[pages, :, slot % page] * c["decay"]
    had = torch.where((slot < (n - (cu[1:] - cu[:-1]))[b])[:, None], had, 0.0)
    pool[pages, :, slot % page] = had + got.transpose(1, 2)[b, slot]
    return dict(weights=pool)


def _select(s):
    c, table = s["case"], s["table"].long()
    layers, batch, _ = table.shape
    page, length, most = s["weights"].shape[2], s["max_len"], s["moves"].shape[3]
    n, kept, keep = s["seq_lens"].long(), s["kept_lens"].long(), s["keep_lens"].long()
    slot = torch.arange(length, device="cuda")
    pages = table[:, :, slot // page]  # [layers, B, L]
    new = (s["next_positions"].long() - n)[:, None] + slot  # [B, L]
    fresh = (slot >= kept[:, None]) & (slot < n[:, None])
    pos = s["positions"][pages, :, slot % page]  # [layers, B, L, Hkv]
    pos = torch.where(fresh[None, ..., None], new.int()[None, ..., None], pos)
    li, bi, si = torch.nonzero(fresh[None].expand(layers, -1, -1), as_tuple=True)
    s["positions"][pages[li, bi, si], :, si % page] = pos[li, bi, si]
    w = s["weights"][pages, :, slot % page]
    edge = (s["next_positions"].long() - c["recent"])[None, :, None, None]
    w = torch.where((pos < c["first"]) | (pos >= edge), math.inf, w)
    w = torch.where((slot < n[:, None])[None, ..., None], w, -math.inf).transpose(2, 3)  # [layers, B, Hkv, L]
    order = torch.argsort(w, dim=-1, descending=True, stable=True)
    keep = torch.minimum(keep, n)[None, :, None, None]
    stays = torch.zeros_like(order, dtype=torch.bool).scatter_(-1, order, (slot < keep).expand(order.shape))
    goes_in, comes_from = ~stays & (slot < keep), stays & (slot >= keep)
    for side, taken in ((0, comes_from), (1, goes_in)):
        where = taken.nonzero(as_tuple=True)
        s["moves"][where[0], where[1], where[2], (taken.cumsum(-1) - 1)[where], side] = where[3].int()
    s["num_moves"].copy_(goes_in.sum(-1))
    s["new_lens"].copy_(keep.flatten())
    return {k: s[k] for k in ("moves", "num_moves", "new_lens", "positions")}


def _move(s):
    table, page = s["table"].long(), s["weights"].shape[2]
    taken = torch.arange(s["moves"].shape[3], device="cuda") < s["num_moves"][..., None]
    layer, b, h, j = taken.nonzero(as_tuple=True)
    at, to = s["moves"][layer, b, h, j].long().unbind(-1)
    source, target = table[layer, b, at // page], table[layer, b, to // page]
    for pool in (s["key_pool"], s["value_pool"]):
        pool[target, 0, h, to % page] = pool[source, 0, h, at % page]
    for pool in (s["weights"], s["positions"]):
        pool[target, h, to % page] = pool[source, h, at % page]
    return {k: s[k] for k in ("key_pool", "value_pool", "weights", "positions")}


def run(s):
    if own:
        if "call" not in s:
            s["call"], s["outputs"] = _own_call(s)
        s["call"]()
        return s["outputs"]
    return {"attend": _attend, "weigh": _weigh, "select": _select, "move": _move}[s["case"]["kind"]](s)


# ---- from the definitions, in 64 bits --------------------------------------

def _exact_rows(c, t):
    """For every request and KV head: (request, head, its query heads and tokens, page ids, scores [G, q, n] in 64 bits)."""
    hq, hkv, d = SHAPES[c["model"]]
    group = hq // hkv
    owner, pos, lo, hi = _ranges(c)
    for b in range(c["batch"]):
        n = int(t["seq_lens"][b])
        mine = np.flatnonzero(owner == b)
        tokens = slice(int(mine[0]), int(mine[-1]) + 1)
        ids = torch.from_numpy(t["table"][b, :math.ceil(n / c["page"])]).cuda().long()
        key = np.arange(n)
        hidden = torch.from_numpy((key < lo[mine][:, None]) | (key >= hi[mine][:, None])).cuda()
        away = torch.from_numpy(pos[mine]).cuda()[:, None] - torch.arange(n, device="cuda")
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            k = t["key_pool"][ids, 0, h].reshape(-1, d)[:n].double()
            x = torch.matmul(t["q"][heads, tokens].double().reshape(-1, d), k.t()).view(group, -1, n) / math.sqrt(d)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["slopes"]:
                x = x - torch.from_numpy(t["slopes"][heads]).cuda().double()[:, None, None] * away.abs()
            yield b, h, heads, tokens, ids, x.masked_fill(hidden, -math.inf)


def _exact_attend(c, t):
    d = SHAPES[c["model"]][2]
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(t["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, h, heads, tokens, ids, x in _exact_rows(c, t):
        n = x.shape[-1]
        v = t["value_pool"][ids, 0, h].reshape(-1, d)[:n].double()
        lse[heads, tokens] = torch.logsumexp(x, -1)
        p = torch.softmax(x, -1).nan_to_num(0.0)
        out[heads, tokens] = torch.matmul(p.view(-1, n), v).view(x.shape[0], x.shape[1], d)
    return dict(out=out, lse=lse)


def _exact_weigh(c, t, lse):
    pool = t["weights"].double()
    for b, h, heads, tokens, ids, x in _exact_rows(c, t):
        n, page = x.shape[-1], c["page"]
        got = torch.exp(x - lse[heads, tokens].double()[..., None]).sum((0, 1))
        rows = pool[ids, h].reshape(-1)
        old = int(t["seq_lens"][b] - t["q_lens"][b])
        rows[:old] *= c["decay"]
        rows[old:n] = 0.0
        rows[:n] += got
        pool[ids, h] = rows.view(-1, page)
    return dict(weights=pool)


def _exact_move(c, s):
    pools = {k: s[k].double() for k in ("key_pool", "value_pool", "weights")}
    page, table = c["page"], s["table"].long()
    layers, batch, hkv = s["num_moves"].shape
    counts = s["num_moves"].cpu()
    for layer in range(layers):
        for b in range(batch):
            for h in range(hkv):
                m = s["moves"][layer, b, h, :int(counts[layer, b, h])].long()
                source, target = table[layer, b, m[:, 0] // page], table[layer, b, m[:, 1] // page]
                for pool in (pools["key_pool"][:, 0], pools["value_pool"][:, 0], pools["weights"]):
                    pool[target, h, m[:, 1] % page] = pool[source, h, m[:, 0] % page]
    return dict(pools, positions=None)


def exact(c, seed):
    if c["kind"] == "select":
        return None
    if c["kind"] == "attend":
        return _exact_attend(c, _inputs(c, seed))
    s = prepare(c, seed)
    if c["kind"] == "move":
        return _exact_move(c, s)
    return _exact_weigh(c, _inputs(c, seed), s["lse"])
