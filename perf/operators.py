"""The calls of speculative decoding with a tree of drafted tokens, for timing and for comparing outputs.

One step of such a server, per layer: the drafts' queries and keys are normalised and rotated, and keys and values
appended to their pages (append); the drafts attend the cache and their ancestors (tree); once per step the accepted
path's rows move to the front of the drafts' slots, in the tables of every layer (compact), and a request that is
forked, or whose last page is shared, gets copies of pages (copy).  Head shapes are those of perf/cases.py, and its
distributions: queries and keys N(0, 1.5^2) and N(0, 1), so that scores after the 1/sqrt(head_dim) scale spread by
about 1.5.

Lengths and the trees' shapes belong to the case; the seed gives the values and the pages' order.
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
    "llama-3.2-3b": (24, 8, 128),
}
DTYPES = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
MAX_BYTES = 2.2e9      # K/V of the largest listed tree call
MAX_FLOPS = 3.3e11     # and its products
MAX_GATHER = 1.2e9     # elements of K (or V) that the plain form gathers, padded to the longest request
MAX_MOVED = 1.2e8      # elements of the key pool in the calls that update it


def _case(name, kind, model, dtype, **sizes):
    """kind: tree, append, compact or copy.  batch requests of lo..hi cached tokens with nodes_lo..nodes new ones each
    (a chain or a tree of drafts where tree is set), page tokens per page.  compact: the accepted path of each request
    in layers tables.  copy: copies pages, the first 1..page tokens of each where partial is set."""
    c = dict(kind=kind, model=model, dtype=dtype, batch=1, lo=0, hi=0, nodes=1, nodes_lo=0, page=16, tree=True,
             interleaved=False, layers=1, copies=0, partial=False)
    c.update(sizes)
    c["nodes_lo"] = c["nodes_lo"] or c["nodes"]
    return dict(name=name, **c) if name else c


def listed():
    return [
        # One chat with the smallest model, F32, a few drafts: launches and latency.
        _case("tree f32 1x8 on 512", "tree", "qwen2-0.5b", "f32", batch=1, lo=512, hi=512, nodes=8),
        # A verification step of a server, contexts of all lengths, small trees of unequal sizes: bound by HBM.
        _case("tree f16 16x16 ragged", "tree", "llama-3-8b", "f16", batch=16, lo=1024, hi=16384, nodes=16,
              nodes_lo=5),
        # A few users, wide trees: the products weigh as much as the reads.
        _case("tree f16 4x64 on 2048", "tree", "qwen2-7b", "f16", batch=4, lo=2048, hi=2048, nodes=64),
        # A full batch at long contexts.
        _case("tree f16 64x32 on 8192", "tree", "llama-3-8b", "f16", batch=64, lo=8192, hi=8192, nodes=32),
        # F32 at odd sizes, pages that end inside tiles.
        _case("tree f32 3x21 ragged", "tree", "llama-3.2-3b", "f32", batch=3, lo=300, hi=3001, nodes=21, nodes_lo=7,
              page=24),
        # One decode step of a busy server: a token per request.
        _case("append f16 64x1", "append", "llama-3-8b", "f16", batch=64, lo=100, hi=900, nodes=1, tree=False),
        # A prefill step of four requests.
        _case("append f16 4x256", "append", "qwen2-7b", "f16", batch=4, lo=700, hi=700, nodes=256, tree=False),
        # Trees of drafts, F32, the other pairing, pages of an odd size.
        _case("append f32 16x26 trees", "append", "llama-3.2-1b", "f32", batch=16, lo=33, hi=700, nodes=26,
              nodes_lo=9, page=5, interleaved=True),
        # One chat: a short path in the tables of 24 layers.
        _case("compact f32 1x8 24 layers", "compact", "qwen2-0.5b", "f32", batch=1, lo=90, hi=90, nodes=8, layers=24),
        # A batch after a step of large trees, 32 layers.
        _case("compact f16 32x64 32 layers", "compact", "llama-3-8b", "f16", batch=32, lo=30, hi=70, nodes=64,
              nodes_lo=20, layers=32),
        # Two samples fork off one prompt: the last pages of 32 layers, partly filled.
        _case("copy f16 64 partial", "copy", "llama-3-8b", "f16", copies=64, partial=True),
        # A batch is forked: whole pages of every layer.
        _case("copy f16 3500 pages", "copy", "qwen2-7b", "f16", copies=3500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["tree", "tree", "tree", "append", "compact", "copy"])
        dtype = "f16" if rng.random() < 0.7 else "f32"
        s = dict(page=rng.choice([16, 16, 16, 32, 24, 8, 5]))
        if kind == "copy":
            s["copies"] = _log(rng, 1, 4000)
            s["partial"] = rng.random() < 0.5
        else:
            s["batch"] = _log(rng, 1, 64)
            s["nodes"] = _log(rng, 6 if kind == "compact" else 1, 128)
            s["nodes_lo"] = s["nodes"] if rng.random() < 0.4 else rng.randint(1, s["nodes"])
            s["hi"] = _log(rng, 16, 16384 if kind == "tree" else 900 if kind == "append" else 100)
            s["lo"] = s["hi"] if rng.random() < 0.4 else rng.randint(max(1, s["hi"] // 9), s["hi"])
            s["tree"] = kind == "compact" or rng.random() < 0.8
            s["interleaved"] = kind == "append" and rng.random() < 0.3
            s["layers"] = rng.randint(1, 32) if kind == "compact" else 1
        c = _case("", kind, rng.choice(sorted(SHAPES)), dtype, **s)
        w = work(c)
        _, hkv, d = SHAPES[c["model"]]
        if kind == "tree":
            n = _lengths(c)[1]
            fits = len(n) * int(n.max()) * hkv * d <= MAX_GATHER
        else:
            fits = _pool_pages(c) * c["page"] * hkv * d <= MAX_MOVED
        if fits and w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS / (1 if dtype == "f16" else 8):
            return c


def _es(c):
    return 2 if c["dtype"] == "f16" else 4


def _lengths(c):
    """(new tokens, total tokens) per request; seq_lens counts the new ones."""
    rng = np.random.default_rng([c["batch"], c["lo"], c["hi"], c["nodes"]])
    q = rng.integers(c["nodes_lo"], c["nodes"], size=c["batch"], endpoint=True).astype(np.int32)
    q[-1] = c["nodes"]
    cached = rng.integers(c["lo"], c["hi"], size=c["batch"], endpoint=True).astype(np.int32)
    return q, (cached + q).astype(np.int32)


def _trees(c):
    """Parent of every new token within its request (-1: the root, the first one).  Drafts grow from recent nodes and
    near the root more often, as a tree of a draft model's best continuations; a chain where the case has no trees."""
    rng = random.Random(c["batch"] * 1000003 + c["nodes"] * 1009 + c["hi"])
    parents = []
    for q in _lengths(c)[0].tolist():
        p = [-1] + [i - 1 if not c["tree"] or rng.random() < 0.35 else rng.randrange(max(0, i // 2 - 4), i)
                    for i in range(1, q)]
        parents.append(p)
    return parents


def _ancestors(parent):
    """[q, q] truth values: node i sees itself and its ancestors."""
    seen = np.zeros((len(parent), len(parent)), bool)
    for i, p in enumerate(parent):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def _path(parent):
    """The accepted path: from the root to the last node of the deepest branch that ends in the tree's second half."""
    depth = []
    for p in parent:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    at = max(range(len(parent) // 2, len(parent)), key=lambda i: depth[i])
    path = []
    while at >= 0:
        path.append(at)
        at = parent[at]
    return path[::-1]


def _tables(c):
    """Block tables needed: layers tables of every request's pages."""
    return [math.ceil(int(n) / c["page"]) for n in _lengths(c)[1]]


def _pool_pages(c):
    return 2 * c["copies"] + 3 if c["kind"] == "copy" else c["layers"] * sum(_tables(c))


def _copied(c):
    """Tokens that each copy moves."""
    if not c["partial"]:
        return np.full(c["copies"], c["page"], np.int32)
    return np.random.default_rng([c["copies"], c["page"]]).integers(1, c["page"], size=c["copies"],
                                                                    endpoint=True).astype(np.int32)


def work(c):
    hq, hkv, d = SHAPES[c["model"]]
    row = hkv * d * _es(c)  # K or V of one token
    if c["kind"] == "copy":
        return {"bytes": int(_copied(c).sum()) * row * 2 * 2 + c["copies"] * 12, "flops": 0}
    q, n = _lengths(c)
    tokens = int(q.sum())
    if c["kind"] == "append":  # q, k, v in and out, one cos and one sin row, a position and a page id
        return {"bytes": tokens * ((hq + 2 * hkv) * d * _es(c) * 2 + d * _es(c) + 8) + 2 * d * _es(c),
                "flops": tokens * (hq + hkv) * d * 6}
    if c["kind"] == "compact":
        moved = sum(j != s for p in _trees(c) for j, s in enumerate(_path(p)))
        return {"bytes": c["layers"] * moved * row * 2 * 2 + 12 * c["batch"], "flops": 0}
    pairs = sum(len(p) * (int(b) - int(a)) + int(_ancestors(p).sum()) for p, a, b in zip(_trees(c), q, n))
    ids = sum(_tables(c))
    masks = tokens * math.ceil(c["nodes"] / 32)
    return {"bytes": int(n.sum()) * row * 2 + tokens * hq * d * _es(c) * 2 + 4 * (ids + masks),
            "flops": 4 * hq * d * pairs}


def _inputs(c, seed):
    """Host tables and device values of a case."""
    hq, hkv, d = SHAPES[c["model"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std, mean=0.0):
        return torch.empty(shape, dtype=DTYPES[c["dtype"]], device="cuda").normal_(mean, std, generator=gen)

    pages = _pool_pages(c)
    pool = (pages, 1, hkv, c["page"], d)
    t = dict(key_pool=normal(pool, 1.0), value_pool=normal(pool, 1.0))
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    if c["kind"] == "copy":
        return dict(t, src=order[:c["copies"]], dst=order[c["copies"]:2 * c["copies"]],
                    tokens=_copied(c) if c["partial"] else None)
    q_lens, seq_lens = _lengths(c)
    need = _tables(c)
    table = np.zeros((c["layers"], c["batch"], max(need)), np.int32)
    used = 0
    for layer in range(c["layers"]):
        for b in range(c["batch"]):
            table[layer, b, :need[b]] = order[used:used + need[b]]
            used += need[b]
    parents = _trees(c)
    tokens = int(q_lens.sum())
    t.update(table=table if c["kind"] == "compact" else table[0], q_lens=q_lens, seq_lens=seq_lens,
             cu=np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32))
    if c["kind"] == "compact":
        paths = [_path(p) for p in parents]
        accepted = np.zeros((c["batch"], max(map(len, paths))), np.int32)
        for b, p in enumerate(paths):
            accepted[b, :len(p)] = p
        return dict(t, accepted=accepted, accepted_lens=np.array([len(p) for p in paths], np.int32))
    t["q"] = normal((hq, tokens, d), 1.5)
    if c["kind"] == "append":
        t.update(k=normal((hkv, tokens, d), 1.0), v=normal((hkv, tokens, d), 1.0), q_weight=normal((d,), 0.2, 1.0),
                 k_weight=normal((d,), 0.2, 1.0))
        length = int(seq_lens.max())
        angle = np.arange(length)[:, None] * 1000000.0 ** (-np.arange(0, d, 2) / d)[None, :]
        for name, f in (("cos", np.cos), ("sin", np.sin)):
            t[name] = torch.from_numpy(f(angle)).to("cuda", DTYPES[c["dtype"]])
        positions = []
        for p, cached in zip(parents, (seq_lens - q_lens).tolist()):
            depth = _ancestors(p).sum(1) - 1
            positions.extend((cached + depth).tolist())
        t["positions"] = np.array(positions, np.int32)
        return t
    words = math.ceil(c["nodes"] / 32)
    bits = np.zeros((tokens, words * 32), np.uint8)
    at = 0
    for p in parents:
        bits[at:at + len(p), :len(p)] = _ancestors(p)
        at += len(p)
    t["masks"] = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    return t


def prepare(c, seed):
    t = _inputs(c, seed)
    s = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in t.items()}
    s["case"] = c
    if c["kind"] != "copy":  # what the scheduler that built the tables has on the host
        s.update(max_q=int(t["q_lens"].max()), max_len=int(t["seq_lens"].max()), host_seq_lens=t["seq_lens"],
                 host_cu=t["cu"])
    if c["kind"] == "compact":
        s["new_lens"] = torch.zeros(c["batch"], dtype=torch.int32, device="cuda")
    elif c["kind"] != "copy":
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- the framework's calls -------------------------------------------------

def _own_call(s):
    """The call of one layer (or step), its argument block and workspace made once and kept, as a runner keeps them."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-vllm-rs_amd"))
    import mvr_draft as D

    kind = s["case"]["kind"]
    if kind == "tree":
        a = D.make_tree_call(s["q"], s["key_pool"], s["value_pool"], s["table"], s["seq_lens"], s["cu"], s["masks"],
                             s["out"], max_q_len=s["max_q"], max_seq_len=s["max_len"],
                             sum_seq_lens=int(s["host_seq_lens"].sum()), seq_lens_host=s["host_seq_lens"],
                             cu_q_lens_host=s["host_cu"])
        return a, s["out"]
    if kind == "append":
        a = D.make_norm_rope_append_call(
            s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["table"], s["seq_lens"],
            s["cu"], s["key_pool"], s["value_pool"], s["out"], eps=EPS, positions=s["positions"],
            max_seq_len=s["max_len"],
            rope_type=D.ROPE_INTERLEAVED if s["case"]["interleaved"] else D.ROPE_NEOX)
        return a, dict(q=s["out"], key_pool=s["key_pool"], value_pool=s["value_pool"])
    if kind == "compact":
        a = D.make_compact_drafts_call(s["key_pool"], s["value_pool"], s["table"], s["seq_lens"], s["cu"],
                                       s["accepted"], s["accepted_lens"], s["new_lens"], max_seq_len=s["max_len"])
        return a, dict(key_pool=s["key_pool"], value_pool=s["value_pool"], lens=s["new_lens"])
    a = D.make_copy_pages_call(s["key_pool"], s["value_pool"], s["src"], s["dst"], s["tokens"])
    return a, dict(key_pool=s["key_pool"], value_pool=s["value_pool"])


# ---- plain forms -----------------------------------------------------------

def _token_index(s):
    """(request, index within the request) of every packed token."""
    t = torch.arange(s["q"].shape[1], device="cuda")
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return b, t - s["cu"].long()[b]


def _tree(s):
    q, pool = s["q"], s["key_pool"]
    hq, tokens, d = q.shape
    hkv, page = pool.shape[2], pool.shape[3]
    batch, qm, length = s["table"].shape[0], s["max_q"], s["max_len"]
    cu, n = s["cu"].long(), s["seq_lens"].long()
    index = (cu[:-1, None] + torch.arange(qm, device="cuda")).clamp(max=tokens - 1)  # [B, qm]
    rows = q[:, index].float().view(hkv, hq // hkv, batch, qm, d).permute(2, 0, 1, 3, 4)
    rows = rows.reshape(batch, hkv, hq // hkv * qm, d)

    def gather(x):
        x = x[s["table"].long(), 0].float()  # [B, pages, Hkv, P, D]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :length]

    scores = rows @ gather(pool).transpose(-1, -2).contiguous() * (1.0 / math.sqrt(d))
    key = torch.arange(length, device="cuda")
    prefix = (n - (cu[1:] - cu[:-1]))[:, None]  # [B, 1]
    slot = key - prefix  # [B, L]
    drafted = (slot >= 0) & (key < n[:, None])
    slot = slot.clamp(0, 32 * s["masks"].shape[1] - 1)
    word = s["masks"][index[:, :, None], (slot // 32)[:, None, :]]  # [B, qm, L]
    bit = (word >> (slot % 32)[:, None, :]) & 1
    visible = (key < prefix)[:, None, :] | (drafted[:, None, :] & (bit != 0))
    scores = scores.view(batch, hkv, hq // hkv, qm, length)
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(batch, hkv, -1, length)
    o = (p @ gather(s["value_pool"])).view(batch, hq, qm, d)
    b, i = _token_index(s)
    s["out"].copy_(o[b, :, i].transpose(0, 1))
    return s["out"]


def _append(s):
    d, page = s["q"].shape[2], s["key_pool"].shape[3]
    pos = s["positions"].long()
    cos, sin = s["cos"][pos].float(), s["sin"][pos].float()  # [T, D/2]

    def norm_rope(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if s["case"]["interleaved"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    s["out"].copy_(norm_rope(s["q"], s["q_weight"]))
    b, i = _token_index(s)
    cu = s["cu"].long()
    at = s["seq_lens"].long()[b] - (cu[b + 1] - cu[b]) + i
    pages = s["table"].long()[b, at // page]
    s["key_pool"][pages, 0, :, at % page] = norm_rope(s["k"], s["k_weight"]).transpose(0, 1).to(s["k"].dtype)
    s["value_pool"][pages, 0, :, at % page] = s["v"].transpose(0, 1)
    return dict(q=s["out"], key_pool=s["key_pool"], value_pool=s["value_pool"])


def _compact(s):
    page = s["key_pool"].shape[3]
    cu, n, table = s["cu"].long(), s["seq_lens"].long(), s["table"].long()  # table [layers, B, pages]
    first = n - (cu[1:] - cu[:-1])
    batch, most = s["accepted"].shape
    j = torch.arange(most, device="cuda").expand(batch, most)
    b = torch.arange(batch, device="cuda")[:, None].expand(batch, most)
    taken = j < s["accepted_lens"][:, None]
    to = first[:, None] + torch.where(taken, j, 0)  # past a path's end: the root moves to itself
    at = first[:, None] + torch.where(taken, s["accepted"].long(), s["accepted"][:, :1].long())
    for pool in (s["key_pool"], s["value_pool"]):
        rows = pool[table[:, b, at // page], 0, :, at % page]
        pool[table[:, b, to // page], 0, :, to % page] = rows
    s["new_lens"].copy_(first + s["accepted_lens"])
    return dict(key_pool=s["key_pool"], value_pool=s["value_pool"], lens=s["new_lens"])


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pool in (s["key_pool"], s["value_pool"]):
        rows = pool[src]
        if s["tokens"] is not None:
            taken = torch.arange(pool.shape[3], device="cuda")[None] < s["tokens"][:, None]
            rows = torch.where(taken[:, None, None, :, None], rows, pool[dst])
        pool[dst] = rows
    return dict(key_pool=s["key_pool"], value_pool=s["value_pool"])


def run(s):
    if own:
        if "call" not in s:
            s["call"], s["outputs"] = _own_call(s)
        s["call"]()
        return s["outputs"]
    return {"tree": _tree, "append": _append, "compact": _compact, "copy": _copy}[s["case"]["kind"]](s)


# ---- from the definitions, in 64 bits --------------------------------------

def _exact_tree(c, t):
    hq, hkv, d = SHAPES[c["model"]]
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, parent in enumerate(_trees(c)):
        n, q = int(t["seq_lens"][b]), len(parent)
        ids = torch.from_numpy(t["table"][b, :math.ceil(n / c["page"])]).cuda().long()
        hidden = torch.zeros((q, n), dtype=torch.bool)
        hidden[:, n - q:] = ~torch.from_numpy(_ancestors(parent))
        hidden = hidden.cuda()
        for h in range(hkv):
            heads = slice(h * hq // hkv, (h + 1) * hq // hkv)
            k = t["key_pool"][ids, 0, h].reshape(-1, d)[:n].double()
            v = t["value_pool"][ids, 0, h].reshape(-1, d)[:n].double()
            x = t["q"][heads, at:at + q].double().reshape(-1, d) @ k.t() / math.sqrt(d)
            x = x.view(-1, q, n).masked_fill(hidden, -math.inf)
            out[heads, at:at + q] = (torch.softmax(x, -1).view(-1, n) @ v).view(-1, q, d)
        at += q
    return out


def _exact_append(c, t):
    hq, hkv, d = SHAPES[c["model"]]
    key, val = t["key_pool"].double(), t["value_pool"].double()
    q = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    pos = torch.from_numpy(t["positions"]).cuda().long()
    # One rotation matrix per position applied to each pair.
    turn = torch.complex(t["cos"].double(), t["sin"].double())[pos]

    def rotated(x, w):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        pairs = x.unflatten(-1, (-1, 2)) if c["interleaved"] else x.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)

    q = rotated(t["q"], t["q_weight"])
    k = rotated(t["k"], t["k_weight"])
    at = 0
    for b in range(c["batch"]):
        n, new = int(t["seq_lens"][b]), int(t["q_lens"][b])
        slots = np.arange(n - new, n)
        pages = torch.from_numpy(t["table"][b][slots // c["page"]]).cuda().long()
        inside = torch.from_numpy(slots % c["page"]).cuda()
        key[pages, 0, :, inside] = k[:, at:at + new].transpose(0, 1)
        val[pages, 0, :, inside] = t["v"][:, at:at + new].double().transpose(0, 1)
        at += new
    return dict(q=q, key_pool=key, value_pool=val)


def _exact_compact(c, t):
    pools = dict(key_pool=t["key_pool"].double(), value_pool=t["value_pool"].double())
    lens = []
    page = c["page"]
    moves = []
    for b, parent in enumerate(_trees(c)):
        first = int(t["seq_lens"][b]) - len(parent)
        path = _path(parent)
        lens.append(first + len(path))
        moves += [(b, first + s, first + j) for j, s in enumerate(path) if s != j]
    if moves:
        b, at, to = (np.array(x) for x in zip(*moves))
        for pool in pools.values():
            old = pool.clone()
            for layer in range(c["layers"]):
                table = t["table"][layer]
                src, dst = (torch.from_numpy(x).cuda().long() for x in (table[b, at // page], table[b, to // page]))
                a, z = (torch.from_numpy(x % page).cuda() for x in (at, to))
                pool[dst, 0, :, z] = old[src, 0, :, a]
    return dict(pools, lens=None)


def _exact_copy(c, t):
    pools = dict(key_pool=t["key_pool"].double(), value_pool=t["value_pool"].double())
    tokens = torch.from_numpy(_copied(c)).cuda()
    src, dst = (torch.from_numpy(t[k]).cuda().long() for k in ("src", "dst"))
    for pool in pools.values():
        for slot in range(c["page"]):
            to = tokens > slot
            pool[dst[to], 0, :, slot] = pool[src[to], 0, :, slot]
    return pools


def exact(c, seed):
    t = _inputs(c, seed)
    return {"tree": _exact_tree, "append": _exact_append, "compact": _exact_compact,
            "copy": _exact_copy}[c["kind"]](c, t)
