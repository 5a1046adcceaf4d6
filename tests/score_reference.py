"""Plain 64-bit forms of the calls on scores, and the batches that their tests run."""
import math

import numpy as np
import torch

from draft_reference import EPS, random_tables


class Batch:
    """Requests of `cached` tokens and `q` new ones each, random values on the CPU, and the rules of their scores.

    first_keys: a number per packed token, prefix: one per request, or None.  tail: rows behind the last request."""

    def __init__(self, seed, dtype, hq, hkv, d, page, cached, q, cap=0.0, slopes=False, window=0, first_keys=None,
                 prefix=None, spare=3, q_std=1.5, tail=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.page, self.tail = dtype, hq, hkv, d, page, tail
        self.q_lens, self.cached = np.array(q, np.int32), np.array(cached, np.int32)
        self.seq_lens = (self.cached + self.q_lens).astype(np.int32)
        self.cu = np.concatenate([[0], np.cumsum(self.q_lens)]).astype(np.int32)
        need = [math.ceil(n / page) for n in self.seq_lens]
        self.num_pages = max(sum(need), 1) + spare
        self.table = random_tables(rng, need, self.num_pages)
        self.tokens = int(self.cu[-1]) + tail
        self.max_q, self.max_len = max(int(self.q_lens.max()), 1), max(int(self.seq_lens.max()), 1)
        normal = lambda shape, std=1.0: (torch.randn(shape, generator=gen) * std).to(dtype)  # noqa: E731
        self.queries = normal((hq, max(self.tokens, 1), d), q_std)
        self.key_pool = normal((self.num_pages, 1, hkv, page, d))
        self.value_pool = normal((self.num_pages, 1, hkv, page, d))
        self.weights = torch.rand((self.num_pages, hkv, page), generator=gen)
        self.cap, self.window = cap, window
        self.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]) if slopes is True else slopes or None
        self.first_keys = None if first_keys is None else np.resize(np.array(first_keys, np.int32), max(self.tokens, 1))
        self.prefix = None if prefix is None else np.resize(np.array(prefix, np.int32), len(self.q_lens))

    def ids(self, b):
        return torch.from_numpy(self.table[b, :math.ceil(self.seq_lens[b] / self.page)]).long()

    def keys(self, b, pool):
        """Rows of request b in 64 bits: [Hkv, n, D]."""
        x = pool[self.ids(b), 0].double()
        return x.permute(1, 0, 2, 3).reshape(self.hkv, -1, self.d)[:, :int(self.seq_lens[b])]

    def visible(self, b):
        """[q, n] truth values."""
        q, n = int(self.q_lens[b]), int(self.seq_lens[b])
        pos, key = torch.arange(n - q, n)[:, None], torch.arange(n)
        last = pos + 1
        if self.prefix is not None:
            last = last.clamp(min=min(int(self.prefix[b]), n))
        seen = key < last
        if self.window:
            seen &= key > pos - self.window
        if self.first_keys is not None:
            seen &= key >= torch.from_numpy(self.first_keys[self.cu[b]:self.cu[b + 1]]).long()[:, None]
        return seen

    def scores(self, b, h, scale):
        """Scores [G, q, n] of KV head h (-inf where not seen) and how far 32-bit ones may be off (0 there).

        A score is off by its D products and sums in 32 bits, the scale's rounding among them (2^-24 each of the sum of
        |q k|); what the cap makes of it: 2^-21 of the capped score by the polynomial, six roundings of a half step, and
        where a score near it leaves the polynomial's range (0.625 of the cap, 0.09 of caps past 1e4) 2^-21 of the cap by
        1 - 2 / (e^2y + 1), a reciprocal of 2 at most off by 2^-22 and an exponential off by as much at a slope of 1/2;
        the slope, its factor log2(e) and the distance's product (2^-22 of it).  Differences to the row's maximum and the
        exponential: 2^-20 + 2^-23 of the score."""
        group = self.hq // self.hkv
        heads = slice(h * group, (h + 1) * group)
        q, n = int(self.q_lens[b]), int(self.seq_lens[b])
        x = self.queries[heads, self.cu[b]:self.cu[b + 1]].double()
        k = self.keys(b, self.key_pool)[h]
        s, size = x @ k.T * scale, (x.abs() @ k.abs().T * scale).nan_to_num(0.0, 0.0, 0.0)
        off = 2.0 ** -24 * (self.d + 8) * size
        if self.cap:
            far = bool((s.abs() > 0.08 * self.cap).any())
            s = self.cap * torch.tanh(s / self.cap)
            off = off + (2.0 ** -21 * self.cap if far else 0.0)
        off = off + 2.0 ** -21 * s.abs().nan_to_num(0.0, 0.0, 0.0)
        if self.slopes is not None:
            away = (torch.arange(n - q, n)[:, None] - torch.arange(n)).abs().double()
            bias = self.slopes[heads].double()[:, None, None] * away
            s, off = s - bias, off + 2.0 ** -22 * bias.abs()
        off = off + 2.0 ** -20 + 2.0 ** -23 * s.abs().nan_to_num(0.0, 0.0, 0.0)
        seen = self.visible(b)
        return s.masked_fill(~seen, -math.inf), off.masked_fill(~seen, 0.0)

    def attention(self, scale=None):
        """(output, its tolerance, lse, its tolerance) in 64 bits; rows of no request are NaN in the values.

        Half a step of the output; each probability's relative error `off` above and below the fraction; half a step of
        each F16 probability (of the sum p |v|); the sums of n terms in 32 bits, twice."""
        scale = scale or 1.0 / math.sqrt(self.d)
        out = torch.full(self.queries.shape, math.nan, dtype=torch.float64)
        lse = torch.full(self.queries.shape[:2], math.nan, dtype=torch.float64)
        tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
        group, u = self.hq // self.hkv, EPS[self.dtype]
        for b in range(len(self.q_lens)):
            lo, hi, n = int(self.cu[b]), int(self.cu[b + 1]), int(self.seq_lens[b])
            if lo == hi:
                continue
            v = self.keys(b, self.value_pool)
            for h in range(self.hkv):
                rows = slice(h * group, (h + 1) * group)
                s, off = self.scores(b, h, scale)
                row_lse = torch.logsumexp(s, -1)
                p = torch.exp(s - torch.where(row_lse == -math.inf, 0.0, row_lse)[..., None])
                p = torch.where(torch.isnan(s), math.nan, p)
                finite = v[h].nan_to_num(0.0, 0.0, 0.0)
                o = p @ finite
                for j in torch.nonzero(~torch.isfinite(v[h]).all(-1)).flatten().tolist():  # a masked key adds nothing
                    x = torch.where(torch.isfinite(v[h, j]), 0.0, v[h, j])
                    o += torch.where(p[..., j, None] == 0, 0.0, p[..., j, None] * x)
                off = p.nan_to_num(0.0) * off
                mean, doubt = p.nan_to_num(0.0) @ finite.abs(), off.sum(-1)
                out[rows, lo:hi] = o
                half = self.dtype == torch.float16
                tol[rows, lo:hi] = u * o.abs() + off @ finite.abs() + doubt[..., None] * o.abs() + mean * (
                    (u if half else 0.0) + 2 * n * 2.0 ** -24) + 2.0 ** -24 * half
                lse[rows, lo:hi] = row_lse
                lse_tol[rows, lo:hi] = doubt + n * 2.0 ** -24 + 2.0 ** -22 * row_lse.abs().nan_to_num(0.0, 0.0, 0.0) + 2.0 ** -21
        return out, tol, lse, lse_tol

    def key_weights(self, lse, decay=1.0, fresh=None, scale=None):
        """(weights pool, its tolerance) in 64 bits, from log-sum-exps in 32 bits [Hq, tokens].

        Each e^(score - lse) is off by the score's error and the lse's conversion to another base; the sum over rows by a
        rounding per row, the product and sum with what the key had by one each."""
        scale = scale or 1.0 / math.sqrt(self.d)
        pool, tol = self.weights.double(), torch.zeros_like(self.weights, dtype=torch.float64)
        group = self.hq // self.hkv
        for b in range(len(self.q_lens)):
            lo, hi, n = int(self.cu[b]), int(self.cu[b + 1]), int(self.seq_lens[b])
            if lo == hi:
                continue
            old = n - (hi - lo) if fresh is None else int(fresh[b])
            for h in range(self.hkv):
                s, off = self.scores(b, h, scale)
                row = lse[h * group:(h + 1) * group, lo:hi].double()[..., None]
                p = torch.where(row == -math.inf, 0.0, torch.exp(s - row))
                got, doubt = p.sum((0, 1)), (p * (off + 2.0 ** -22 * row.abs().nan_to_num(0.0, 0.0, 0.0) + 2.0 ** -20)).sum((0, 1))
                flat = pool[self.ids(b), h].reshape(-1)
                had = torch.where(torch.arange(n) < old, flat[:n] * decay if decay else torch.zeros(n).double(), 0.0)
                flat[:n] = had + got
                pool[self.ids(b), h] = flat.view(-1, self.page)
                off_pool = tol[self.ids(b), h].reshape(-1)
                off_pool[:n] = doubt + p.shape[0] * p.shape[1] * 2.0 ** -24 * got + 2.0 ** -22 * (had.abs() + got)
                tol[self.ids(b), h] = off_pool.view(-1, self.page)
        return pool, tol

    def device(self, **changed):
        """The attention call's positional tensors on the GPU."""
        t = dict(q=self.queries, key_pool=self.key_pool, value_pool=self.value_pool,
                 block_tables=torch.from_numpy(self.table), seq_lens=torch.from_numpy(self.seq_lens),
                 cu_q_lens=torch.from_numpy(self.cu))
        t.update(changed)
        return {k: v.cuda() for k, v in t.items()}

    def rules(self):
        """The rules' keyword arguments, on the GPU."""
        table = lambda x: None if x is None else torch.as_tensor(x).cuda()  # noqa: E731
        return dict(cap=self.cap, window=self.window, slopes=table(self.slopes), first_keys=table(self.first_keys),
                    prefix_lens=table(self.prefix), max_q_len=self.max_q, max_seq_len=self.max_len)


def within(got, want, tol, note=""):
    """Every value within its tolerance, infinities and NaN equal."""
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{note}: finite where the reference is not, or the reverse"
    odd = ~finite
    assert torch.equal(torch.isnan(want), torch.isnan(got)), f"{note}: NaN"
    odd &= ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), f"{note}: infinities"
    off = (got - want).abs()[finite] / tol[finite].clamp(min=1e-300)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{note}: {worst:.3g} times the tolerance"
    return worst


def check_attention(out, lse, batch, scale=None, note=""):
    """Every row of a request within its tolerance; rows of no request are not looked at."""
    want, tol, want_lse, lse_tol = batch.attention(scale)
    rows = int(batch.cu[-1])
    worst = within(out[:, :rows], want[:, :rows], tol[:, :rows], note + " out")
    if lse is not None:
        worst = max(worst, within(lse[:, :rows], want_lse[:, :rows], lse_tol[:, :rows], note + " lse"))
    return worst


def select(weights, positions, table, seq_lens, next_positions, kept_lens, keep_lens, recent, first, max_moves):
    """(moves as a list per [layer][request][head], new lengths, positions): numpy, token by token."""
    layers, batch, _ = table.shape
    pages, hkv, page = weights.shape
    positions, new_lens = positions.copy(), np.zeros(batch, np.int32)
    moves = [[[[] for _ in range(hkv)] for _ in range(batch)] for _ in range(layers)]
    for b in range(batch):
        n = int(seq_lens[b])
        keep = max(0, min(int(keep_lens[b]), n))
        if min(keep, n - keep) > max_moves:
            keep = n
        new_lens[b] = keep
        slots = np.arange(n)
        for layer in range(layers):
            ids = table[layer, b, slots // page]
            inside = (ids >= 0) & (ids < pages)
            safe = np.where(inside, ids, 0)
            for h in range(hkv):
                pos = np.where(slots >= kept_lens[b], next_positions[b] - (n - slots), positions[safe, h, slots % page])
                fresh = inside & (slots >= kept_lens[b])
                positions[ids[fresh], h, slots[fresh] % page] = pos[fresh]
                if keep in (0, n):
                    continue
                w = weights[safe, h, slots % page].astype(np.float64)
                w = np.where(np.isnan(w), -np.inf, w)
                guarded = (pos < first) | (pos >= next_positions[b] - recent)
                w = np.where(inside, w, -np.inf)
                order = sorted(range(n), key=lambda t: (0, 0, t) if guarded[t] and inside[t] else (1, -w[t], t))
                stay = np.zeros(n, bool)
                stay[order[:keep]] = True
                moves[layer][b][h] = list(zip(slots[stay & (slots >= keep)].tolist(), slots[~stay & (slots < keep)].tolist()))
    return moves, new_lens, positions
