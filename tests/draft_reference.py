"""Plain 64-bit forms of the drafted-tree calls, and the batches that their tests run."""
import math

import numpy as np
import torch

EPS = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def random_tables(rng, need, num_pages, width=None, pad=0):
    """Block tables with every request's pages distinct; unused entries hold `pad`."""
    order = rng.permutation(num_pages)
    table = np.full((len(need), width or max(max(need), 1)), pad, np.int32)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = order[used:used + n]
        used += n
    return table


class Batch:
    """Requests of `cached` tokens and `q` drafts each, random values and masks, on the CPU; .cuda() copies."""

    def __init__(self, seed, dtype, hq, hkv, d, page, cached, q, masks="random", spare=3, q_std=1.5, tail=0, words=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.page, self.tail = dtype, hq, hkv, d, page, tail
        self.q_lens, self.cached = np.array(q, np.int32), np.array(cached, np.int32)
        self.seq_lens = (self.cached + self.q_lens).astype(np.int32)
        self.cu = np.concatenate([[0], np.cumsum(self.q_lens)]).astype(np.int32)
        need = [math.ceil(n / page) for n in self.seq_lens]
        self.num_pages = max(sum(need), 1) + spare
        self.table = random_tables(rng, need, self.num_pages)
        tokens = int(self.cu[-1]) + tail
        self.max_q, self.max_len = max(int(self.q_lens.max()), 1), max(int(self.seq_lens.max()), 1)
        normal = lambda shape, std=1.0: (torch.randn(shape, generator=gen) * std).to(dtype)  # noqa: E731
        self.queries = normal((hq, max(tokens, 1), d), q_std)
        self.key_pool = normal((self.num_pages, 1, hkv, page, d))
        self.value_pool = normal((self.num_pages, 1, hkv, page, d))
        self.words = max(words, math.ceil(self.max_q / 32))
        bits = rng.random((max(tokens, 1), self.words * 32)) < 0.5
        if masks == "tree":
            bits[:] = False
            for b, n in enumerate(self.q_lens):
                seen = np.zeros((n, n), bool)
                for i in range(n):
                    if i:
                        seen[i] = seen[rng.integers(max(0, i - 5), i)]
                    seen[i, i] = True
                bits[self.cu[b]:self.cu[b + 1], :n] = seen
        elif masks == "chain":
            bits[:] = False
            for b, n in enumerate(self.q_lens):
                bits[self.cu[b]:self.cu[b + 1], :n] = np.tril(np.ones((n, n), bool))
        elif masks == "none":
            bits[:] = False
        self.bits = bits  # (random: bits from q_len on are set too, and count for nothing)

    @property
    def masks(self):
        return np.packbits(self.bits, axis=1, bitorder="little").view(np.int32)

    def keys(self, b):
        """K, V of request b in 64 bits: [Hkv, n, D]."""
        n = int(self.seq_lens[b])
        ids = torch.from_numpy(self.table[b, :math.ceil(n / self.page)]).long()
        return [p[ids, 0].double().permute(1, 0, 2, 3).reshape(self.hkv, -1, self.d)[:, :n] for p in
                (self.key_pool, self.value_pool)]

    def visible(self, b):
        """[q, n] truth values."""
        q, n = int(self.q_lens[b]), int(self.seq_lens[b])
        seen = torch.ones((q, n), dtype=torch.bool)
        seen[:, n - q:] = torch.from_numpy(self.bits[self.cu[b]:self.cu[b + 1], :q])
        return seen

    def attention(self, scale=None):
        """(output, tolerance) in 64 bits: [Hq, tokens, D]; rows of no request are NaN in the output.

        The tolerance is the sum of what the kernel rounds: the output (half a step of it), each probability to the
        activation dtype (half a step of sum p |v| at most; nothing in F32), each score's D products and sums in 32
        bits and its exponential (the relative error of a probability, twice: above and below the fraction), and the
        sums of n terms in 32 bits, twice."""
        scale = scale or 1.0 / math.sqrt(self.d)
        out = torch.full(self.queries.shape, math.nan, dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.hq // self.hkv
        for b in range(len(self.q_lens)):
            lo, hi, n = int(self.cu[b]), int(self.cu[b + 1]), int(self.seq_lens[b])
            if lo == hi:
                continue
            k, v = self.keys(b)
            seen = self.visible(b)
            for h in range(self.hkv):
                x = self.queries[h * group:(h + 1) * group, lo:hi].double()  # [G, q, D]
                s = (x @ k[h].T * scale).masked_fill(~seen, -math.inf)
                size = (x.abs() @ k[h].abs().T * scale).masked_fill(~seen, 0.0).nan_to_num(0.0, 0.0, 0.0).amax(-1)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                o = torch.where(p[..., None] == 0, 0.0, p[..., None] * v[h]).sum(-2)  # a masked key adds nothing
                mean = (p @ v[h].nan_to_num(0.0, 0.0, 0.0).abs())
                u = EPS[self.dtype]
                delta = 2.0 ** -24 * (self.d + 8) * size[..., None] + 2.0 ** -20
                rows = slice(h * group, (h + 1) * group)
                out[rows, lo:hi] = o
                tol[rows, lo:hi] = u * o.abs() + mean * ((u if self.dtype == torch.float16 else 0.0) + 2 * delta +
                                                         2 * n * 2.0 ** -24) + 2.0 ** -24 * (self.dtype == torch.float16)
        return out, tol

    def device(self, **changed):
        """The call's tensors on the GPU."""
        t = dict(q=self.queries, key_pool=self.key_pool, value_pool=self.value_pool,
                 block_tables=torch.from_numpy(self.table), seq_lens=torch.from_numpy(self.seq_lens),
                 cu_q_lens=torch.from_numpy(self.cu), masks=torch.from_numpy(self.masks))
        t.update(changed)
        return {k: v.cuda() for k, v in t.items()}


def check_attention(got, batch, scale=None, note=""):
    """Every row of a request within its tolerance, non-finite ones equal; rows of no request are not looked at."""
    want, tol = batch.attention(scale)
    rows = int(batch.cu[-1])
    got, want, tol = got.double().cpu()[:, :rows], want[:, :rows], tol[:, :rows]
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{note}: finite where the reference is not, or the reverse"
    same = torch.isnan(want) == torch.isnan(got)
    assert bool(same.all()) and torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), note
    off = (got - want).abs()[finite] / tol[finite].clamp(min=1e-300)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{note}: {worst:.3g} times the tolerance"
    return worst
