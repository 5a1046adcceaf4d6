"""mvr_paged_attention_tree in F16: what the probabilities lose on their way into the product with V.  The keys have a
score of 0 or one whose probability lies half an F16 step from the next F16 number, so the rounding of each goes the same
way.
  * Values that are all equal come back as they are, in every row tile: the weights of the keys add up to 1.
  * Values that all but cancel, in the row tiles of 16 and 32, whose products take the probabilities with 20 bits: an error
    of theirs is not hidden by the rounding of the output.
Keys whole and in parts, in child processes (a process reads the planner's overrides once)."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mvr_draft as D  # noqa: E402

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIM, QUERY = 64, 8.0  # q = 8 e_0, k = 0 or x e_0: the scores are 0 and 8 x / sqrt(64) = x, both exact


def far_from_f16():
    """The F16 number x in (-0.69, -0.6) whose e^x, in [0.5, 0.55], F16 rounds worst."""
    x = -np.arange(0.6, 0.69, 2.0 ** -11).astype(np.float16)
    p = np.exp(x.astype(np.float64))
    off = np.abs(p.astype(np.float16).astype(np.float64) - p) / p
    assert off.max() > 0.9 * 2.0 ** -11
    return float(x[off.argmax()])


def attention(page, cached, nodes, low, values):
    """Outputs [rows, DIM] in 64 bits of one request whose key t has the low score where low(t), and value values[low(t)]."""
    hq, hkv, n = 8, 2, cached + nodes
    x = far_from_f16()
    pages = math.ceil(n / page)
    order = np.random.default_rng(n).permutation(pages + 2)[:pages]
    key, val = (torch.zeros((pages + 2, 1, hkv, page, DIM), dtype=torch.float16) for _ in range(2))
    for t in range(n):
        key[int(order[t // page]), 0, :, t % page, 0] = x if low(t) else 0.0
        val[int(order[t // page]), 0, :, t % page] = values[low(t)]
    q = torch.zeros((hq, nodes, DIM), dtype=torch.float16)
    q[:, :, 0] = QUERY
    return D.paged_attention_tree(
        q.cuda(), key.cuda(), val.cuda(), torch.from_numpy(order.astype(np.int32)[None]).cuda(),
        torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, nodes], dtype=torch.int32).cuda(),
        torch.full((nodes, math.ceil(nodes / 32)), -1, dtype=torch.int32).cuda(), max_q_len=nodes,
        max_seq_len=n).double().cpu()


def check_equal_values(page, cached, nodes):
    """One key in 16 with a score of 0.  Sums of n terms in 32 bits, above and below the fraction, are off by 2 n 2^-24 at
    most, less than the half step that would change the output: 2^-11 on values just below 2."""
    value, n = 2.0 - 2.0 ** -10, cached + nodes
    assert value * 2 * n * 2.0 ** -24 < 2.0 ** -12
    got = attention(page, cached, nodes, lambda t: t % 16 != 3, (value, value))
    print(f"equal values, page {page}, {cached} + {nodes}: {got.min()} to {got.max()}", flush=True)
    assert bool((got == value).all())


def check_cancelling_values(page, cached, nodes):
    n, p = cached + nodes, math.exp(far_from_f16())
    value = float(np.float16(1 / p))
    got = attention(page, cached, nodes, lambda t: t % 2 == 1, (-1.0, value))
    odd = n // 2
    even = n - odd
    total = even + odd * p
    want = (odd * p * value - even) / total
    size = (odd * p * value + even) / total  # sum p |v|
    # The output's half step; a probability's 2^-20 (its two F16 parts), 2^-22 for its exponential and argument in 32
    # bits (|x| < 1); sums of n terms in 32 bits above and below the fraction.
    tol = 2.0 ** -11 * abs(want) + 2.0 ** -24 + size * (2.0 ** -20 + 2 * 2.0 ** -22 + 2 * n * 2.0 ** -24)
    worst = float((got - want).abs().max())
    print(f"cancelling values, page {page}, {cached} + {nodes}: off by {worst:.3g}, tolerance {tol:.3g}", flush=True)
    # (Probabilities of one F16 number each: off by this much.)
    assert tol < 0.3 * odd * value * abs(float(np.float16(p)) - p) / total
    assert worst <= tol


@pytest.mark.parametrize("units", ["1", str(1 << 20)])  # of 64 keys in a part
@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_probabilities_reach_the_product_with_their_bits(rows, units):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    env = dict(os.environ, MVR_DRAFT_TILE_ROWS=str(rows), MVR_DRAFT_PART_UNITS=units, PYTHONPATH=os.pathsep.join(
        [os.path.join(ROOT, "mini-vllm-rs_amd"), os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], env=env, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=110)
    print(r.stdout[-3000:], flush=True)
    assert r.returncode == 0, r.stdout[-3000:]
    assert "ran every case" in r.stdout


if __name__ == "__main__":
    for args in ((16, 40, 1), (16, 200, 8), (24, 97, 20), (5, 60, 33), (16, 300, 70)):
        check_equal_values(*args)
        if int(os.environ["MVR_DRAFT_TILE_ROWS"]) <= 32:
            check_cancelling_values(*args)
    print("ran every case", flush=True)
