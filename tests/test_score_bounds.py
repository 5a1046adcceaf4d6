"""Sizes at which the calls on scores are accepted or refused, on the CPU: nothing is launched."""
import ctypes

import numpy as np
import pytest

import mvr_attn as M
import mvr_score as S
from test_score_api import move_args, scored_args, select_args, weights_args


def refused(validate, *args, text, code=M.MVR_E_UNSUPPORTED):
    with pytest.raises(M.MvrError) as e:
        validate(*args)
    assert e.value.code == code and text in e.value.message, e.value.message


def test_longest_request_of_a_selection():
    """A block steps over 4,096 slots at a time, and counts them in 32 bits."""
    sizes = dict(page_size=4096, max_pages_per_seq=1 << 19)
    arrays = ("weights", "positions", "block_tables", "seq_lens", "next_positions", "kept_lens", "keep_lens", "moves",
              "num_moves", "new_seq_lens")
    sizes.update((name, (i + 1) << 28) for i, name in enumerate(arrays))  # (where they do not overlap)
    S.validate_select(select_args(**sizes, max_seq_len=2 ** 31 - 1 - 4096))
    for n in (2 ** 31 - 4096, 2 ** 31 - 2049, 2 ** 31 - 1):
        refused(S.validate_select, select_args(**sizes, max_seq_len=n), text="too close to 2^31")


def test_most_moves_of_a_row():
    """A row's blocks step over up to 2^23 moves at a time, and count them in 32 bits."""
    S.validate_move(move_args(max_moves=2 ** 31 - 1 - 2 ** 23))
    for n in (2 ** 31 - 2 ** 23, 2 ** 31 - 1):
        refused(S.validate_move, move_args(max_moves=n), text="too close to 2^31")


def workspace(q, keys, total=True, **kw):
    """Bytes that a call asks for whose requests have these new tokens and keys, its host tables given."""
    seq, cu = np.array(keys, np.int32), np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    sizes = dict(num_seqs=len(q), max_q_len=int(max(q)), max_seq_len=int(max(keys)), max_pages_per_seq=1 << 14,
                 total_q=int(cu[-1]) if total else 0, lse_stride_head=int(cu[-1]), q_stride_head=1 << 28,
                 seq_lens_host=seq.ctypes.data, cu_q_lens_host=cu.ctypes.data, num_q_heads=28, num_kv_heads=4)
    refs = [ctypes.byref(x) for x in scored_args(**{**sizes, **kw})]
    return S.load_library().mvr_paged_attention_scored_workspace_size(*refs)


def test_a_split_never_asks_for_more_than_its_budget():
    """Partial results hold a slot for every part of every place, also where few row tiles have so many parts."""
    budget = 96 << 20
    for dtype in (M.DTYPE_F16, M.DTYPE_F32):
        for total in (True, False):
            prompt = [2509] + [1] * 190
            assert workspace(prompt, [2518] * 191, total, dtype=dtype) <= budget
            for q, keys in (([2131, 1], [34602] * 2), ([1024, 1024], [34602] * 2), ([1] * 63 + [2000], [2000] * 64)):
                assert workspace(q, keys, total, dtype=dtype) <= budget, (q, total)
            rng = np.random.default_rng(5)
            for _ in range(300):
                q = rng.integers(0, int(2 ** rng.uniform(1, 12)), rng.integers(1, 200)) + (rng.random() < 0.5)
                keys = q + rng.integers(0, int(2 ** rng.uniform(1, 16)), len(q))
                q[0] += not q.any()
                heads = rng.choice([1, 2, 8])
                assert workspace(q, np.maximum(keys, q), total, dtype=dtype, num_kv_heads=heads, num_q_heads=heads * rng.integers(1, 9),
                                 head_dim=int(rng.choice([32, 64, 128, 256]))) <= budget
    assert workspace([1] * 4, [30000] * 4) > 0  # (and calls are split)


def mixed(num_seqs, longest, **kw):
    """One prompt among single tokens."""
    return dict(num_seqs=num_seqs, max_q_len=longest, max_seq_len=max(longest, 64), max_pages_per_seq=1 << 12,
                total_q=num_seqs - 1 + longest, lse_stride_head=1 << 24, q_stride_head=1 << 28, **kw)


@pytest.mark.parametrize("num_seqs,longest", [(256, 8192), (512, 4096), (1024, 2048), (4000, 32768), (65536, 4)])
def test_mixed_batches_count_the_tokens_that_are_there(num_seqs, longest):
    """Accepted as mvr_paged_attention accepts them, whatever the longest request would take in every place."""
    S.validate_scored(*scored_args(**mixed(num_seqs, longest)))
    S.validate_weights(*weights_args(**mixed(num_seqs, longest)))


def test_most_row_tiles_of_a_call():
    """2^24 blocks of 256 threads: by max_q_len where the tokens are not known."""
    sizes = dict(num_q_heads=16, num_kv_heads=1)  # a tile per token
    for total in (0, 1 << 24):
        S.validate_scored(*scored_args(**{**mixed(2040, 8192, **sizes), "total_q": 0}))
        refused(S.validate_scored, *scored_args(**{**mixed(2049, 8192, **sizes), "total_q": total}), text="more than one call takes")
    S.validate_scored(*scored_args(**{**mixed(2049, 8192, **sizes), "total_q": 1 << 23}))
    weights = weights_args(**{**mixed(2049, 8192, **sizes), "total_q": 0})
    S.validate_weights(*weights)  # whose blocks are those of the keys
