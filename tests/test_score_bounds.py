"""Sizes at which the calls on scores are accepted or refused, on the CPU: nothing is launched."""
import pytest

import mvr_attn as M
import mvr_score as S
from test_score_api import move_args, select_args


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
