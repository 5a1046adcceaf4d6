"""Block tables that do not cover max_seq_len are refused, where max_seq_len plus a page passes 2^31 too."""
import ctypes

import pytest

import mvr_attn as M
import mvr_draft as D
from test_draft_api import tree_args


@pytest.mark.parametrize("page,pages", [(4096, 1), (1 << 20, 2047), (2048, (1 << 20) - 2)])
def test_tables_that_are_too_short_for_the_longest_lengths(page, pages):
    lib = D.load_library()
    a, t = tree_args(max_seq_len=2 ** 31 - 1025, page_size=page, max_pages_per_seq=pages, max_q_len=1)
    need = -(-(2 ** 31 - 1025) // page)
    assert pages < need
    assert lib.mvr_paged_attention_tree_validate(ctypes.byref(a), ctypes.byref(t), *[None] * 4) == M.MVR_E_PAGES_UNCOVERED
    assert lib.mvr_paged_attention_validate(ctypes.byref(a), *[None] * 3) == M.MVR_E_PAGES_UNCOVERED
    a.max_pages_per_seq = need
    assert lib.mvr_paged_attention_tree_validate(ctypes.byref(a), ctypes.byref(t), *[None] * 4) == M.MVR_OK
    assert lib.mvr_paged_attention_validate(ctypes.byref(a), *[None] * 3) == M.MVR_OK
