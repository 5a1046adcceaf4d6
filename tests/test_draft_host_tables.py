"""Host tables shorter than a call's arguments say: the binding's validate_* refuse them, and the library does not read
behind their ends."""
import numpy as np
import pytest

import mvr_attn as M
import mvr_draft as D
from test_draft_api import append_args, compact_args, copy_args, tree_args


def refused(f, *args, **tables):
    with pytest.raises(M.MvrError, match="must hold") as e:
        f(*args, **tables)
    assert e.value.code == M.MVR_E_INVALID_ARGUMENT
    return e.value.message


def shortened(ok, name):
    x = np.asarray(ok[name])
    return {**ok, name: x.reshape(-1)[:-1]}


def test_tree():
    a, t = tree_args(total_q=60)
    ok = dict(block_tables_host=np.arange(128).reshape(2, 64), seq_lens_host=np.array([100, 1024]),
              cu_q_lens_host=np.array([0, 0, 40]), masks_host=np.full((40, 2), -1, np.int32))
    D.validate_tree(a, t, **ok)  # (masks: rows of the requests' tokens; those of a padded batch are not read)
    for name in ok:
        assert name in refused(D.validate_tree, a, t, **shortened(ok, name))
    a, t = tree_args(num_seqs=1, cu_q_lens=None)  # one request of max_q_len drafts
    D.validate_tree(a, t, masks_host=np.full((40, 2), -1, np.int32))
    refused(D.validate_tree, a, t, masks_host=np.full((39, 2), -1, np.int32))


def test_append():
    a, n = append_args()
    ok = dict(block_tables_host=np.arange(16).reshape(2, 8), seq_lens_host=np.array([7, 40]),
              cu_q_lens_host=np.array([0, 0, 9]), positions_host=np.arange(9), page_writable_host=np.ones(64))
    D.validate_norm_rope_append(a, n, **ok)
    for name in ok:
        assert name in refused(D.validate_norm_rope_append, a, n, **shortened(ok, name))
    a, n = append_args(num_seqs=1, cu_q_lens=None, total_q=10)
    refused(D.validate_norm_rope_append, a, n, positions_host=np.arange(9))


def test_compact():
    a = compact_args()
    ok = dict(block_tables_host=np.arange(32).reshape(2, 2, 8), seq_lens_host=np.array([12, 9]),
              cu_q_lens_host=np.array([0, 5, 9]), accepted_host=np.array([[0, 2, 4, 9], [1, 3, -1, -1]]),
              accepted_lens_host=np.array([3, 2]))
    D.validate_compact_drafts(a, **ok)
    for name in ok:
        assert name in refused(D.validate_compact_drafts, a, **shortened(ok, name))


def test_copy():
    a = copy_args()
    ok = dict(src_pages_host=np.array([1, 1, 2]), dst_pages_host=np.array([3, 4, 5]), tokens_host=np.array([0, 4, 2]))
    D.validate_copy_pages(a, **ok)
    for name in ok:
        assert name in refused(D.validate_copy_pages, a, **shortened(ok, name))


def test_arguments_that_the_library_refuses_are_its_to_name():
    """Sizes out of range are reported as such, whatever the tables hold."""
    a, t = tree_args(num_seqs=0)
    with pytest.raises(M.MvrError, match="at least one request"):
        D.validate_tree(a, t, seq_lens_host=np.array([1]))
    with pytest.raises(M.MvrError, match="num_copies"):
        D.validate_copy_pages(copy_args(num_copies=-1), np.array([1]))
