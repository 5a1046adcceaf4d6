"""A step in which no request has a token: the drafted-tree binding's calls on tensors of no rows do nothing, as on a padded
batch of empty requests.  (The entry points of the library see no such call: its tensors have no address.)"""
import contextlib

import pytest

torch = pytest.importorskip("torch")

import mvr_attn as M  # noqa: E402
import mvr_draft as D  # noqa: E402


@pytest.fixture()
def no_gpu(monkeypatch):
    """CPU tensors pass for a GPU's, and nothing may be launched on them."""
    monkeypatch.setattr(D, "_same_device", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(M, "_stream_handle", lambda stream: 0)
    monkeypatch.setattr(D, "_scope", lambda device, stream: contextlib.nullcontext())


def tensors(hq=4, hkv=2, d=64):
    pool = torch.zeros((4, 1, hkv, 16, d), dtype=torch.float16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(q=pool.new_zeros((hq, 0, d)), key_pool=pool, value_pool=pool.clone(), block_tables=i32(3, 2), seq_lens=i32(3),
                cu_q_lens=i32(4))


def test_attention_of_no_rows(no_gpu):
    t = tensors()
    masks = torch.zeros((0, 1), dtype=torch.int32)
    out = D.paged_attention_tree(**t, masks=masks, max_q_len=8, max_seq_len=20)
    assert out.shape == t["q"].shape and out.dtype == t["q"].dtype
    call = D.make_tree_call(**t, masks=masks, out=out, max_q_len=8, max_seq_len=20)
    call()
    call()
    with pytest.raises(M.MvrError, match="masks"):  # the tensors are checked all the same
        D.paged_attention_tree(**t, masks=torch.zeros((2, 1), dtype=torch.int32), max_q_len=8, max_seq_len=20)


def test_append_of_no_rows(no_gpu):
    t = tensors()
    kv = t["key_pool"].new_zeros((2, 0, 64))
    cos = t["key_pool"].new_zeros((32, 32))
    t["key_pool"] += 3
    got = D.norm_rope_append(**t, k=kv, v=kv, q_weight=None, k_weight=None, cos_table=cos, sin_table=cos, eps=1e-6,
                             max_seq_len=20, positions=torch.zeros(0, dtype=torch.int32))
    assert got.shape == t["q"].shape and bool((t["key_pool"] == 3).all())
    with pytest.raises(M.MvrError, match="head_dim"):
        D.norm_rope_append(**t, k=kv[..., :32], v=kv[..., :32], q_weight=None, k_weight=None, cos_table=cos, sin_table=cos,
                           eps=1e-6, max_seq_len=20)
