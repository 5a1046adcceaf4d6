"""What a call object of the drafted-tree binding tells the allocator of the workspace that it made itself: every stream
that it launches on other than the one that the memory came from, so that the memory is not handed out again while kernels
there still use it.  Stub tensors and streams; the launches are copies of no pages, which launch nothing."""
from types import SimpleNamespace

import pytest

import mvr_attn as M
import mvr_draft as D
from test_draft_api import copy_args

HOME, SIDE, OTHER = 0, 0x1000, 0x2000


class Memory:
    """A tensor as far as the allocator is concerned."""

    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream.cuda_stream)


@pytest.fixture()
def current(monkeypatch):
    """The current stream's handle, in a list: tests set current[0]."""
    handle = [HOME]
    cuda = SimpleNamespace(current_device=lambda: 0, current_stream=lambda index: SimpleNamespace(cuda_stream=handle[0]))
    monkeypatch.setattr(M, "_torch", lambda: SimpleNamespace(cuda=cuda))
    monkeypatch.setattr(D, "_raw_current_stream", lambda index: handle[0])
    return handle


def call(stream=None, **kw):
    device = SimpleNamespace(index=0)
    if stream is not None:
        stream = SimpleNamespace(cuda_stream=stream, device=device)
    args = copy_args(num_copies=0, src_pages=None, dst_pages=None)
    tensor = Memory()
    return D.Call("mvr_copy_pages", args, None, (tensor,), device, stream, **kw), tensor


def test_own_workspace_is_kept_for_every_stream_that_it_is_launched_on(current):
    ws = Memory()
    c, tensor = call(workspace=ws, workspace_stream=HOME)
    c()
    assert ws.streams == []
    for current[0] in (SIDE, SIDE, OTHER, HOME, SIDE):
        c()
    assert ws.streams == [SIDE, OTHER]  # (once is enough until the memory is freed)
    assert tensor.streams == []  # the caller's tensors on the current stream: the caller's matter, as for any operation


def test_own_workspace_of_a_call_with_a_stream_of_its_own(current):
    ws = Memory()
    c, tensor = call(SIDE, workspace=ws, workspace_stream=SIDE)
    c()
    assert ws.streams == [] and tensor.streams == [SIDE]
    current[0] = SIDE
    c()
    assert ws.streams == [] and tensor.streams == [SIDE]


def test_workspace_of_the_caller(current):
    ws = Memory()
    c, _ = call(SIDE, workspace=ws)
    c()
    assert ws.streams == [SIDE]
    ws = Memory()
    c, _ = call(workspace=ws)
    current[0] = SIDE
    c()
    assert ws.streams == []


def test_the_tree_call_names_the_stream_of_its_allocation(current, monkeypatch):
    """make_tree_call itself, its tensors and library stubbed."""
    import contextlib
    made = {}
    device = SimpleNamespace(index=0)
    monkeypatch.setattr(D, "_same_device", lambda *t: device)
    monkeypatch.setattr(D, "_pools", lambda *t: None)
    monkeypatch.setattr(D, "_table", lambda *t: None)
    monkeypatch.setattr(D, "_scope", lambda d, s: contextlib.nullcontext())
    monkeypatch.setattr(M, "make_args", lambda *a, **kw: M.PagedAttentionArgs(num_seqs=1, total_q=1))
    monkeypatch.setattr(M, "new_workspace", lambda n, d: SimpleNamespace(data_ptr=lambda: 256, numel=lambda: n,
                                                                        element_size=lambda: 1))
    monkeypatch.setattr(D, "load_library", lambda: SimpleNamespace(mvr_paged_attention_tree_workspace_size=lambda *a: 512))
    monkeypatch.setattr(D, "Call", lambda *a, **kw: made.update(kw, positional=a))
    t = SimpleNamespace(shape=(1, 1, 64, 16, 64), dtype="f16")
    current[0] = OTHER
    D.make_tree_call(t, t, t, t, t, t, t, t, max_q_len=1, max_seq_len=1)
    assert made["workspace_stream"] == OTHER
    given = M.new_workspace(512, device)
    D.make_tree_call(t, t, t, t, t, t, t, t, max_q_len=1, max_seq_len=1, workspace=given)
    assert made["workspace_stream"] is None
