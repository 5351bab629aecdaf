"""What stays of a workspace that was outgrown (host side)."""
import pytest
import torch


@pytest.fixture
def grow(monkeypatch):
    """grow(kind, nbytes) on CPU memory; grow.capturing: whether the stream is captured."""
    from src import b200
    real = torch.zeros

    def call(kind, nbytes, device=0):
        return b200.workspace(kind, nbytes, torch.device("cuda", device))

    call.capturing = False
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **kw: real(*a, **kw))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: call.capturing)
    monkeypatch.setattr(b200, "_stream_captured", lambda: call.capturing)
    monkeypatch.setattr(b200, "_raw_stream", lambda dev: 0x7003)
    monkeypatch.setattr(b200, "_workspaces", {})
    monkeypatch.setattr(b200, "_outgrown", [])
    monkeypatch.setattr(b200, "_captured", set(), raising=False)
    return call


MB = 1 << 20


@pytest.mark.parametrize("kind", ["attn", "gemm", "shared_prefix@7000"])
def test_growth_without_a_capture_keeps_nothing(grow, kind):
    """The context of an eager decode grows by and by."""
    from src import b200
    for n in range(1, 65):
        assert grow(kind, n * MB).numel() == n * MB
        assert grow(kind, MB).numel() == n * MB
    assert b200._outgrown == []


def test_what_a_graph_writes_to_is_kept(grow):
    from src import b200
    first = grow("attn", 3 * MB)
    grow.capturing = True
    assert grow("attn", 2 * MB) is first
    grow.capturing = False
    second = grow("attn", 4 * MB)
    assert second is not first and second.numel() == 6 * MB
    assert [(k, b is first) for k, b in b200._outgrown] == [((0, "attn"), True)]
    # the second was in no capture, nor any of the other device or kind
    grow("gemm", MB), grow("attn", MB, device=1)
    for n in (7, 8, 9):
        grow("attn", n * MB), grow("gemm", n * MB), grow("attn", n * MB, device=1)
    assert len(b200._outgrown) == 1


def test_what_is_kept_is_less_than_what_is_in_use(grow):
    from src import b200
    for n in range(1, 2000, 3):
        grow.capturing = False
        grow("attn", n * MB // 64)
        grow.capturing = True
        buf = grow("attn", 1)
    assert 0 < sum(b.numel() for _, b in b200._outgrown) < buf.numel()
    with pytest.raises(RuntimeError, match="before CUDA-graph capture"):
        grow("attn", 2 * buf.numel())
