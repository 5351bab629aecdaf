"""Which workspace a call of shared-prefix attention gets (host side): one that
no call which may run at the same time has."""
import contextlib

import pytest
import torch


@pytest.fixture
def host(monkeypatch):
    """The binding on CPU tensors: `stream` is the current stream's handle, `capturing` whether it is
    captured, `used` the workspaces (address, bytes) that the calls were given, kept alive in `held`."""
    from src import b200

    class Host:
        stream, capturing, used, held = 0, False, [], []

        def call(self, **kw):
            i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
            q, kv = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((2, 4, 128), (3, 256, 2, 128)))
            b200.shared_prefix_attention(q, kv, kv, i32(3), i32(3), kw.pop("keys", 1000), 0.1, i32(2, 3), i32(2),
                                         i32(1), **kw)
            return self.used[-1]

    h = Host()
    h.used, h.held = [], []
    real_zeros, real_empty = torch.zeros, torch.empty

    def on_cpu(make):
        def made(*a, device=None, **kw):
            t = make(*a, **kw)
            h.held.append(t)
            return t
        return made

    monkeypatch.setattr(torch, "zeros", on_cpu(real_zeros))
    monkeypatch.setattr(torch, "empty", on_cpu(real_empty))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: h.capturing)
    monkeypatch.setattr(b200, "_stream_captured", lambda: h.capturing, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(b200, "_raw_stream", lambda dev: h.stream)
    monkeypatch.setattr(b200, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(b200, "shared_prefix_workspace_bytes", lambda seqs, keys, hq, hkv: 2 << 20 if keys > 5000 else 4096)
    monkeypatch.setattr(b200, "_call", lambda name, dev, *a: h.used.append((a[-2], a[-1])))
    monkeypatch.setattr(b200, "_workspaces", {})
    monkeypatch.setattr(b200, "_outgrown", [])
    monkeypatch.setattr(b200, "_prefix_ws_bytes", {})
    monkeypatch.setattr(b200, "_prefix_workspaces", [], raising=False)
    return h


def test_streams_have_workspaces_of_their_own(host):
    first = host.call()
    host.stream = 0x7001
    other = host.call()
    assert other[0] != first[0]
    host.stream = 0x7002
    assert host.call()[0] not in (first[0], other[0])
    host.stream = 0
    assert host.call() == first  # the same stream, the same workspace
    host.stream = 0x7001
    assert host.call() == other


def test_captured_calls_share_nothing_with_eager_ones_or_other_graphs(host):
    host.stream = 0x7003  # every capture runs on the same side stream
    eager = host.call()
    host.capturing = True
    graphs = [host.call(), host.call()]
    assert len({eager[0], *(g[0] for g in graphs)}) == 3
    for at, _ in graphs:  # zeroed by the graph itself
        buf = next(t for t in host.held if t.data_ptr() == at)
        assert not bool(buf[:256].any())
    host.capturing = False
    assert host.call() == eager


def test_a_caller_may_hold_the_workspace(host):
    from src import b200
    ws = b200.shared_prefix_workspace(2, 1000, 4, 2, torch.device("cuda", 0))
    room = torch.zeros(4096 + 512, dtype=torch.uint8)
    at = -room.data_ptr() % 256
    for stream, capturing in ((0, False), (5, False), (5, True)):
        host.stream, host.capturing = stream, capturing
        assert host.call(workspace=room[at:at + 4096]) == (room.data_ptr() + at, 4096)
    assert ws.numel() == 4096
    with pytest.raises(ValueError, match="4096 needed"):
        host.call(workspace=room[at:at + 4095])
    with pytest.raises(ValueError, match="boundary"):
        host.call(workspace=room[at + 16:])
    with pytest.raises(TypeError, match="uint8"):
        host.call(workspace=torch.zeros(4096))
    with pytest.raises(TypeError, match="contiguous"):
        host.call(workspace=room[at::2])
    with pytest.raises(ValueError, match="2097152 needed"):
        host.call(workspace=room[at:], keys=6000)


def test_held_and_stream_workspaces_are_cleared_after_a_timeout(host, monkeypatch):
    import types
    from src import b200

    def error_word(p, clear):
        p._obj.value = 1
        return 0
    host.stream = 0x7001
    host.call()
    ws = b200.shared_prefix_workspace(2, 1000, 4, 2, torch.device("cuda", 0))
    gone = b200.shared_prefix_workspace(2, 1000, 4, 2, torch.device("cuda", 0))
    host.held[:] = [t for t in host.held if t is not gone]
    del gone
    assert sum(r() is not None for r in b200._prefix_workspaces) == 1
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(b200, "load_library", lambda: types.SimpleNamespace(b200_device_error=error_word))
    monkeypatch.setattr(b200, "attention_workspace_bytes", lambda *a: 512)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    (buf,) = b200._workspaces.values()
    buf.fill_(1)
    ws.fill_(1)
    assert b200.device_error(clear=True) == 1
    assert int(buf.sum()) == buf.numel() - 256 and int(ws.sum()) == ws.numel() - 256
