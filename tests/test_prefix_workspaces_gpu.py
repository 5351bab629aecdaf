"""Shared-prefix attention from several streams, graphs and host threads at
once: every call gives what it gives alone, bit for bit."""
import pytest
import torch

from test_shared_prefix_gpu import Batch, i32

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _clean_error_word(monkeypatch):
    from src import b200
    monkeypatch.setenv("B200_SHARED_PREFIX", "always")
    b200.device_error(clear=True)
    yield
    assert b200.device_error(clear=True) == 0, "device error word set"


def batches():
    """Different shapes, so that parts of one batch would be wrong in another."""
    made = [Batch(8, 2, [(1024, 1024, [400, 3, 90] * 5)], alone=[700], seed=21),
            Batch(16, 2, [(512, 512, [40, 1200, 8, 9])], alone=[30] * 9, seed=22),
            Batch(32, 8, [(1536, 1536, [5, 600] * 12), (256, 256, [3, 4])], seed=23)]
    for b in made:
        b.args = dict(group=i32(b.group), prefix=i32(b.prefix))
        b.want = b.run(**b.args)
        b.check(b.want)
    torch.cuda.synchronize()
    return made


def test_calls_on_several_streams_at_once():
    from src import b200
    made = batches()
    streams = [torch.cuda.Stream() for _ in made]
    outs = [[] for _ in made]
    for _ in range(8):
        for b, st, out in zip(made, streams, outs):
            with torch.cuda.stream(st):
                out.append(b.run(**b.args))
    torch.cuda.synchronize()
    for b, out in zip(made, outs):
        assert all(torch.equal(o, b.want) for o in out)
    used = [b200._workspaces[0, f"shared_prefix@{st.cuda_stream:x}"] for st in streams]
    assert len({w.data_ptr() for w in used}) == len(made)
    assert not any(bool(w[:256].any()) for w in used)


def test_graphs_replayed_on_several_streams_at_once():
    """Captured one after the other on the capture stream, without a call
    before that would have sized anything; replayed side by side."""
    made = batches()
    streams = [torch.cuda.Stream() for _ in made]
    outs = [[torch.zeros_like(b.q) for _ in range(3)] for b in made]
    graphs = []
    for b, out in zip(made, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for o in out:
                b.run(out=o, **b.args)
    for _ in range(3):
        for out in outs:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        for b in made:  # and eager calls beside them
            assert torch.equal(b.run(**b.args), b.want)
        torch.cuda.synchronize()
        for b, out in zip(made, outs):
            assert all(torch.equal(o, b.want) for o in out)


def test_workspace_of_the_caller():
    from src import b200
    made = batches()
    ws = b200.shared_prefix_workspace(64, 4096, 32, 8)
    for b in made:
        assert torch.equal(b.run(workspace=ws, **b.args), b.want)
    graph = torch.cuda.CUDAGraph()
    outs = [torch.zeros_like(b.q) for b in made]
    with torch.cuda.graph(graph):
        for b, out in zip(made, outs):
            b.run(out=out, workspace=ws, **b.args)
    for _ in range(2):
        graph.replay()
    for b, out in zip(made, outs):
        assert torch.equal(out, b.want)
    assert not bool(ws[:256].any())
    with pytest.raises(ValueError, match="needed"):
        made[0].run(workspace=ws[:4096], **made[0].args)
