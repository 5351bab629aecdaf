"""A graph goes on using the workspace that it was captured with after eager
calls have outgrown it."""
import pytest
import torch

from test_shared_prefix_gpu import Batch

pytestmark = pytest.mark.gpu


def test_replay_after_growth():
    from src import b200

    def attend(b, out):
        return b200.paged_attention(b.q, None, None, b.kc, b.vc, b.cu_q, b.cu_k, 1, b.max_k, b.scale, b.table, out=out)

    small = Batch(16, 2, [], alone=[1500, 700, 2000, 3], seed=41)
    out = torch.zeros_like(small.q)
    want = attend(small, out).clone()
    small.check(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(small, out)
    key = (torch.cuda.current_device(), "attn")
    first = b200._workspaces[key]
    b200.workspace("attn", first.numel() + 1, small.q.device)
    assert b200._workspaces[key].numel() >= 2 * first.numel()
    assert any(buf is first for _, buf in b200._outgrown)
    large = Batch(16, 2, [], alone=[900] * 40, seed=42)
    for _ in range(3):
        large.check(attend(large, torch.zeros_like(large.q)), range(0, 40, 9))
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert b200.device_error(clear=True) == 0
