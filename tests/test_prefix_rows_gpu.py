"""Rows that shared-prefix attention does not answer: they are left out and
flagged, the others are answered as if they were not there."""
import pytest
import torch

from test_shared_prefix_gpu import Batch, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["", "always"])
@pytest.mark.parametrize("group", [-1, 0])
@pytest.mark.parametrize("queries", [2, 5])
@pytest.mark.parametrize("at", [0, 2, 4])
def test_a_sequence_of_several_queries_is_left_out(at, queries, group, mode, monkeypatch):
    from src import b200
    monkeypatch.setenv("B200_SHARED_PREFIX", mode)
    b200.device_error(clear=True)
    b = Batch(8, 2, [(512, 512, [3, 700, 5, 90])], alone=[300], seed=31)
    b.group[at] = group
    kw = dict(group=i32(b.group), prefix=i32(b.prefix))
    # one row of q for every query, the others' rows moved back
    rows = [r for r in range(b.B)]
    q = b.q.repeat_interleave(i32([queries if r == at else 1 for r in rows]).long(), 0)
    starts = [r + (queries - 1 if r > at else 0) for r in rows]
    b.cu_q = i32(starts + [b.B + queries - 1])
    out = torch.full_like(q, 7.0)
    b.run(q=q, out=out, **kw)
    assert b200.device_error(clear=True) == 4
    assert bool((out[at:at + queries] == 7.0).all())
    b.check(out[i32(starts).long()], [r for r in rows if r != at])
