"""Groups that a caller puts into the step's context himself (rows of a page
pool): singles and unused ones among them are allowed, so there can be more
groups than the captured graphs have places for."""
import pytest
import torch

from oracle.weights import random_weights
from oracle.metadata import SeqState
from test_shared_pool_gpu import PAGE, SHAPE, runner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [1, 2, 3, 5, 9, 40])
def test_more_groups_than_half_the_batch(groups):
    from src import b200
    W = random_weights(SHAPE, seed=6)
    r = runner(W, 40, shared_prefix=True)
    g = torch.Generator().manual_seed(groups)
    seqs = []
    for i in range(3):
        tokens = torch.randint(0, SHAPE.vocab, (2 * PAGE + 20 + i,), generator=g).tolist()
        seqs.append(SeqState(token_ids=tokens, block_table=list(range(4 * i, 4 * i + 4))))
    for s in seqs:
        s.num_cached_tokens, s.num_scheduled_tokens = 0, len(s.token_ids)
        ids, pos, ctx = r.prepare([s])
        r.run_model(ids, pos, ctx)
    for s in seqs:
        s.num_cached_tokens = len(s.token_ids)
        s.token_ids.append(5)
        s.num_scheduled_tokens = 1

    def step():
        ids, pos, ctx = r.prepare(seqs)
        # the last groups, of one sequence each
        ctx.prefix_group = torch.tensor([max(groups - 1 - i, 0) for i in range(3)], dtype=torch.int32, device="cuda")
        if groups < 3:
            ctx.prefix_group.fill_(-1)
        ctx.prefix_lens = torch.full((groups,), 2 * PAGE, dtype=torch.int32, device="cuda")
        return r.run_model(ids, pos, ctx).clone()

    b200.device_error(clear=True)
    want = step()
    r.capture_cudagraph([4, 16])
    got = step()
    assert b200.device_error(clear=True) == 0
    assert torch.equal(got, want)
    r.release_graphs()
