"""The page pool, forks and shared-prefix attention together, as a serving
loop uses them: one prompt is prefilled, forked into several rows, decoded
with its prefix attended once, pruned, forked again and compacted -- against
the same sequences each with its own pages and plain paged attention."""
import pytest
import torch

from oracle import layers as L
from oracle.metadata import SeqState
from oracle.weights import Qwen3Shape, random_weights

pytestmark = pytest.mark.gpu

SHAPE = Qwen3Shape(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, inter=1024, vocab=4096, max_pos=8192)
PAGE = 256


@pytest.fixture(autouse=True)
def _clean_error_word():
    from src import b200
    b200.device_error(clear=True)
    yield
    assert b200.device_error(clear=True) == 0, "device error word set"


def runner(W, blocks, **kw):
    from src.engine.model_runner import ModelRunner
    r = ModelRunner(SHAPE.hf_config(), max_num_seqs=32, max_seq_len=4096, **kw)
    r.load_weights(W.items())
    r.allocate_kv_cache(blocks)
    r.kv_cache.zero_()
    return r


class Plain:
    """Sequences with their own blocks, decoded through ModelRunner.prepare."""

    def __init__(self, r):
        self.r, self.next, self.seqs = r, 0, {}

    def step(self, rows, tokens):
        """One step over the rows (tokens: list of new tokens per row)."""
        seqs = []
        for row, new in zip(rows, tokens):
            s = self.seqs.get(row)
            if s is None:
                s = self.seqs[row] = SeqState(token_ids=[], block_table=list(range(self.next, self.next + 8)))
                self.next += 8
            s.num_cached_tokens = len(s.token_ids)
            s.token_ids = s.token_ids + list(new)
            s.num_scheduled_tokens = len(new)
            seqs.append(s)
        ids, pos, ctx = self.r.prepare(seqs)
        return self.r.run_model(ids, pos, ctx)

    def fork(self, parent, child):
        """The child's tokens prefilled again into its own blocks."""
        tokens = self.seqs[parent].token_ids
        self.seqs.pop(child, None)
        self.step([child], [tokens])


@pytest.mark.parametrize("prompt", [1300, 1024, 700])
@pytest.mark.parametrize("mode", ["", "always"])
def test_fork_decode_prune_compact(prompt, mode, monkeypatch):
    monkeypatch.setenv("B200_SHARED_PREFIX", mode)
    W = random_weights(SHAPE, seed=3)
    g = torch.Generator().manual_seed(prompt)
    words = torch.randint(0, SHAPE.vocab, (prompt + 400,), generator=g).tolist()
    plain = Plain(runner(W, 200))
    r = runner(W, 64)
    pool = r.page_pool(16)
    i32 = dict(dtype=torch.int32, device="cuda")

    def pooled(rows, tokens, prefix=None):
        positions, ctx, done = pool.step(rows, [len(t) for t in tokens])
        if prefix is not None:
            ctx.prefix_group, ctx.prefix_lens = torch.zeros(len(rows), **i32), torch.tensor([prefix], **i32)
        ids = torch.tensor([t for new in tokens for t in new], dtype=torch.int64, device="cuda")
        out = r.run_model(ids, positions, ctx)
        assert done.tolist() == [1] * len(rows)
        return out

    def decode(rows, prefix, steps):
        nonlocal words
        for _ in range(steps):
            new = [[words.pop()] for _ in rows]
            got, want = pooled(rows, new, prefix), plain.step(rows, new)
            assert L.rel_err(got.cpu(), want.float().cpu()) <= 2e-2

    got, want = pooled([5], [words[:prompt]]), plain.step([5], [words[:prompt]])
    assert L.rel_err(got.cpu(), want.float().cpu()) <= 2e-2
    children = [0, 1, 2, 9, 11, 12, 13]
    pool.fork([5] * 7, children)
    for c in children:
        plain.fork(5, c)
    shared = prompt // PAGE * PAGE
    decode([5] + children, prompt, 3)
    # one page of prompt once, whatever the number of rows
    assert int((pool.refs == 8).sum()) == prompt // PAGE
    # prune: three rows go, one survivor is forked into two of them
    pool.free([5, 2, 13])
    pool.fork([11, 11], [2, 13])
    for row in (5, 2, 13):
        plain.seqs.pop(row)
    for c in (2, 13):
        plain.fork(11, c)
    rows = [0, 1, 2, 9, 11, 12, 13]
    decode(rows, shared, 2)
    # compaction moves pages and changes no result: the same step before and after
    lens = pool.seq_lens.clone()
    new = [[words.pop()] for _ in rows]
    before = pooled(rows, new, shared)
    pool.seq_lens.copy_(lens)
    place = pool.compact()
    live = int((pool.refs > 0).sum())
    assert bool((pool.refs[:live] > 0).all()) and bool((pool.block_tables < live).all())
    assert int((place >= 0).sum()) == live
    after = pooled(rows, new, shared)
    assert torch.equal(before, after)
    plain.step(rows, new)
    decode(rows, shared, 2)
    pool.free(list(range(16)))
    assert int(pool.refs.abs().sum()) == 0


@pytest.mark.parametrize("eager", [True, False])
def test_runner_with_prefix_cache_hits(eager):
    """ModelRunner(shared_prefix=True): sequences whose block tables begin with
    the same blocks, decoded eagerly and from captured graphs with padding,
    against the runner without it; batches with and without shared blocks
    through the same graphs."""
    W = random_weights(SHAPE, seed=4)
    g = torch.Generator().manual_seed(9)
    a, b = runner(W, 120), runner(W, 120, shared_prefix=True)
    system = torch.randint(0, SHAPE.vocab, (1536,), generator=g).tolist()
    other = torch.randint(0, SHAPE.vocab, (600,), generator=g).tolist()
    seqs, nxt = [], 20
    for i in range(13):
        head, blocks = (system, list(range(6))) if i % 3 else (other, [10, 11])
        tail = torch.randint(0, SHAPE.vocab, (5 + 37 * i,), generator=g).tolist()
        n = len(blocks)
        own = list(range(nxt, nxt + 4))
        nxt += 4
        seqs.append(SeqState(token_ids=head[:n * PAGE] + tail, block_table=blocks + own))
    for r in (a, b):
        for s in seqs:  # whole prompts, the shared blocks written again with the same values
            s.num_cached_tokens, s.num_scheduled_tokens = 0, len(s.token_ids)
            ids, pos, ctx = r.prepare([s])
            r.run_model(ids, pos, ctx)
        if not eager:
            r.capture_cudagraph([4, 16])
    for step, batch in enumerate((seqs, seqs[:3], seqs[4:5], seqs[1:], seqs)):
        for s in batch:
            s.num_cached_tokens = len(s.token_ids)
            s.token_ids.append(int(torch.randint(0, SHAPE.vocab, (1,), generator=g)))
            s.num_scheduled_tokens = 1
        outs = []
        for r in (a, b):
            ids, pos, ctx = r.prepare(batch)
            if r is b and step == 0:
                assert ctx.prefix_lens.tolist() in ([1536, 512], [512, 1536])
            outs.append(r.run_model(ids, pos, ctx).float().cpu())
        assert L.rel_err(outs[1], outs[0]) <= 2e-2, step
    for r in (a, b):
        r.release_graphs()
