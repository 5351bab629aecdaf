"""Grouping of sequences by the blocks their tables begin with (host side)."""
import itertools
import random

import numpy as np
import pytest
import torch


def groups(tables, lens, block=256):
    from src.engine.metadata import shared_prefixes
    return shared_prefixes(tables, lens, block)


def saved(group, prefix, block=256):
    """Block reads that the groups save."""
    return sum((int((group == g).sum()) - 1) * int(n) // block for g, n in enumerate(prefix))


def best(tables, lens, block):
    """The most that any cut of the sorted tables into runs saves, by recursion."""
    order = sorted(range(len(tables)), key=lambda b: tables[b])

    def common(members):
        n = min(min(len(tables[b]), lens[b] // block) for b in members)
        k = 0
        while k < n and len({tables[b][k] for b in members}) == 1:
            k += 1
        return k

    def solve(run):
        if len(run) < 2:
            return 0
        one = (len(run) - 1) * common(run)
        return max([one] + [solve(run[:i]) + solve(run[i:]) for i in range(1, len(run))])

    return solve(order)


def test_one_system_prompt():
    tables = [[7, 8, 9 + i] for i in range(5)] + [[50, 51]]
    group, prefix = groups(tables, [600] * 5 + [400])
    assert group.tolist() == [0] * 5 + [-1] and prefix.tolist() == [512]


def test_partial_blocks_and_short_sequences_do_not_count():
    # the second block is full in two of three sequences only
    group, prefix = groups([[1, 2], [1, 2, 3], [1, 2, 4]], [400, 520, 700])
    assert saved(group, prefix) == 2
    group, prefix = groups([[1], [1]], [255, 256])
    assert group.tolist() == [-1, -1] and prefix.size == 0


def test_the_longer_prefixes_win_over_the_common_one():
    # everybody shares one block, two pairs share five: 2 * 4 + ... > 3
    tables = [[1, 2, 3, 4, 5, 10], [1, 2, 3, 4, 5, 11], [1, 6, 7, 8, 9, 12], [1, 6, 7, 8, 9, 13]]
    group, prefix = groups(tables, [6 * 256] * 4)
    assert sorted(prefix.tolist()) == [1280, 1280] and group[0] == group[1] != group[2] == group[3]
    # and the common one wins where it saves more
    tables = [[1, 2, i] for i in range(10, 18)] + [[1, 2, 3, 20], [1, 2, 3, 21]]
    group, prefix = groups(tables, [1024] * 10)
    assert set(group.tolist()) == {0} and prefix.tolist() == [512]


def test_empty_and_single():
    assert groups([], [])[0].size == 0
    group, prefix = groups([[3, 4]], [512])
    assert group.tolist() == [-1] and prefix.size == 0
    group, prefix = groups([[], []], [0, 0])
    assert group.tolist() == [-1, -1]


@pytest.mark.parametrize("seed", range(30))
def test_against_exhaustive_search(seed):
    rng = random.Random(seed)
    fresh = itertools.count(1000)
    tables = [[rng.choice([1, 2])]]
    for _ in range(rng.randint(1, 9)):
        t = list(rng.choice(tables))
        t = t[:rng.randint(0, len(t))] + [next(fresh) for _ in range(rng.randint(0, 3))]
        tables.append(t or [next(fresh)])
    lens = [max(1, len(t) * 4 - rng.randint(0, 5)) for t in tables]
    group, prefix = groups(tables, lens, 4)
    # (rows that inner groups leave over may form a group of their own: more than any cut into runs)
    assert saved(group, prefix, 4) >= best(tables, lens, 4)
    for g, n in enumerate(prefix):
        members = [b for b in range(len(tables)) if group[b] == g]
        assert len(members) >= 2 and n > 0 and all(lens[b] >= n for b in members)
        assert len({tuple(tables[b][:n // 4]) for b in members}) == 1


def test_a_thousand_nested_prefixes():
    """Deep nesting does not recurse."""
    tables = [list(range(i + 1)) for i in range(1000)]
    group, prefix = groups(tables, [len(t) * 256 for t in tables])
    assert saved(group, prefix) >= 249 * 500 - 1000
    assert group.dtype == np.int32 and prefix.dtype == np.int32


@pytest.mark.parametrize("rows,counts", [([0, -1], [1, 1]), ([0, 4], [1, 1]), ([2, 2], [1, 1]), ([0, 1, 2], [1]),
                                         ([0, 1], [1, 0]), ([], [])])
def test_pool_steps_refuse_rows_that_have_no_place(rows, counts):
    from src.engine.pages import PagePool
    pool = PagePool(torch.zeros(2, 1, 6, 16, 1, 8), 4, 64)
    with pytest.raises(ValueError, match="step"):
        pool.step(rows, counts)
    assert pool.seq_lens.tolist() == [0] * 4


@pytest.mark.parametrize("kw", [dict(max_num_seqs=1025), dict(block_size=128), dict(heads=(9, 1))])
def test_a_runner_refuses_what_the_kernel_cannot(kw):
    from types import SimpleNamespace
    from src.engine.model_runner import ModelRunner
    q, kv = kw.pop("heads", (16, 8))
    config = SimpleNamespace(num_attention_heads=q, num_key_value_heads=kv)
    with pytest.raises(ValueError, match="shared_prefix"):
        ModelRunner(config, shared_prefix=True, device=torch.device("cpu"), **kw)
