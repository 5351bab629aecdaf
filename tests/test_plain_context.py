"""Attention over a step record that has only the reference's fields
(src/utils/context.py:5-14): the layers are copied into trees that keep their
own Context, which knows nothing of shared prefixes."""
from types import SimpleNamespace

import pytest
import torch


@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("paged", [True, False])
def test_a_context_without_prefix_fields_takes_the_paged_path(monkeypatch, q_len, paged):
    from src import b200
    from src.layers import attention
    seen = []
    monkeypatch.setattr(b200, "paged_attention", lambda *a, **kw: seen.append(a) or a[0])
    monkeypatch.setattr(b200, "shared_prefix_attention", lambda *a, **kw: pytest.fail("no groups were given"))
    i = torch.zeros(2, dtype=torch.int32)
    ctx = SimpleNamespace(is_prefill=q_len > 1, cu_seqlens_q=i, cu_seqlens_k=i, max_seqlen_q=q_len, max_seqlen_k=3,
                          slot_mapping=i, context_lens=i, block_tables=i.view(1, 2) if paged else None)
    q = torch.zeros(q_len, 2, 128)
    assert attention.attend(q, q, q, q, q, ctx, 0.1) is q
    assert len(seen) == 1 and (seen[0][10] is None) == (not paged)


def test_a_context_with_groups_takes_the_shared_path(monkeypatch):
    from src import b200
    from src.layers import attention
    from src.utils.context import Context
    seen = []
    monkeypatch.setattr(b200, "shared_prefix_attention", lambda *a, **kw: seen.append(a) or a[0])
    i = torch.zeros(2, dtype=torch.int32)
    ctx = Context(cu_seqlens_q=i, cu_seqlens_k=i, max_seqlen_q=1, max_seqlen_k=3, block_tables=i.view(1, 2),
                  prefix_group=i[:1], prefix_lens=i)
    q = torch.zeros(1, 2, 128)
    assert attention.attend(q, q, q, q, q, ctx, 0.1) is q and len(seen) == 1
