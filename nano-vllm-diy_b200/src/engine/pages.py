"""A pool of KV-cache pages whose tables live on the device.

The reference's BlockManager (src/engine/block_manager.py:47) owns its tables
on the host and never copies a page.  PagePool keeps the same three things
next to the cache -- block tables (-1 padded), token counts and per-page
reference counts -- as int32 tensors that kernels change in stream order, so a
step can fork sequences (parallel samples, beams), drop them, or squeeze the
cache without the host reading anything back:

    pool = PagePool(runner.kv_cache, max_rows=256, max_len=8192)
    positions, ctx, done = pool.step([0], [len(prompt)])   # pages + metadata of a prefill
    pool.fork([0, 0, 0], [1, 2, 3])                       # three more samples of row 0
    positions, ctx, done = pool.step([0, 1, 2, 3], [1] * 4)  # one decode token each
    pool.free([2]); pool.compact()

Rows are given as lists or as int32 device tensors; -1 entries are skipped
(but not in a step).
`done` is an int32 device tensor, 1 where the row got what it asked for (0
when pages ran out, see src/b200.py).
"""
from __future__ import annotations

import torch

from src import b200
from src.utils.context import Context


class PagePool:

    def __init__(self, kv_cache: torch.Tensor, max_rows: int, max_len: int):
        self.kv_cache = kv_cache
        self.num_pages, self.page = kv_cache.shape[-4], kv_cache.shape[-3]
        self.device = kv_cache.device
        self.width = (max_len + self.page - 1) // self.page
        i32 = dict(dtype=torch.int32, device=self.device)
        self.block_tables = torch.full((max_rows, self.width), -1, **i32)
        self.seq_lens = torch.zeros(max_rows, **i32)
        self.refs = torch.zeros(self.num_pages, **i32)

    def _vec(self, x) -> torch.Tensor:
        return x if torch.is_tensor(x) else torch.tensor(x, dtype=torch.int32).to(self.device, non_blocking=True)

    def take(self, rows, new_lens) -> torch.Tensor:
        """The rows grow to new_lens tokens."""
        return b200.take_pages(self.block_tables, self.seq_lens, self.refs, self._vec(rows), self._vec(new_lens),
                               self.page)

    def fork(self, parents, children) -> torch.Tensor:
        """children[i] (empty rows) become copies of parents[i]."""
        return b200.fork_pages(self.kv_cache, self.block_tables, self.seq_lens, self.refs, self._vec(parents),
                               self._vec(children))

    def free(self, rows) -> None:
        b200.free_pages(self.block_tables, self.seq_lens, self.refs, self._vec(rows))

    def compact(self) -> torch.Tensor:
        """Live pages into the front of the cache; returns where each page went (-1: free).  The contexts of
        steps prepared before it name the old places."""
        return b200.compact_pages(self.kv_cache, self.block_tables, self.refs)

    def copy(self, src, dst, num_tokens=None) -> None:
        """Pages dst[i] := src[i]; the tables stay as they are."""
        b200.copy_pages(self.kv_cache, self._vec(src), self._vec(dst),
                        None if num_tokens is None else self._vec(num_tokens))

    def step(self, rows, counts: list[int]) -> tuple[torch.Tensor, Context, torch.Tensor]:
        """Pages for counts[i] more tokens of each row and the step's metadata:
        (positions int64 [T], Context, done).  The Context is that of the rows
        in the order given, as src/engine/metadata.py builds it.  Every row is
        one of the pool's, named once: a step skips none (a row with done = 0 has
        no page for its tokens: their slots are refused and flagged)."""
        if not torch.is_tensor(rows) and (len(set(rows)) != len(rows) or
                                          not all(0 <= r < self.seq_lens.shape[0] for r in rows)):
            raise ValueError(f"step: rows {rows} of a pool of {self.seq_lens.shape[0]}, each once")
        if len(counts) != len(rows) or not counts or min(counts) < 1:
            raise ValueError(f"step: {len(counts)} token counts (of at least 1) for {len(rows)} rows")
        rows = self._vec(rows)
        at = rows.long()
        count = self._vec(counts)
        start = self.seq_lens[at]
        done = self.take(rows, start + count)
        table = self.block_tables[at]
        end = start + count
        # (a refused row may ask for more pages than a table has places)
        held = torch.clamp((end + self.page - 1) // self.page, max=self.width)
        info = torch.stack([start, count, held])
        total = sum(counts)
        positions, slots, cu_q, cu_k, lens = b200.step_metadata(info, table, self.page, total, total)
        most = max(counts)
        # the largest length is known on the device only: the pool's bound stands in for it
        ctx = Context(is_prefill=most != 1, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=most,
                      max_seqlen_k=self.width * self.page, slot_mapping=slots, context_lens=lens, block_tables=table)
        return positions, ctx, done
