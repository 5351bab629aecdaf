"""Page operators (copy, take, fork, free, compact) against the same rules
restated with Python lists.  Tables, lengths, counts and cache bytes have to
be equal: nothing here rounds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _clean_error_word():
    from src import b200
    b200.device_error(clear=True)
    yield
    assert b200.device_error(clear=True) == 0, "device error word set"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Model:
    """The rules, on lists; the cache on the CPU."""

    def __init__(self, kv, rows, width):
        self.kv = kv
        self.pages, self.page = kv.shape[-4], kv.shape[-3]
        self.width = width
        self.table = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.refs = [0] * self.pages

    def free_list(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def held(self, n):
        return -(-n // self.page)

    def take(self, rows, new_lens):
        free, used, done, seen = self.free_list(), 0, [], set()
        for r, n in zip(rows, new_lens):
            ok = 0 <= r < len(self.lens) and r not in seen and n >= self.lens[r] and self.held(n) <= self.width
            seen.add(r)
            need = self.held(n) - self.held(self.lens[r]) if ok else 0
            used += need
            ok = ok and (need == 0 or used <= len(free))
            done.append(int(ok))
            if ok:
                h = self.held(self.lens[r])
                for j, p in enumerate(free[used - need:used]):
                    self.table[r][h + j] = p
                    self.refs[p] = 1
                self.lens[r] = n
        return done

    def free(self, rows):
        for r in rows:
            if r < 0:
                continue
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r] = [-1] * self.width
            self.lens[r] = 0

    def fork(self, parents, children):
        lens, free, used, done, seen = list(self.lens), self.free_list(), 0, [], set()
        for a, c in zip(parents, children):
            if a < 0 or c < 0:
                done.append(0)
                continue
            ok = c not in seen and lens[c] == 0
            seen.add(c)
            full, part = divmod(lens[a], self.page)
            used += int(ok and part > 0)
            ok = ok and (part == 0 or used <= len(free))
            done.append(int(ok))
            if not ok:
                continue
            for j in range(full):
                self.table[c][j] = self.table[a][j]
                self.refs[self.table[a][j]] += 1
            if part:
                p = free[used - 1]
                self.refs[p] = 1
                self.table[c][full] = p
                self.kv[..., p, :part, :, :] = self.kv[..., self.table[a][full], :part, :, :]
            self.lens[c] = lens[a]
        return done

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        movers = [p for p in range(n, self.pages) if self.refs[p] > 0]
        place = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        for a, b in zip(movers, holes):
            self.kv[..., b, :, :, :] = self.kv[..., a, :, :, :]
            self.refs[b], self.refs[a], place[a] = self.refs[a], 0, b
        self.table = [[place[e] if e >= 0 else -1 for e in row] for row in self.table]
        return place


def make(shape, rows, width, dtype=torch.bfloat16, seed=0):
    from src.engine.pages import PagePool
    g = torch.Generator().manual_seed(seed)
    kv = torch.randint(-1000, 1000, shape, generator=g).to(dtype)
    pool = PagePool(kv.to(DEV), rows, width * shape[-3])
    return pool, Model(kv.clone(), rows, width)


def same(pool, model):
    assert pool.block_tables.tolist() == model.table
    assert pool.seq_lens.tolist() == model.lens
    assert pool.refs.tolist() == model.refs
    assert torch.equal(pool.kv_cache.cpu(), model.kv)


SHAPES = [  # planes, pages, page, heads, dim: one plane, odd counts, pages of a piece and of several, a ragged last piece
    ((9, 16, 1, 8), torch.bfloat16), ((2, 3, 37, 32, 1, 128), torch.bfloat16),
    ((2, 2, 23, 256, 8, 128), torch.bfloat16), ((3, 41, 48, 3, 24), torch.bfloat16),
    ((2, 1, 19, 512, 3, 128), torch.float8_e4m3fn), ((2, 2, 13, 256, 1, 64), torch.float32),
]


@pytest.mark.parametrize("shape,dtype", SHAPES)
def test_copy_pages(shape, dtype):
    pool, model = make(shape, 1, 1, dtype, seed=1)
    pages, page = model.pages, model.page
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).tolist()
    half = pages // 2
    src, dst = perm[:half], perm[half:2 * half]
    src[-1] = src[0]  # one source, two destinations
    src, dst = src + [-1, src[1]], dst + [perm[0], -1]  # skipped on either side
    n = [(i * 13) % (page + 1) for i in range(len(src))]
    n[0], n[1] = 0, page
    for tokens in (n, None):
        pool.copy(src, dst, tokens)
        for k, (a, b) in enumerate(zip(src, dst)):
            if a >= 0 and b >= 0:
                t = page if tokens is None else tokens[k]
                model.kv[..., b, :t, :, :] = model.kv[..., a, :t, :, :]
        assert torch.equal(pool.kv_cache.cpu().view(torch.uint8), model.kv.view(torch.uint8))


def test_copy_pages_of_strided_planes():
    """Planes interleaved page by page, and a part of the layers: only strides change."""
    from src import b200
    base = torch.randint(-99, 99, (11, 2, 5, 32, 2, 64)).to(torch.bfloat16)
    dev = base.to(DEV)
    view, ref = dev.permute(1, 2, 0, 3, 4, 5)[:, 1:4], base.permute(1, 2, 0, 3, 4, 5)[:, 1:4]
    b200.copy_pages(view, i32([3, 7]), i32([0, 10]), i32([32, 5]))
    ref[:, :, 0] = ref[:, :, 3].clone()
    ref[:, :, 10, :5] = ref[:, :, 7, :5].clone()
    assert torch.equal(dev.cpu(), base)


def test_copy_pages_past_31_bits():
    """Pages more than 2^31 bytes (and elements) from the start of the cache."""
    from src import b200
    kv = torch.zeros(1, 2, 4200, 256, 8, 128, dtype=torch.bfloat16, device=DEV)  # 2.2e9 elements
    kv[0, 1, 4199] = 3.0
    kv[0, 0, 4199] = 2.0
    b200.copy_pages(kv, i32([4199]), i32([4150]))
    assert bool((kv[0, 1, 4150] == 3).all()) and bool((kv[0, 0, 4150] == 2).all())
    assert int(torch.count_nonzero(kv[0, 1, :4150])) == 0


@pytest.mark.parametrize("rows,width,pages,seed", [(3, 2, 7, 0), (40, 5, 90, 1), (300, 9, 1500, 2), (17, 64, 1029, 3),
                                                    (1000, 3, 2100, 4)])
def test_random_histories(rows, width, pages, seed):
    """Take, fork, free and compact in random order, pages running out on the
    way, with repeated and skipped rows: everything equal after every call."""
    pool, model = make((2, 1, pages, 16, 1, 8), rows, width, seed=seed)
    g = torch.Generator().manual_seed(seed + 100)

    def some(n, lo, hi):
        return torch.randint(lo, hi, (n,), generator=g).tolist()

    for step in range(24):
        n = some(1, 1, min(rows, 300) + 1)[0]
        kind = ("take", "take", "fork", "free", "take", "compact")[step % 6]
        if kind == "take":
            r = some(n, -1, rows)
            lens = [model.lens[x] + k for x, k in zip(r, some(n, -3, 16 * width // 2))]
            r_model = [x if x >= 0 else len(model.lens) + 1 for x in r]
            assert pool.take(r, [max(x, -5) for x in lens]).tolist() == model.take(r_model, lens), step
        elif kind == "fork":
            a, c = some(n, -1, rows), some(n, -1, rows)
            if step % 12 == 2:
                pool.free(c)
                model.free(c)
            assert pool.fork(a, c).tolist() == model.fork(a, c), step
        elif kind == "free":
            r = some(max(1, n // 2), -1, rows)
            r += r[:2]
            pool.free(r)
            model.free(r)
        else:
            place = pool.compact()
            assert place.tolist() == model.compact(), step
        same(pool, model)


def test_fork_edges():
    """Full last page (nothing copied), empty parent, one parent of many, a
    child that is also a parent, no free page left."""
    pool, model = make((2, 2, 6, 16, 2, 8), 8, 4, seed=5)
    for x in (pool, model):
        x.take([0, 1], [32, 17])       # two full pages; one full and one token: 4 of 6 pages
    calls = [([0, 3, 1], [2, 4, 5]),   # full pages only; an empty parent; a copied page
             ([1, 5], [6, 7]),         # one page left, two wanted
             ([7, 0], [3, 7])]         # 7 is empty before the call and forked in it
    for a, c in calls:
        assert pool.fork(a, c).tolist() == model.fork(a, c)
        same(pool, model)
    assert pool.fork([0], [1]).tolist() == [0]  # holds pages
    same(pool, model)
    assert pool.fork([], []).numel() == 0


def test_refs_not_aligned_and_uneven():
    """refs as a view that does not start on 16 bytes, table rows wider than the table."""
    from src import b200
    refs = torch.zeros(1 + 777, dtype=torch.int32, device=DEV)[1:]
    wide = torch.full((5, 16), -1, dtype=torch.int32, device=DEV)
    table, lens = wide[:, 3:12], torch.zeros(5, dtype=torch.int32, device=DEV)
    refs[::2] = 7
    done = b200.take_pages(table, lens, refs, i32([4, 2]), i32([16 * 9, 33]), 16)
    assert done.tolist() == [1, 1]
    assert table[4].tolist() == list(range(1, 19, 2)) and table[2].tolist() == [19, 21, 23] + [-1] * 6
    assert int((wide >= 0).sum()) == 12 and int(refs.sum()) == 7 * 389 + 12
    b200.free_pages(table, lens, refs, i32([2, 4, 4, -1]))
    assert int((wide >= 0).sum()) == 0 and int(refs.sum()) == 7 * 389 and lens.tolist() == [0] * 5


def test_captured_in_a_graph_and_on_another_stream():
    """A beam step (free + fork) and a compaction replayed from a graph give
    what the eager calls give."""
    pool, model = make((2, 2, 40, 16, 2, 8), 12, 4, seed=6)
    for x in (pool, model):
        x.take(list(range(8)), [5, 20, 33, 48, 64, 1, 16, 17])
    parents, children = i32([0, 1, 1, 2, -1]), i32([5, 6, 9, 10, 11])
    state = [t.clone() for t in (pool.block_tables, pool.seq_lens, pool.refs, pool.kv_cache)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.free(children)
        pool.fork(parents, children)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.free(children)
        done = pool.fork(parents, children)
        place = pool.compact()
    for t, s in zip((pool.block_tables, pool.seq_lens, pool.refs, pool.kv_cache), state):
        t.copy_(s)
    p, c = parents.tolist(), children.tolist()
    for _ in range(2):
        graph.replay()
        model.free(c)
        assert done.tolist() == model.fork(p, c)
        assert place.tolist() == model.compact()
        same(pool, model)


def test_bad_entries_are_skipped_and_flagged():
    """Rows, pages and token counts out of range change nothing and set the
    error bit."""
    from src import b200
    pool, model = make((1, 2, 9, 16, 1, 8), 4, 3, seed=7)
    for x in (pool, model):
        x.take([0, 1], [20, 40])
    bad = [lambda: pool.copy([9, 1], [2, 1 << 30]), lambda: pool.copy([1, 1], [6, 6], [17, -1]),
           lambda: pool.take([4, -2], [5, 5]), lambda: pool.free([4, 1 << 30, -7]),
           lambda: pool.fork([0, 4, -3], [7, 2, 2])]
    for call in bad:
        done = call()
        assert b200.device_error(clear=True) == 4
        assert done is None or not any(done.tolist())
        same(pool, model)
    # a table that names pages which are not there
    pool.block_tables[1, 0] = 9
    pool.block_tables[1, 1] = -9
    pool.free([1])
    assert b200.device_error(clear=True) == 4
    assert pool.block_tables[1].tolist() == [-1] * 3 and pool.refs.sum().item() == 4
    pool.block_tables[0, 1] = 77
    assert pool.fork([0], [3]).tolist() == [0]
    assert b200.device_error(clear=True) == 4


def test_pool_step_matches_host_metadata():
    """The pool's step metadata against the host builder on the same tables."""
    from oracle.metadata import SeqState, prepare_seqs
    from src.engine.pages import PagePool
    kv = torch.zeros(2, 1, 64, 256, 1, 128, dtype=torch.bfloat16, device=DEV)
    pool = PagePool(kv, 8, 2048)
    lens = [0] * 8
    for rows, counts in (([0, 3, 5], [300, 1, 700]), ([5, 0, 3], [1, 1, 1]), ([3, 7], [600, 256])):
        positions, ctx, done = pool.step(rows, counts)
        assert done.tolist() == [1] * len(rows)
        table = pool.block_tables.tolist()
        seqs = [SeqState(token_ids=[0] * (lens[r] + c), num_cached_tokens=lens[r], num_scheduled_tokens=c,
                         block_table=[p for p in table[r] if p >= 0]) for r, c in zip(rows, counts)]
        want = prepare_seqs(seqs, 256)
        assert positions.tolist() == want["positions"].tolist()
        for name in ("cu_seqlens_q", "cu_seqlens_k", "slot_mapping"):
            assert getattr(ctx, name).tolist() == want[name].tolist(), name
        for r, c in zip(rows, counts):
            lens[r] += c
        assert pool.seq_lens.tolist() == lens


def test_many_pages():
    """A pool of more than 65,536 pages, whose free pages are searched in the
    counts themselves, and rows of thousands of pages."""
    pool, model = make((1, 70001, 16, 1, 8), 40, 2000, seed=9)
    lens = [16 * 1900 + 5 * i for i in range(36)]
    for x in (pool, model):
        done = x.take(list(range(36)), lens)
        x.free(list(range(1, 36, 2)))
    assert torch.as_tensor(done).tolist() == [1] * 36
    same(pool, model)
    assert pool.fork([0, 2, 34], [1, 3, 36]).tolist() == model.fork([0, 2, 34], [1, 3, 36])
    calls = [[5, 7, 8, 9, 37, 38], [16 * 2000, 1, 16 * 1999, 16 * 1500, 3, 16 * 2000]]
    assert pool.take(*calls).tolist() == model.take(*calls)
    same(pool, model)
    assert pool.compact().tolist() == model.compact()
    same(pool, model)
    pool.free(list(range(40)))
    model.free(list(range(40)))
    same(pool, model)
    assert sum(model.refs) == 0


def test_launches_that_may_overlap(monkeypatch):
    """The same results where every launch may begin before the one in front of
    it has ended."""
    monkeypatch.setenv("B200_PDL", "1")
    pool, model = make((2, 2, 64, 16, 2, 8), 12, 6, seed=10)
    for _ in range(3):
        for x in (pool, model):
            x.take([0, 1, 2], [90, 33, 16])
            x.fork([0, 1, 2, 0], [3, 4, 5, 6])
            x.free([1, 3])
            x.compact()
            x.take([1, 3], [16, 7])
            x.free([0, 1, 2, 3, 4, 5, 6])
    same(pool, model)


def test_pool_step_past_the_longest_row_is_refused():
    """A row that would outgrow its table keeps its pages and its length; its
    tokens without a page have no slot, and the other rows get theirs."""
    from src import b200
    from src.engine.pages import PagePool
    kv = torch.zeros(2, 1, 9, 16, 1, 8, dtype=torch.bfloat16, device=DEV)
    pool = PagePool(kv, 3, 64)
    pool.step([2, 0], [60, 17])
    table = pool.block_tables.tolist()
    positions, ctx, done = pool.step([0, 2], [2, 6])
    assert done.tolist() == [1, 0] and b200.device_error(clear=True) == 4
    assert pool.block_tables.tolist() == table and pool.seq_lens.tolist() == [19, 0, 60]
    last = table[2][3] * 16
    assert ctx.slot_mapping.tolist() == [table[0][1] * 16 + 1, table[0][1] * 16 + 2,
                                         last + 12, last + 13, last + 14, last + 15, -1, -1]
    assert positions.tolist() == [17, 18, 60, 61, 62, 63, 64, 65]
