"""Decode attention with shared prefixes against softmax attention in 64 bits.

Bound of an element, from the roundings on its way: P is rounded to bf16
before the PV product (half a step, 2^-8 of each weight), the result once more
(2^-8 of it); the scores are fp32 sums of 128 products (each within 2^-24 of
the running sum, at most 2^-17 of sum |q k|, which shifts numerator and
denominator), the sums over keys and the exponentials are fp32 (2^-13 covers
10k keys added in tiles).  With w the exact weights:
  |out - exact| <= 2^-8 (sum w |v| + |exact|) + (2^-13 + 2^-15 max sum |q k| scale) sum w |v|
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(autouse=True, params=["", "always"])
def _clean_error_word(request, monkeypatch):
    """Every case twice: with the library's choice of the groups for which
    sharing pays, and with every group of two or more sharing."""
    from src import b200
    monkeypatch.setenv("B200_SHARED_PREFIX", request.param)
    b200.device_error(clear=True)
    yield
    assert b200.device_error(clear=True) == 0, "device error word set"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Batch:
    """groups: (keys given as prefix_len, keys really shared in pages, own lengths behind them);
    alone: lengths of sequences in no group; the order of the batch is shuffled."""

    def __init__(self, Hq, Hkv, groups, alone=(), page=256, seed=0, pad=0, grow=0.0, spare=3, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        seqs, n_pages = [], 0
        self.prefix = []
        for i, (given, shared, owns) in enumerate(groups):
            head = list(range(n_pages, n_pages + shared // page))
            n_pages += len(head)
            self.prefix.append(given)
            for own in owns:
                need = -(-(shared + own) // page) - len(head)
                seqs.append((i, shared + own, head + list(range(n_pages, n_pages + need))))
                n_pages += need
        for n in alone:
            need = -(-n // page)
            seqs.append((-1, n, list(range(n_pages, n_pages + need))))
            n_pages += need
        total = n_pages + spare
        perm = torch.randperm(total, generator=g).tolist()
        seqs = [seqs[i] for i in torch.randperm(len(seqs), generator=g).tolist()]
        self.B, self.Hq, self.Hkv, self.page = len(seqs) + pad, Hq, Hkv, page
        self.group = [s[0] for s in seqs] + [0 if groups else -1] * pad
        self.lens = [s[1] for s in seqs] + [0] * pad
        self.live = len(seqs)
        width = max([len(s[2]) for s in seqs] + [1])
        table = torch.full((self.B, width), -1, dtype=torch.int32)
        kc = torch.full((total, page, Hkv, 128), float("nan"), dtype=BF)
        vc = kc.clone()
        for b, (_, n, pages) in enumerate(seqs):
            for j, p in enumerate(pages):
                table[b, j] = perm[p]
                m = min(page, n - j * page)
                if torch.isnan(kc[perm[p], 0, 0, 0]) or torch.isnan(kc[perm[p], m - 1, 0, 0]):
                    # (later keys larger by `grow` a key: row maxima that keep growing)
                    at = 1 + grow * (torch.arange(m) + j * page)[:, None, None]
                    kc[perm[p], :m] = (torch.randn(m, Hkv, 128, generator=g) * at).to(BF)
                    vc[perm[p], :m] = torch.randn(m, Hkv, 128, generator=g).to(BF)
        self.q = (torch.randn(self.B, Hq, 128, generator=g) * q_scale).to(BF).to(DEV)
        self.table, self.kc, self.vc = table.to(DEV), kc.to(DEV), vc.to(DEV)
        self.cu_q = i32(list(range(self.live + 1)) + [self.live] * pad)
        cu = [0]
        for n in self.lens:
            cu.append(cu[-1] + n)
        self.cu_k = i32(cu)
        self.max_k = max(self.lens + [1])
        self.scale = 128 ** -0.5

    def run(self, **kw):
        from src import b200
        return b200.shared_prefix_attention(kw.pop("q", self.q), self.kc, self.vc, self.cu_q, self.cu_k,
                                            kw.pop("max_k", self.max_k), self.scale, self.table,
                                            kw.pop("group", None) if "group" in kw else i32(self.group),
                                            kw.pop("prefix", None) if "prefix" in kw else i32(self.prefix), **kw)

    def check(self, out, rows=None):
        table = self.table.tolist()
        for b in rows if rows is not None else range(self.live):
            n = self.lens[b]
            if n == 0:
                assert torch.count_nonzero(out[b]) == 0
                continue
            pages = table[b][:-(-n // self.page)]
            G = self.Hq // self.Hkv
            k = self.kc[pages].flatten(0, 1)[:n].double().repeat_interleave(G, 1)
            v = self.vc[pages].flatten(0, 1)[:n].double().repeat_interleave(G, 1)
            q = self.q[b].double()
            w = torch.softmax(torch.einsum("hd,nhd->hn", q, k) * self.scale, -1)
            want = torch.einsum("hn,nhd->hd", w, v)
            mass = torch.einsum("hn,nhd->hd", w, v.abs())
            qk = (torch.einsum("hd,nhd->hn", q.abs(), k.abs()) * self.scale).amax(-1, keepdim=True)
            tol = 2 ** -8 * (mass + want.abs()) + (2 ** -13 + 2 ** -15 * qk) * mass
            off = (out[b].double() - want).abs()
            assert bool((off <= tol).all()), (b, n, self.group[b], float((off / tol).max()))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (3, 1), (5, 1), (6, 2), (7, 1), (8, 1), (16, 8), (32, 8), (40, 8),
                                    (64, 8), (4, 4)])
def test_heads(Hq, Hkv):
    """Every number of query heads to a kv head; groups of two up to more than one row block."""
    b = Batch(Hq, Hkv, [(512, 512, [1, 300, 77]), (256, 256, [5] * (300 // (Hq // Hkv) // 2)),
                        (1536, 1536, [700, 2])], alone=[1, 257, 900], seed=Hq)
    b.check(b.run())


@pytest.mark.parametrize("page", [256, 512, 768])
@pytest.mark.parametrize("members", [2, 31, 64, 65, 129, 200])
def test_members_and_pages(members, page):
    g = torch.Generator().manual_seed(members)
    own = torch.randint(0, 2 * page, (members,), generator=g).tolist()
    b = Batch(8, 2, [(5 * page, 5 * page, own)], alone=[3], page=page, seed=members)
    b.check(b.run())


CASES = {
    # prefix_len inside a page: only the whole pages before it count
    "ragged prefix_len": [(700, 512, [200, 300]), (255, 256, [9, 10]), (513, 512, [1, 1])],
    # members that end inside the prefix, or with it: what all of them see counts
    "short members": [(1024, 1024, [0, 0, 5]), (1024, 512, [0, 100, 511]), (2048, 256, [0, 1])],
    "one member": [(512, 512, [40]), (256, 256, [1])],
    "nothing shared": [(0, 0, [1, 600]), (-5, 0, [20, 30])],
    "many groups": [(256 * (1 + i % 3), 256 * (1 + i % 3), [1 + 13 * i, 2, 3][:2 + i % 2]) for i in range(40)],
}


@pytest.mark.parametrize("name", list(CASES))
def test_groups(name):
    b = Batch(10, 2, CASES[name], alone=[255, 256, 257], seed=3)
    b.check(b.run())


def test_no_groups_and_no_sequences():
    b = Batch(8, 2, [], alone=[1, 256, 700, 4000])
    b.check(b.run())
    from src import b200
    none = b200.shared_prefix_attention(b.q[:0], b.kc, b.vc, i32([0]), i32([0]), 1, 0.1, b.table[:0], i32([]), i32([]))
    assert none.shape == (0, 8, 128)


@pytest.mark.parametrize("grow,q_scale", [(0.0, 8.0), (0.01, 4.0), (0.1, 1.0)])
def test_growing_and_peaked_scores(grow, q_scale):
    """Scores in the hundreds whose maximum keeps growing along the keys (the
    accumulators are rescaled again and again), and nearly one-hot weights."""
    b = Batch(16, 2, [(1024, 1024, [300, 0, 20, 513, 7]), (512, 512, [1, 1])], alone=[1500], grow=grow, q_scale=q_scale)
    b.check(b.run())


def test_infinite_values_in_keys():
    """Keys of -inf score (a column of K at the lowest values) weigh nothing; a
    sequence whose own keys all do so keeps its prefix."""
    b = Batch(4, 1, [(512, 512, [130, 40, 300])], seed=9)
    b.q[..., 0] = 1.0
    b.kc[b.table[0, 0].long(), :200, :, 0] = -float("inf")
    b.kc[b.table[1, 2].long(), :40, :, 0] = -float("inf")
    b.kc[b.table[0, 1].long(), 17, :, 0] = torch.finfo(BF).min
    out = b.run()
    assert bool(torch.isfinite(out).all())
    table = b.table.tolist()
    for r in range(b.live):
        n = b.lens[r]
        k = b.kc[table[r][:-(-n // 256)]].flatten(0, 1)[:n].double()
        v = b.vc[table[r][:-(-n // 256)]].flatten(0, 1)[:n].double()
        w = torch.softmax(torch.einsum("hd,nd->hn", b.q[r].double(), k[:, 0]) * b.scale, -1)
        want, mass = w @ v[:, 0], w @ v[:, 0].abs()
        assert bool(((out[r].double() - want).abs() <= 2 ** -8 * (mass + want.abs()) + 2 ** -10 * mass).all())


def test_nan_reaches_only_its_sequences():
    b = Batch(4, 1, [(256, 256, [10, 20]), (512, 512, [30, 40])], seed=11)
    first = [r for r in range(b.live) if b.group[r] == 0]
    b.vc[b.table[first[0], 0].long(), 3, 0, 5] = float("nan")
    out = b.run()
    for r in range(b.live):
        bad = torch.isnan(out[r]).any(0)
        assert bad.nonzero()[:, 0].tolist() == ([5] if r in first else [])
    b.check(out, [r for r in range(b.live) if r not in first])


def test_padding_rows_are_left_alone_and_empty_rows_are_zero():
    b = Batch(8, 2, [(256, 256, [3, 4, 5])], alone=[0, 9], pad=4)
    out = torch.full_like(b.q, 7.0)
    b.run(out=out)
    b.check(out)
    assert bool((out[b.live:] == 7.0).all())


def test_strided_q_and_out():
    """q as the head of a fused projection's rows, out as a slice of wider ones."""
    b = Batch(6, 2, [(512, 512, [3, 400, 5])], alone=[90])
    wide = torch.zeros(b.B, 6 + 2 + 2, 128, dtype=BF, device=DEV)
    wide[:, :6] = b.q
    into = torch.zeros(b.B, 8, 128, dtype=BF, device=DEV)
    b.run(q=wide[:, :6], out=into[:, 1:7])
    b.check(into[:, 1:7])
    assert torch.count_nonzero(into[:, 0]) == 0 and torch.count_nonzero(into[:, 7]) == 0
    assert torch.equal(b.run(), into[:, 1:7])
    b.check(b.run(q=b.q.transpose(0, 1).contiguous().transpose(0, 1)))


def test_same_bits_every_time():
    b = Batch(32, 8, [(2048, 2048, [i * 7 % 600 for i in range(50)]), (512, 512, [5, 6, 7])], alone=[1000] * 9)
    first = b.run()
    for _ in range(5):
        assert torch.equal(b.run(), first)


def test_captured_graph_with_changing_groups():
    """One captured launch, replayed on batches with other lengths, groups and
    paddings in the same buffers."""
    batches = [Batch(16, 4, [(1024, 1024, [100] * 10), (256, 256, [20, 30, 40])], alone=[700] * 3, seed=1),
               Batch(16, 4, [(512, 512, [1, 2])], alone=[100, 900], pad=12, seed=2),
               Batch(16, 4, [], alone=[300] * 9, pad=7, seed=3),
               Batch(16, 4, [(2048, 2048, [0] * 16)], seed=4)]
    B, width, pages = 16, 10, max(b.kc.shape[0] for b in batches)
    s = Batch(16, 4, [], alone=[1] * B)
    s.kc, s.vc = (torch.zeros(pages, 256, 4, 128, dtype=BF, device=DEV) for _ in range(2))
    s.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    group, prefix = i32([-1] * B), i32([0] * 3)
    out = torch.zeros_like(s.q)
    s.run(group=group, prefix=prefix, max_k=4096, out=out)  # sizes the workspace
    s.table[:] = -1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(group=group, prefix=prefix, max_k=4096, out=out)
    from src import b200
    b200.device_error(clear=True)  # (the warm-up's tables were empty)
    for b in batches + batches[::-1]:
        n = b.kc.shape[0]
        s.kc[:n], s.vc[:n] = b.kc, b.vc
        s.q.copy_(b.q)
        s.table.fill_(-1)
        s.table[:, :b.table.shape[1]] = b.table
        s.cu_q.copy_(b.cu_q)
        s.cu_k.copy_(b.cu_k)
        group.copy_(i32(b.group))
        prefix.zero_()
        if b.prefix:
            prefix[:len(b.prefix)] = i32(b.prefix)
        out.fill_(5.0)
        graph.replay()
        b.check(out)
        assert bool((out[b.live:] == 5.0).all())


def test_long_cache_offsets():
    """Pages behind 2^31 elements of the cache."""
    b = Batch(8, 8, [(512, 512, [100, 200, 3])], alone=[600], seed=5)
    n = b.kc.shape[0]
    kc, vc = (torch.empty(8300, 256, 8, 128, dtype=BF, device=DEV) for _ in range(2))
    kc[-n:], vc[-n:] = b.kc, b.vc
    b.kc, b.vc = kc, vc
    b.table[b.table >= 0] += 8300 - n
    b.check(b.run())


def test_missing_pages_count_for_nothing_and_are_flagged():
    from src import b200
    for at, value in ((1, -1), (0, 1 << 20)):
        b = Batch(8, 2, [(768, 768, [40, 50])], seed=6)
        b.table[:, at] = value
        out = b.run()
        assert b200.device_error(clear=True) == 4
        # the same sequences without that page's keys
        keep = [j for j in range(3) if j != at] + [3]
        b.table = b.table[:, keep].contiguous()
        b.lens = [n - 256 for n in b.lens]
        b.check(out)
    b = Batch(8, 2, [(256, 256, [40, 50])], alone=[30], seed=6)
    b.check(b.run(group=i32([-2 if g < 0 else 1 for g in b.group])))  # groups that are not there
    assert b200.device_error(clear=True) == 4


def test_lengths_past_max_seqlen_k_are_flagged():
    """More own keys than max_seqlen_k allows for: the error word says so, nothing
    is read or written out of place, and the next call is right."""
    from src import b200
    b = Batch(8, 8, [], alone=[1400], seed=2)
    n = 300
    b.table = b.table.expand(n, -1).contiguous()
    b.q = torch.randn(n, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    b.cu_q = i32(list(range(n + 1)))
    b.cu_k = i32([1400 * i for i in range(n + 1)])
    b.B, b.live, b.lens, b.group = n, n, [1400] * n, [-1] * n
    out = torch.full((n + 1, 8, 128), 7.0, dtype=BF, device=DEV)
    b.run(max_k=1, out=out[:n])
    assert b200.device_error(clear=True) == 4
    assert bool((out[n] == 7.0).all())
    b.check(b.run(), range(0, n, 30))


@pytest.mark.parametrize("group", [-1, 0])
def test_rows_outside_q_are_flagged(group):
    """A sequence whose query row lies behind q is left out, the others are answered."""
    from src import b200
    b = Batch(8, 2, [(512, 512, [3, 700, 5, 9])], alone=[300], seed=4)
    b.group[-1] = group
    out = torch.full((b.B, 8, 128), 7.0, dtype=BF, device=DEV)
    b.run(q=b.q[:-1], out=out[:-1], group=i32(b.group))
    assert b200.device_error(clear=True) == 4
    b.check(out, range(b.live - 1))
    assert bool((out[-1] == 7.0).all())


@pytest.mark.parametrize("B,prefix,Hq,Hkv", [(256, 8192, 32, 8), (1024, 1024, 16, 2)])
def test_large_batches(B, prefix, Hq, Hkv):
    g = torch.Generator().manual_seed(B)
    b = Batch(Hq, Hkv, [(prefix, prefix, torch.randint(0, 400, (B,), generator=g).tolist())], seed=B)
    out = b.run()
    b.check(out, range(0, B, B // 32))
    from src import b200
    ref = b200.paged_attention(b.q, None, None, b.kc, b.vc, b.cu_q, b.cu_k, 1, b.max_k, b.scale, b.table)
    # both round P and the result: twice the bound against 64 bits, with |v| at most 6 here
    assert float((out.float() - ref.float()).abs().max()) <= 4 * 2 ** -8 * 6


def test_on_another_stream():
    b = Batch(8, 2, [(512, 512, [100, 200, 3])], alone=[50])
    want = b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = b.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_as_many_groups_as_there_can_be():
    b = Batch(8, 1, [(256, 256, [3, 1 + i % 60]) for i in range(512)], seed=12)
    b.check(b.run(), range(0, b.live, 11))


def test_two_captured_graphs_with_one_workspace():
    """Graphs of different batches replayed in turn: every call leaves the
    workspace as the next one needs it."""
    pair = [Batch(16, 2, [(1024, 1024, [40, 700, 3] * 6)], alone=[1500, 2], seed=13),
            Batch(8, 8, [(512, 512, [90] * 5), (256, 256, [600, 1])], seed=14)]
    outs = [torch.zeros_like(b.q) for b in pair]
    index = [(i32(b.group), i32(b.prefix)) for b in pair]
    for b, out, (g, p) in zip(pair, outs, index):
        b.run(group=g, prefix=p, out=out)
    want = [o.clone() for o in outs]
    graphs = []
    for b, out, (g, p) in zip(pair, outs, index):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            b.run(group=g, prefix=p, out=out)
    for turn in (0, 1, 1, 0, 0, 1):
        outs[turn].zero_()
        graphs[turn].replay()
        assert torch.equal(outs[turn], want[turn])
    for b, out in zip(pair, outs):
        b.check(out)


def test_launches_that_may_overlap(monkeypatch):
    monkeypatch.setenv("B200_PDL", "1")
    b = Batch(8, 2, [(512, 512, [100, 200, 3, 900])], alone=[50], seed=15)
    first = b.run()
    for _ in range(4):
        b.q.mul_(1.0)
        assert torch.equal(b.run(), first)
    b.check(first)


def test_one_query_for_all_sequences():
    """q expanded over the batch (rows that lie on one another), and single rows
    whose strides say nothing."""
    from src import b200
    b = Batch(8, 2, [(512, 512, [3, 400, 5])], seed=16)
    b.q = b.q[:1].expand(b.B, -1, -1)
    b.check(b.run())
    with pytest.raises(ValueError, match="rows apart"):
        b.run(out=torch.zeros(1, 8, 128, dtype=BF, device=DEV).expand(b.B, -1, -1))
    one = Batch(8, 2, [], alone=[700], seed=17)
    want = one.run()
    odd = torch.as_strided(one.q, (1, 8, 128), (3, 128, 1))
    into = torch.as_strided(torch.zeros_like(one.q), (1, 8, 128), (0, 128, 1))
    assert torch.equal(one.run(q=odd, out=into), want)
    assert b200.device_error(clear=True) == 0


def test_two_streams_with_workspaces_of_their_own():
    """Calls on two streams at once through the C entry, each with its own workspace."""
    from src import b200
    lib = b200.load_library()
    pair = [Batch(8, 2, [(1024, 1024, [400, 3, 90] * 5)], alone=[700], seed=18),
            Batch(16, 2, [(512, 512, [40, 1200, 8, 9])], alone=[30] * 9, seed=19)]
    want = [b.run() for b in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    outs, keep = [torch.zeros_like(b.q) for b in pair], []
    torch.cuda.synchronize()
    for turn in range(6):
        for b, st, out in zip(pair, streams, outs):
            if turn == 0:
                n = b200.shared_prefix_workspace_bytes(b.B, b.max_k, b.Hq, b.Hkv)
                keep.append([torch.zeros(n, dtype=torch.uint8, device=DEV), i32(b.group), i32(b.prefix)])
                torch.cuda.synchronize()
            ws, g, p = keep[pair.index(b)]
            rc = lib.b200_shared_prefix_attention(
                b.q.data_ptr(), b.q.stride(0), b.B, b.kc.data_ptr(), b.vc.data_ptr(), b.kc.shape[0] * b.page,
                b.table.data_ptr(), b.table.stride(0), b.table.shape[1], b.cu_q.data_ptr(), b.cu_k.data_ptr(), b.B,
                b.max_k, b.Hq, b.Hkv, b.page, b.scale, g.data_ptr(), p.data_ptr(), p.numel(), out.data_ptr(),
                out.stride(0), ws.data_ptr(), ws.numel(), st.cuda_stream)
            assert rc == 0
    torch.cuda.synchronize()
    for out, w, (ws, _, _) in zip(outs, want, keep):
        assert torch.equal(out, w)
        assert not bool(ws[:256].any())
