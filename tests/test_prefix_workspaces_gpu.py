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


def in_threads(*loops):
    """The loops at once, each on a host thread of its own; the first exception is raised here."""
    import sys
    import threading
    failed, gate = [], threading.Barrier(len(loops))

    def body(loop):
        try:
            gate.wait(60)
            loop()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    threads = [threading.Thread(target=body, args=(loop,)) for loop in loops]
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    torch.cuda.synchronize()
    if failed:
        raise failed[0]


def test_host_threads_on_one_stream():
    """The launches of a call stay together: with one workspace and one stream,
    calls of two threads would otherwise merge each other's parts."""
    made = batches()
    outs = [[torch.zeros_like(b.q) for _ in range(150)] for b in made]
    torch.cuda.synchronize()
    in_threads(*[lambda b=b, out=out: [b.run(out=o, **b.args) for o in out] for b, out in zip(made, outs)])
    for b, out in zip(made, outs):
        for o in out:
            assert torch.equal(o, b.want)


def test_host_threads_on_the_tables_of_one_pool():
    """Forks, turnovers and compactions of three threads on one stream: in
    whatever order the calls come, the tables hold together and every row has
    its tokens."""
    from src.engine.pages import PagePool
    pages, page = 160, 16
    kv = torch.zeros(2, 2, pages, page, 1, 8, dtype=torch.bfloat16, device=DEV)
    pool = PagePool(kv, 16, 8 * page)
    lens = [100, 37, 64, 5, 128, 81]
    assert pool.take(list(range(6)), lens).tolist() == [1] * 6

    def slots(row, n):
        table = pool.block_tables[row].tolist()
        return [table[i // page] * page + i % page for i in range(n)]

    flat = kv.view(2, 2, pages * page, 8)
    for r, n in enumerate(lens):
        flat[:, :, slots(r, n)] = (torch.arange(n, device=DEV) % 16 + 16 * r).to(kv.dtype)[None, None, :, None]
    rows = {r: i32([r]) for r in range(16)}
    most = i32([7 * page])
    torch.cuda.synchronize()

    def forks():
        for i in range(150):
            pool.free(rows[10])
            pool.fork(rows[i % 6], rows[10])

    def turnovers():
        for _ in range(150):
            pool.free(rows[11])
            pool.take(rows[11], most)

    def compactions():
        for _ in range(150):
            pool.compact()

    in_threads(forks, turnovers, compactions)
    table = pool.block_tables.tolist()
    held = [0] * pages
    for r, entries in enumerate(table):
        n = -(-pool.seq_lens[r].item() // page)
        assert min(entries[:n], default=0) >= 0 and set(entries[n:]) <= {-1}, r
        for e in entries[:n]:
            held[e] += 1
    assert pool.refs.tolist() == held
    assert pool.seq_lens.tolist() == lens + [0] * 4 + [lens[149 % 6], 7 * page] + [0] * 4
    for r, of in [*((r, r) for r in range(6)), (10, 149 % 6)]:
        want = (torch.arange(lens[of], device=DEV) % 16 + 16 * of).to(kv.dtype)
        assert torch.equal(flat[:, :, slots(r, lens[of])], want[None, None, :, None].expand(2, 2, -1, 8)), r
