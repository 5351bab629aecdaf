"""Calls from a host thread that has not used the GPU before."""
import threading

import pytest
import torch

from test_shared_prefix_gpu import Batch, i32

pytestmark = pytest.mark.gpu


def in_fresh_thread(call):
    got = []

    def body():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001
            got.append(e)
    t = threading.Thread(target=body)
    t.start()
    t.join()
    torch.cuda.synchronize()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


def test_attention_is_the_first_call_of_a_thread():
    from src import b200
    b = Batch(8, 2, [(512, 512, [100, 7])], alone=[50])
    kw = dict(group=i32(b.group), prefix=i32(b.prefix), out=torch.zeros_like(b.q))
    want = b.run(**kw).clone()
    kw["out"].zero_()
    assert torch.equal(in_fresh_thread(lambda: b.run(**kw)), want)
    out = torch.zeros_like(b.q)
    args = (b.q, None, None, b.kc, b.vc, b.cu_q, b.cu_k, 1, b.max_k, b.scale, b.table)
    want = b200.paged_attention(*args)
    assert torch.equal(in_fresh_thread(lambda: b200.paged_attention(*args, out=out)), want)


def test_a_matrix_product_is_the_first_call_of_a_thread():
    from src import b200
    x, w = (torch.randn(n, 512, device="cuda").to(torch.bfloat16) for n in (16, 256))
    out = torch.zeros(16, 256, dtype=torch.bfloat16, device="cuda")
    want = b200.linear(x, w)
    assert torch.equal(in_fresh_thread(lambda: b200.linear(x, w, out=out)), want)


def test_launches_of_several_threads_are_all_counted():
    from src import b200
    x = torch.randn(4, 256, device="cuda").to(torch.bfloat16)
    outs = [torch.empty(4, dtype=torch.int64, device="cuda") for _ in range(4)]
    b200.argmax(x)
    torch.cuda.synchronize()
    before = b200.launch_count()
    lib, stream = b200.load_library(), torch.cuda.current_stream().cuda_stream

    def many(out):
        for _ in range(500):
            assert lib.b200_argmax(x.data_ptr(), x.stride(0), 4, 256, out.data_ptr(), stream) == 0
    threads = [threading.Thread(target=many, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert b200.launch_count() - before == 2000
    assert all(torch.equal(o, x.float().argmax(-1)) for o in outs)
