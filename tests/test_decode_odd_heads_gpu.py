"""Decode attention whose split-KV scratch holds an odd number of (head, item)
pairs: odd head counts with an odd item capacity.  The 16-byte vectors of the
partial sums stay aligned whatever the counts are."""
import ctypes

import pytest
import torch

from oracle import layers as L

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (3, 3), (7, 1)])
def test_odd_heads_with_odd_item_capacity(Hq, Hkv):
    from src import b200
    from test_zz_no_alloc import _case, _static_call
    lib = b200.load_library()
    lens = [1500]  # 3 items of 512 keys: capacity 3
    q, kc, vc, bt, cu_q, cu_k = _case(lens, Hq, Hkv, seed=Hq)
    want = L.varlen_attention(q.cpu(), None, None, cu_q.cpu(), cu_k.cpu(), 128 ** -0.5, kc.cpu(), vc.cpu(), bt.cpu())
    n = b200.attention_workspace_bytes(1, 1500, Hq)
    ws = torch.zeros(n, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = lib.b200_paged_attention(p(q), q.stride(0), 1, None, 0, None, 0, p(kc), p(vc), kc.shape[0] * 256, p(bt),
                                  bt.stride(0), bt.shape[1], p(cu_q), p(cu_k), 1, 1, 1500, Hq, Hkv, 256, 128 ** -0.5,
                                  p(out), out.stride(0), p(ws), n, None)
    assert rc == 0, lib.b200_last_error()
    torch.cuda.synchronize()
    assert L.rel_err(out.cpu(), want) <= 1e-2
    static = torch.empty_like(q)
    assert _static_call(q, kc, vc, bt, cu_q, cu_k, 1500, static) == 0
    torch.cuda.synchronize()
    assert torch.equal(static, out)
    assert b200.device_error(clear=True) == 0
