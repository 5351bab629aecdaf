"""Shared prefixes whose scores are finite but huge: keys masked by the lowest
value of the type, and keys that differ by less than a step of their score.
A maximum that is rounded must not lie below the score that it came from by
so much that an exponential overflows."""
import pytest
import torch

from test_shared_prefix_gpu import Batch, _clean_error_word  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.bfloat16).min
Q0 = [1.0, 0.9, 0.75, 0.55, 1.25, 0.3, 2 ** -10, 0.61]


def batch(seed):
    """One group of 12 behind 512 keys; the first column of the queries is positive and
    differs, so that scores round both up and down."""
    b = Batch(8, 2, [(512, 512, [40, 300, 1, 700, 90, 5, 60, 130, 2, 33, 257, 8])], seed=seed)
    b.q[..., 0] = (torch.tensor(Q0) * 1.0)[None, :].to(b.q)
    for r in range(b.B):
        b.q[r, :, 0] *= 1 + r / 16
    return b


def masked(b, pages, upto):
    for p in pages:
        n = min(max(upto, 0), 256)
        b.kc[b.table[0, p].long(), :n] = 0
        b.kc[b.table[0, p].long(), :n, :, 0] = LOWEST
        upto -= 256


@pytest.mark.parametrize("n", [1, 128, 200, 256, 384, 512])
def test_a_prefix_that_begins_with_masked_keys(n):
    b = batch(n)
    masked(b, (0, 1), n)
    out = b.run()
    assert bool(torch.isfinite(out).all())
    b.check(out)


def test_every_key_masked():
    """All scores alike: the mean of the values."""
    b = batch(3)
    b.kc.zero_()
    b.kc[..., 0] = LOWEST
    out = b.run()
    assert bool(torch.isfinite(out).all())
    b.check(out)


@pytest.mark.parametrize("size", [40.0, 1e3, 1e5, 1e7, 1e12, 1e17])
def test_ties_of_huge_scores(size):
    """Three different scores far from each other: the values of the highest are averaged, in
    prefixes and own keys alike (their products are exact in fp32, so that ties stay ties)."""
    b = batch(5)
    g = torch.Generator().manual_seed(5)
    b.q[..., 1:] = 0
    b.q[..., 0] *= size
    pick = torch.randint(0, 3, b.kc.shape[:3], generator=g).to(b.kc.device)
    b.kc.zero_()
    b.kc[..., 0] = torch.tensor([-size, size / 2, size], dtype=b.kc.dtype, device=b.kc.device)[pick]
    out = b.run()
    assert bool(torch.isfinite(out).all())
    table = b.table.tolist()
    for r in range(b.live):
        n = b.lens[r]
        k, v = (c[table[r][:-(-n // 256)]].flatten(0, 1)[:n].double().repeat_interleave(4, 1) for c in (b.kc, b.vc))
        w = torch.softmax(torch.einsum("hd,nhd->hn", b.q[r].double(), k) * b.scale, -1)
        want, mass = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w, v.abs())
        # P and the result rounded to bf16; a tie's scores may differ by what a fused difference keeps of a
        # maximum of 4096 at most, 2^-12
        tol = 2 ** -8 * (mass + want.abs()) + (2 ** -12 + 2 ** -13) * mass
        assert bool(((out[r].double() - want).abs() <= tol).all()), r
