"""Shared-prefix attention over own keys so long that an item is 1024 of them:
2048 own keys a sequence and 512 keys a streaming warp at least.  An item then
lies on up to five pages."""
import pytest
import torch

from test_shared_prefix_gpu import Batch, _clean_error_word, i32  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def long_items(b):
    """Whether the batch's own keys make items of 1024, whatever is shared of the prefixes."""
    warps = 6 * torch.cuda.get_device_properties(0).multi_processor_count
    shared = [b.prefix[g] if g >= 0 else 0 for g in b.group]
    own = sum(n - s for n, s in zip(b.lens, shared))
    return own * b.Hkv >= 512 * warps and own >= 2048 * b.live


@pytest.mark.parametrize("page", [256, 512, 768])
def test_sequences_without_a_prefix(page):
    g = torch.Generator().manual_seed(page)
    lens = torch.randint(2100, 5000, (42,), generator=g).tolist()
    lens[:6] = [2048, 2175, 4096, 4097, 2049, 6143]
    b = Batch(8, 4, [], alone=lens, page=page, seed=page)
    assert long_items(b)
    b.check(b.run())


@pytest.mark.parametrize("page", [256, 512])
def test_own_keys_behind_prefixes(page):
    """The items begin behind a prefix, at the start of a page."""
    g = torch.Generator().manual_seed(page + 1)
    own = torch.randint(2100, 4600, (46,), generator=g).tolist()
    b = Batch(16, 4, [(3 * page, 3 * page, own[:20]), (page, page, own[20:23]), (page + 100, page, own[23:40])],
              alone=own[40:], page=page, seed=page)
    assert long_items(b)
    b.check(b.run())


def test_against_the_same_batch_one_by_one():
    """Long items hold the same keys as the short ones of a sequence alone."""
    from src import b200
    lens = [2500 + 37 * i for i in range(44)]
    b = Batch(8, 4, [], alone=lens, seed=51)
    assert long_items(b)
    out = b.run()
    order = b.lens
    for r in range(0, 44, 7):
        one = b200.shared_prefix_attention(b.q[r:r + 1], b.kc, b.vc, i32([0, 1]), i32([0, order[r]]), order[r], b.scale,
                                           b.table[r:r + 1], i32([-1]), i32([]))
        # both within the bound of the weights' and the result's rounding, |v| at most 6
        assert float((one[0].float() - out[r].float()).abs().max()) <= 4 * 2 ** -8 * 6
    b.check(out, range(0, 44, 7))
