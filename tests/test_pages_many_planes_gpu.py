"""Compaction of a cache whose pages times planes pass 31 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_compaction_of_2_to_the_32_page_planes():
    from src import b200
    pages, planes = 1 << 22, 1024
    if torch.cuda.mem_get_info()[0] < 72 << 30:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 72 << 30:
        pytest.skip("needs 64 GiB of device memory")
    i32 = dict(dtype=torch.int32, device="cuda")
    kv = torch.empty(2, planes // 2, pages, 1, 1, 16, dtype=torch.uint8, device="cuda")  # slots of 16 bytes
    refs = torch.zeros(pages, **i32)
    table = torch.tensor([[0, pages - 1, 5, -1]], **i32)
    refs[table[0, :3].long()] = 1
    want = torch.randint(0, 255, (2, planes // 2, 3, 16), dtype=torch.uint8, device="cuda")
    for j, p in enumerate(table[0, :3].tolist()):
        kv[:, :, p, 0, 0] = want[:, :, j]
    place = b200.compact_pages(kv, table, refs)
    assert b200.device_error(clear=True) == 0
    assert table.tolist() == [[0, 2, 1, -1]]  # page 5 into the first hole, the last page into the second
    assert place[[0, 5, pages - 1]].tolist() == [0, 1, 2] and int((place >= 0).sum()) == 3
    assert refs[:3].tolist() == [1, 1, 1] and int(refs.sum()) == 3
    for j, p in enumerate(table[0, :3].tolist()):
        assert torch.equal(kv[:, :, p, 0, 0], want[:, :, j])
    del kv
    torch.cuda.empty_cache()
