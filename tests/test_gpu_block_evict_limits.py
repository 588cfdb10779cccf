"""Evictions of sequences that their rows of the page table cannot hold."""
import pytest
import torch

from test_gpu_block_evict import B, dev

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("length", [129, 130, 144, 200, 1 << 20, 2 ** 31 - 1])
def test_longer_than_its_row_of_the_table(length):
    """Two pages of 64: the sequence beside it goes back, this one is left as it is, and the error word says so."""
    b = B()
    g = torch.Generator(device=DEV).manual_seed(length)
    k, v = (torch.randint(-127, 128, (2, 9, 1, 64, 16), generator=g, device=DEV).to(torch.int8) for _ in range(2))
    ks, vs, w = (torch.rand((2, 9, 1, 4), generator=g, device=DEV) for _ in range(3))
    before = [t.clone() for t in (k, v, ks, vs, w)]
    kept, shift = torch.full((2, 2, 1, 3), -7, dtype=torch.int32, device=DEV), dev([100, 200])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    b.block_evict(k, v, ks, vs, w, dev([[0, 1], [2, 3]]), dev([length, 128]), dev([[4], [5]]), 3, 1, kept, err, b.stream_ptr(), shift=shift)
    assert err.item() == b.ERR_PAGE_RANGE
    assert shift.tolist() == [100, 200 + 5 * 16]
    assert (kept[:, 0] == -1).all() and (kept[:, 1, 0, 2] == 7).all() and (kept[:, 1] >= 0).all()
    for now, was in zip((k, v, ks, vs, w), before):
        for page in (0, 1, 2, 3, 4, 6, 7, 8):
            assert torch.equal(now[:, page], was[:, page]), page


def test_exactly_its_row_of_the_table():
    b = B()
    k, v = (torch.zeros((1, 4, 1, 64, 16), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs, w = (torch.ones((1, 4, 1, 4), device=DEV) for _ in range(3))
    kept, shift, err = torch.zeros((1, 1, 1, 3), dtype=torch.int32, device=DEV), dev([0]), torch.zeros(1, dtype=torch.int32, device=DEV)
    b.block_evict(k, v, ks, vs, w, dev([[0, 1]]), dev([128]), dev([[2]]), 3, 1, kept, err, b.stream_ptr(), shift=shift)
    assert err.item() == 0 and kept.flatten().tolist() == [0, 1, 7] and shift.tolist() == [80]
