"""copy_cache_blocks where it is refused: nothing names a block that was not copied."""
import pytest
import torch

import on_device_sd_amd as odsd

pytestmark = pytest.mark.gpu


def test_tables_follow_the_last_launch(dev):
    """17 tensors are two launches; the second is refused (a block of more than 2^30 bytes), and the tables still name the old block"""
    small = [torch.zeros(2, 16 + i, dtype=torch.uint8, device=dev) for i in range(16)]
    tables = torch.tensor([1, -1, 0], dtype=torch.int32, device=dev)
    large = torch.empty(2, (1 << 30) + 16, dtype=torch.uint8, device=dev)
    with pytest.raises(odsd._lib.OdsdError):
        odsd.copy_cache_blocks(small + [large], [1], [0], 0, tables)
    assert tables.tolist() == [1, -1, 0]
    pool = odsd.BlockPool(2, 16, small + [large])
    gone, seq = odsd.SequenceSlots(16), odsd.SequenceSlots(16)
    pool.append([gone, seq], [16, 16])
    pool.free(gone)
    with pytest.raises(odsd._lib.OdsdError):
        pool.compact([seq], tables)
    assert tables.tolist() == [1, -1, 0] and seq.block_table == [1] and pool.holders == [0, 1]
    for i, t in enumerate(small):
        t.random_(0, 256)
    was = [t[1].clone() for t in small]
    odsd.copy_cache_blocks(small + [torch.zeros(2, 3, dtype=torch.uint8, device=dev)], [1], [0], 0, tables)
    assert tables.tolist() == [0, -1, 0] and all(torch.equal(t[0], w) and torch.equal(t[1], w) for t, w in zip(small, was))


def test_numbers_in_tensors_of_their_own(dev):
    """two tensors that hold the same number name the same block"""
    c = torch.arange(6 * 8, dtype=torch.float32, device=dev).view(6, 8)
    before, one = c.clone(), lambda *v: list(torch.tensor(v))  # noqa: E731
    tables = torch.arange(6, dtype=torch.int32, device=dev)
    for src, dst, t in ((one(3, 4), one(1, 1), None), (one(3, 1), one(1, 2), None), (one(2), one(2), None), (one(3, 3), one(1, 2), tables)):
        with pytest.raises(ValueError):
            odsd.copy_cache_blocks([c], src, dst, 0, t)
    assert torch.equal(c, before) and tables.tolist() == [0, 1, 2, 3, 4, 5]
    odsd.copy_cache_blocks([c], one(3, 4), one(1, 2))
    assert torch.equal(c[1:3], before[3:5])
