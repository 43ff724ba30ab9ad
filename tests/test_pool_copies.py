"""A pool of blocks whose copies are refused: the books stay as they were."""
import pytest
import torch

import on_device_sd_amd as odsd


def _books(pool, *seqs):
    return list(pool.holders), list(pool._free), [(list(s.block_table), s.num_tokens) for s in seqs]


def test_append_whose_copy_is_refused_changes_nothing():
    cache = torch.zeros(6, 4, 8)                     # (not on a GPU: copy_cache_blocks refuses it)
    pool = odsd.BlockPool(6, 4, [cache])
    a, c = odsd.SequenceSlots(4), odsd.SequenceSlots(4)
    pool.append([a, c], [6, 4])
    b = pool.fork(a)
    before = _books(pool, a, b, c)
    with pytest.raises(RuntimeError, match="GPU only"):
        pool.append([c, b, a], [3, 3, 1])            # b gets a copy of the last block, and with c new ones
    assert _books(pool, a, b, c) == before
    with pytest.raises(RuntimeError, match="GPU only"):                # the same call again is refused again
        pool.append([c, b, a], [3, 3, 1])
    assert _books(pool, a, b, c) == before
    pool.append([c], [3])                            # a call that copies nothing
    assert c.block_table == [2, 3] and c.num_tokens == 7 and pool.num_free == 2


def test_compact_whose_copies_are_refused_changes_nothing():
    pool = odsd.BlockPool(6, 4, [torch.zeros(6, 4, 8)])
    a, b = odsd.SequenceSlots(4), odsd.SequenceSlots(4)
    pool.append([a, b], [5, 9])
    pool.free(a)
    before = _books(pool, a, b)
    with pytest.raises(RuntimeError, match="GPU only"):
        pool.compact([b])
    assert _books(pool, a, b) == before


def test_blocks_are_taken_in_order():
    pool = odsd.BlockPool(12, 4)
    a, b = odsd.SequenceSlots(4), odsd.SequenceSlots(4)
    pool.append([a, b], [6, 0])
    c, d = pool.fork(a), pool.fork(a)
    pool.append([a, c, d, b], [7, 1, 1, 5])          # (the last to write keeps the block)
    assert [a.block_table, c.block_table, d.block_table, b.block_table] == [[0, 2, 3, 4], [0, 5], [0, 1], [6, 7]]
    assert pool.holders == [3, 1, 1, 1, 1, 1, 1, 1, 0, 0, 0, 0] and pool._free == [11, 10, 9, 8]


def test_caches_that_could_not_be_copied_are_refused():
    c8 = lambda k=(6, 2, 16, 64), v=(6, 2, 64, 16), s=(6, 2, 2): odsd.KVCacheFP8(*(torch.zeros(t) for t in (k, v, s)))  # noqa: E731
    rows = torch.zeros(6, 4, 8)
    for caches in ([rows.transpose(1, 2)], [rows, torch.zeros(12, 4, 8)[::2]], [c8(v=(5, 2, 64, 16))], [c8(s=(7, 2, 2))], [rows, c8(k=(5, 2, 16, 64))],
                   [rows, torch.zeros((6, 4), device="meta")], [torch.zeros(())]):
        with pytest.raises(ValueError):
            odsd.BlockPool(6, 16, caches)
    for caches, dim in (([rows], 0), ([c8(), rows], 0), ([torch.zeros(3, 6, 4)], 1), ([], 0)):
        assert odsd.BlockPool(6, 16, caches, dim).num_free == 6
    for dim in (2, -1):
        with pytest.raises(ValueError):
            odsd.BlockPool(6, 16, [torch.zeros(6, 6, 6)], dim)
