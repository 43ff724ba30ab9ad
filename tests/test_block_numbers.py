"""The lists of block numbers that copy_cache_blocks takes: what is compared are the numbers, whatever objects hold them."""
import numpy as np
import pytest
import torch

from on_device_sd_amd.blocks import _block_pairs


@pytest.mark.parametrize("as_given", [list, tuple, lambda t: t, lambda t: list(t), lambda t: t.to(torch.int32), lambda t: list(t.numpy()), lambda t: t.tolist(),
                                      lambda t: t.view(-1, 1)])
def test_pairs(as_given):
    given = lambda *v: as_given(torch.tensor(v))  # noqa: E731
    src, dst = _block_pairs(given(3, 0, 3), given(1, 2, 4), False)
    assert list(src) == [3, 0, 3] and list(dst) == [1, 2, 4]
    for s, d, moves in (((3, 0), (1, 1), False), ((3, 1), (1, 2), False), ((2,), (2,), False), ((3, 0), (1,), False), ((3, 3), (1, 2), True)):
        with pytest.raises(ValueError):
            _block_pairs(given(*s), given(*d), moves)
    assert [list(t) for t in _block_pairs([], [], True)] == [[], []]


def test_past_32_bits():
    for n in (1 << 31, 1 << 40, -(1 << 31) - 1):
        for given in ([n], torch.tensor([n]), [torch.tensor(n)]):
            with pytest.raises(ValueError):
                _block_pairs(given, [1], False)
            with pytest.raises(ValueError):
                _block_pairs([1], given, False)


def test_what_is_no_number():
    for bad in ([0.0], [torch.tensor(0.0)], torch.tensor([0.0]), torch.tensor([True]), torch.tensor([1j]), ["0"], [None], [np.float32(0)]):
        with pytest.raises(TypeError):
            _block_pairs(bad, [1], False)
        with pytest.raises(TypeError):
            _block_pairs([1], bad, False)
