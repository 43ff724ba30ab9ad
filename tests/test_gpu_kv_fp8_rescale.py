"""store_kvcache_fp8 where a scale rises so far that the quotient of the scales is below fp32's numbers: the codes of the rows that stay
become zeros, and a NaN among them stays NaN."""
import pytest
import torch

from tests.test_gpu_kv_fp8 import check, filled, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H, D, bs, first, n", [(2, 128, 64, 5, 3), (1, 64, 16, 1, 15), (2, 128, 64, 1, 40), (1, 64, 512, 7, 300), (4, 64, 32, 31, 1)])
@pytest.mark.parametrize("old, gain", [(-64, 1e37), (-64, 2.0 ** 80), (-30, 1e37), (-64, 1e25), (-64, 1e19), (-9, 1e3)])
def test_rows_that_stay(dev, H, D, bs, first, n, old, gain):
    cache = filled(dev, 3, H, bs, D, 7)
    for codes in (cache.k, cache.v):               # no number in some places, of both signs
        codes.view(torch.uint8).view(3, H, -1)[..., ::37] = 0x7f
        codes.view(torch.uint8).view(3, H, -1)[..., 5::41] = 0xff
    cache.scales.fill_(2.0 ** old)
    slots = torch.arange(bs + first, bs + first + n, dtype=torch.int32, device=dev)
    check(cache, *rows(dev, n, H, D, torch.bfloat16, 3, gain), slots)
    stayed = torch.ones(bs, dtype=torch.bool, device=dev)
    stayed[first:first + n] = False
    for codes in (cache.k[1], cache.v[1].transpose(1, 2)):
        assert bool(torch.isnan(codes.float())[:, stayed].any())


@pytest.mark.parametrize("gain", [1e37, 1.0])
def test_a_block_that_held_nothing(dev, gain):
    """scale 0: whatever bytes are there, NaN among them, count for nothing"""
    cache = filled(dev, 3, 2, 64, 128, 8)
    cache.scales.zero_()
    check(cache, *rows(dev, 4, 2, 128, torch.bfloat16, 3, gain), torch.arange(70, 74, dtype=torch.int32, device=dev))
    assert not torch.isnan(cache.k[1].float()).any() and not torch.isnan(cache.v[1].float()).any()
