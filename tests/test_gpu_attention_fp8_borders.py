"""paged_attention_fp8 at the borders of what it holds: scales of V that are 2^80 apart, and workgroups of the merge that have
one row less than the others (sizes and bounds as in test_gpu_attention_fp8)."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from tests.test_gpu_attention_fp8 import bound, check, expected, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L", [300, 9000])
@pytest.mark.parametrize("heads, q_len", [(4, 1), (14, 3), (16, 9)])
@pytest.mark.parametrize("dtype, low, high", [(torch.bfloat16, -60, 20), (torch.float16, -64, 4)])
def test_scales_of_v_far_apart(dev, L, heads, q_len, dtype, low, high):
    """what a block with a small scale weighs is not lost from the sum of the weights"""
    H, D = 2, 64
    cache, tables = make(dev, H, D, 16, [L, 40], 5)
    g = torch.Generator(device=dev).manual_seed(1)
    cache.scales[..., 1] = torch.exp2(torch.randint(low, high + 1, cache.scales[..., 1].shape, generator=g, device=dev).float())
    # one block has the largest scale, one that few rows attend much; a far larger weight is where the smallest is
    cache.scales[int(tables[0, 3]), :, 1], cache.scales[int(tables[0, 7]), :, 1] = 2.0 ** high, 2.0 ** low
    q = torch.randn(q_len + 1, heads, D, generator=g, device=dev).to(dtype)
    lens, q_lens = [L, 40], [q_len, 1]
    ctx = {"block_tables": tables, "context_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": q_len,
           "verify_query_lens": torch.tensor(q_lens, dtype=torch.int32, device=dev)}
    for scale in (0.125, 2.0):
        got = odsd.paged_attention_fp8(q, cache, ctx, scale).double().cpu().numpy()
        want, mag, top = expected(q, cache, tables, lens, q_lens, scale)
        assert (np.abs(got - want) <= bound(want, mag, top, dtype, D, L)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, H, q_len", [(1, 1, 1), (7, 1, 1), (5, 1, 3), (10, 2, 5), (9, 1, 7), (3, 3, 43)])
@pytest.mark.parametrize("L", [4500, 30001])
def test_rows_that_are_merged(dev, dtype, heads, H, q_len, L):
    """heads of 64: two rows to a workgroup of the merge, and an odd number of rows in a unit"""
    check(dev, heads, H, 64, 64, [L, 40], [q_len, min(q_len, 3)], dtype, context_more={"max_query_len": q_len})


@pytest.mark.parametrize("heads, q_len", [(4, 1), (14, 3), (16, 9), (16, 17)])
@pytest.mark.parametrize("softmax_scale, exponent", [(1e-30, -64), (1e-44, -64), (1e-44, 3), (3e38, -64), (3e4, 119)])
def test_scales_whose_product_fp32_does_not_hold(dev, heads, q_len, softmax_scale, exponent):
    """keys behind a row's last one stay out of it, and a score of 0 is 0, when the scale of K times the softmax scale underflows or overflows"""
    H, D, L = 2, 64, 300
    cache, tables = make(dev, H, D, 16, [L, 40], 5)
    cache.scales[..., 0] = 2.0 ** exponent
    q = torch.randn(q_len + 1, heads, D, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    if softmax_scale > 1:
        q.zero_()
    lens, q_lens = [L, 40], [q_len, 1]
    ctx = {"block_tables": tables, "context_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": q_len,
           "verify_query_lens": torch.tensor(q_lens, dtype=torch.int32, device=dev)}
    got = odsd.paged_attention_fp8(q, cache, ctx, softmax_scale).double().cpu().numpy()
    want, mag, top = expected(q, cache, tables, lens, q_lens, softmax_scale)
    assert (np.abs(got - want) <= bound(want, mag, top, torch.bfloat16, D, L)).all()
