"""Sizes of the attention over the 8-bit cache that the library does not hold are refused, not cut."""
import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import _lib

P = 1 << 20


def test_positions_past_the_lists():
    """positions are counted up to 2^30: a wider table was attended up to there only"""
    lib = _lib.load()
    size = lambda bs, mb: lib.odsd_paged_attention_fp8_workspace_bytes(1, 1, 2, 2, 64, bs, mb)  # noqa: E731
    call = lambda bs, mb: lib.odsd_paged_attention_fp8(P, P, P, P, P, P, None, 1, 1, 1, 2, 2, 64, bs, mb, 8, 0.1, 1, P, P, 0, None)  # noqa: E731
    assert size(16, 1 << 26) > 0 and size(1024, 1 << 20) > 0 and call(16, 1 << 26) == call(1024, 1 << 20) == 5
    assert size(16, (1 << 26) + 1) == size(1024, (1 << 20) + 1) == size(1024, (1 << 31) - 1) == 0
    assert call(16, (1 << 26) + 1) == call(1024, (1 << 20) + 1) == call(1024, (1 << 31) - 1) == 3


@pytest.mark.gpu
def test_python_sizes(dev):
    """a bound on the query lengths of more than 31 bits was taken modulo 2^32"""
    cache = odsd.KVCacheFP8.zeros(4, 2, 16, 64, dev)
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    ctx = {"block_tables": i32(0, 1)[:, None], "context_lens": i32(9, 9), "verify_query_lens": i32(3, 2)}
    for most in ((1 << 32) + 1, (1 << 32) + 3, 1 << 31, 1 << 40, -1):
        with pytest.raises(_lib.OdsdError):
            odsd.paged_attention_fp8(q, cache, ctx, None, most)
        with pytest.raises(_lib.OdsdError):
            odsd.paged_attention_fp8(q, cache, {**ctx, "max_query_len": most})
    assert not odsd.paged_attention_fp8(q, cache, ctx, None, 3).any()
