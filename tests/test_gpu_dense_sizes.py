"""Sizes past 32 bits, in views that take no memory: refused before anything is allocated or copied."""
import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import _lib, ops

pytestmark = pytest.mark.gpu
FAR = 2 ** 32 + 5                                 # cut to 32 bits: 5


def refused(call):
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(_lib.OdsdError, match="unsupported sizes"):
        call()
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


def test_linear(dev):
    one = torch.ones(1, 1, dtype=torch.float16, device=dev)
    refused(lambda: ops.linear(one.expand(FAR, 1), one))
    refused(lambda: ops.linear(one.expand(2, FAR // 2 + 1, 1), one))
    refused(lambda: ops.linear(one, one.expand(FAR, 1)))
    refused(lambda: ops.linear(one.expand(1, FAR), one.expand(1, FAR)))
    refused(lambda: ops.linear(one.expand(2 ** 31, 1), one))


def test_rotary(dev):
    one = torch.ones(1, 1, 2, dtype=torch.float16, device=dev)
    f, p = torch.ones(1, dtype=torch.float64, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    cache, slots = torch.zeros(4, 2, dtype=torch.float16, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    far = one.expand(FAR, 1, 2)
    refused(lambda: odsd.apply_rotary(far, far, p.expand(FAR), f))
    refused(lambda: odsd.rotary_store_kvcache(far, far, far, p.expand(FAR), f, cache, cache.clone(), slots.expand(FAR)))
    refused(lambda: odsd.rotary_store_kvcache(one, one, one, p, f, cache, cache.clone(), slots.expand(FAR), src_index=slots.expand(FAR)))
    wide = one.expand(1, FAR, 2)
    refused(lambda: odsd.apply_rotary(wide, one, p, f))
    refused(lambda: odsd.apply_rotary(one, wide, p, f))
    long = one[..., :1].expand(1, 1, FAR)
    refused(lambda: odsd.apply_rotary(long, long, p, f))


def test_verify(dev):
    x, u = torch.zeros(1, 1, device=dev), torch.zeros(1, device=dev)
    d, lens = torch.zeros(1, dtype=torch.int64, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    refused(lambda: odsd.verify_drafts(x.expand(1, FAR), None, {}, None, u))
    refused(lambda: odsd.verify_drafts(x.expand(FAR, 1), None, {}, None, u.expand(FAR)))
    ctx = {"verify_query_lens": lens, "max_query_len": FAR}
    refused(lambda: odsd.verify_drafts(x, None, ctx, None, u))
    ctx["max_query_len"] = 2
    refused(lambda: odsd.verify_drafts(x.expand(FAR, 1), None, ctx, None, u))
    refused(lambda: odsd.verify_drafts(x.expand(FAR, 1), d.expand(FAR - 1), ctx, u.expand(FAR - 1), u))
