"""verify_drafts where the cumulative weights have borders that a random number can hit: rows whose logits are all equal (or
masked).  Every token left has the weight 1, so the sums are whole numbers, u times their total is exact for u of few bits, and
the token is the definition's, to the one: the lowest whose inclusive sum exceeds u times the total, number floor(u count)."""
import pytest
import torch

import on_device_sd_amd as odsd

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TEMPERATURES = [0.8, 0.3, 1.0, 1.7, 0.05]


def equal_rows(n, V, dtype, seed):
    """rows of one logit each (the first 12.175728), and those logits"""
    g = torch.Generator().manual_seed(seed)
    level = torch.randn(n, generator=g) * 8
    level[0] = 12.175728
    return level[:, None].expand(n, V).to(DT[dtype]).contiguous(), g


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,masked", [(40, 0), (64, 24), (1000, 0), (9000, 808), (131072, 0), (131072, 72)])
def test_sampling_of_equal_logits(dev, V, masked, dtype):
    n, left = 64, V - masked
    x, g = equal_rows(n, V, dtype, V + masked)
    free = torch.arange(V)
    if masked:
        at = torch.randperm(V, generator=g)[:masked]
        x[:, at] = -float("inf")
        free = torch.tensor(sorted(set(range(V)) - set(at.tolist())))
    u = torch.arange(n) / n                                   # 0.25 of 40 is 10: token 10, not 9
    want = [free[(i * left) // n].item() for i in range(n)]
    for t in TEMPERATURES:
        r = odsd.verify_drafts(x.to(dev), None, {}, None, u.to(dev), temperature=t)
        assert r.tokens[:, 0].tolist() == want, t


@pytest.mark.parametrize("V", [41, 513, 4097, 131073])
def test_certain_drafts_on_equal_logits(dev, V):
    """Drafts without logits: a refused one leaves the other V - 1 tokens; the row behind a kept one has all of them (two
    masked: V - 1 again a count that u divides)."""
    n = 64
    x, g = equal_rows(2 * n, V, "fp32", V)
    x[1::2, 7] = -float("inf")
    drafts = torch.randint(0, V, (n,), generator=g)
    drafts[drafts == 7] = 8
    kept = torch.arange(n) % 2 == 0
    u = torch.arange(n) / n
    ctx = {"verify_query_lens": torch.full((n,), 2, dtype=torch.int32, device=dev), "max_query_len": 2}
    number = [(i * (V - 1)) // n for i in range(n)]
    want = [[drafts[i].item(), number[i] + (number[i] >= 7)] if kept[i] else [number[i] + (number[i] >= drafts[i].item()), -1] for i in range(n)]
    for t in TEMPERATURES:
        r = odsd.verify_drafts(x.to(dev), drafts.to(dev), ctx, torch.where(kept, 0.0, 0.999).to(dev), u.to(dev), temperature=t)
        assert r.tokens.tolist() == want, t


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("half", [32, 4096, 65536])
def test_refused_drafts_of_uniform_models(dev, half, dtype):
    """p uniform over 2 half tokens, q over the first half of them: a draft has p / q = 1/2, and p - q is 1 / (2 half) on the
    second half, powers of two all of them."""
    n = 64
    x, g = equal_rows(2 * n, 2 * half, dtype, half)
    q, _ = equal_rows(n, 2 * half, dtype, half + 1)
    q[:, half:] = -float("inf")
    drafts = torch.randint(0, half, (n,), generator=g)
    kept = torch.arange(n) % 4 == 0
    u = torch.arange(n) / n
    ctx = {"verify_query_lens": torch.full((n,), 2, dtype=torch.int32, device=dev), "max_query_len": 2}
    want = [[drafts[i].item(), (i * 2 * half) // n] if kept[i] else [half + (i * half) // n, -1] for i in range(n)]
    for t in TEMPERATURES:
        r = odsd.verify_drafts(x.to(dev), drafts.to(dev), ctx, torch.where(kept, 0.25, 0.75).to(dev), u.to(dev), draft_logits=q.to(dev), temperature=t)
        assert r.tokens.tolist() == want, t
