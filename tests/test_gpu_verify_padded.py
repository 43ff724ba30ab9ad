"""verify_drafts on padded batches: as many rows of logits and random numbers as the batch has places, lengths on the device that
say which of them are taken."""
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import dense_oracle as orc

pytestmark = pytest.mark.gpu


def expected(x, lens, u, t):
    return orc.verify(x.double().cpu().numpy(), None, lens, None, u.cpu().numpy(), None, t, 1)[0][:, 0].tolist()


@pytest.mark.parametrize("V", [5, 700, 70000])
@pytest.mark.parametrize("lens", [[1, 0, 1, 1, 0], [0, 0, 1], [1, 1, 1, 0], [0] * 70 + [1] * 3 + [0] * 300 + [1], [0, 0], [1, 1]])
@pytest.mark.parametrize("t", [0.8, 0.0])
def test_decode_batch_with_free_places(dev, lens, V, t):
    """a place of length 0 draws nothing and takes no row: the rows follow each other, those behind the last are nobody's"""
    n = len(lens)
    g = torch.Generator(device=dev).manual_seed(n + V)
    x = torch.randn(n, V, generator=g, device=dev) * 3
    x[sum(lens):] = float("nan")
    u = torch.rand(n, generator=g, device=dev)
    ctx = {"verify_query_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": 1}
    want = expected(x, lens, u, float(torch.tensor(t)))
    assert want.count(-1) == lens.count(0)
    for temperature in (t, torch.full((n,), t, device=dev)):
        r = odsd.verify_drafts(x, None, ctx, None, u, temperature=temperature)
        assert r.tokens[:, 0].tolist() == want and r.num_accepted.tolist() == [0] * n


def test_places_change_between_replays(dev):
    n, V = 6, 3000
    g = torch.Generator(device=dev).manual_seed(1)
    x, u = torch.randn(n, V, generator=g, device=dev), torch.rand(n, generator=g, device=dev)
    lens = torch.ones(n, dtype=torch.int32, device=dev)
    ctx = {"verify_query_lens": lens, "max_query_len": 1}
    odsd.verify_drafts(x, None, ctx, None, u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = odsd.verify_drafts(x, None, ctx, None, u)
    for now in ([1] * 6, [1, 0, 1, 0, 1, 0], [0, 1, 1, 1, 1, 0], [0] * 6, [1] * 6):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        x.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        assert out.tokens[:, 0].tolist() == expected(x, now, u, 1.0) == odsd.verify_drafts(x, None, ctx, None, u).tokens[:, 0].tolist(), now
