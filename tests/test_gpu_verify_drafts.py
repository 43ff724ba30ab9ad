"""verify_drafts against the 64-bit definition: kept drafts and drawn tokens exactly, probabilities to what their sums' fp32
statistics allow: each of the two sums of a probability's ratio is off by at most 2^-23 (the hardware's exp2, 1 ulp) + 6 2^-24
(roundings of a sum of 32: 3 along 4 logits, 3 up the tree) + 17 ln 2 2^-24 (a difference of logits rounded to fp32, 17 bits
below the largest, where 131 072 tokens still weigh as much as it), 1.2e-6; the ratio of two 2.4e-6, rounded to fp32 (2^-24)."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import dense_oracle as orc

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
PROB_TOL = 2 * (2.0 ** -23 + 6 * 2.0 ** -24 + 17 * 0.6932 * 2.0 ** -24) + 2.0 ** -24


def make(lens, V, dtype="bf16", seed=0, with_q=True, near=0.7, T=0.8):
    g = torch.Generator().manual_seed(seed)
    n_q, n_d = sum(lens), sum(max(n - 1, 0) for n in lens)
    base = torch.randn(n_q, V, generator=g) * 2
    rows, at = [], 0
    for n in lens:
        rows += list(range(at, at + max(n - 1, 0)))
        at += n
    q = base[rows] + near * torch.randn(n_d, V, generator=g)
    noise = -torch.log(-torch.log(torch.rand(n_d, V, generator=g).clamp(1e-6, 1 - 1e-6)))
    drafts = (q / T + noise).argmax(1) if n_d else torch.zeros(0, dtype=torch.int64)
    return {"logits": base.to(DT[dtype]), "draft_logits": q.to(DT[dtype]) if with_q else None, "drafts": drafts,
            "accept_u": torch.rand(n_d, generator=g), "sample_u": torch.rand(len(lens), generator=g), "lens": lens}


def check(dev, m, temperature=0.8, width=None, logits=None, draft_logits=None):
    """`logits` / `draft_logits`: the device's view of the same values"""
    lens = m["lens"]
    width = width or max(lens)
    t = temperature if isinstance(temperature, float) else torch.tensor(temperature, dtype=torch.float32)
    on = lambda v: None if v is None else v.to(dev)  # noqa: E731
    q = m["draft_logits"]
    r = odsd.verify_drafts(on(m["logits"]) if logits is None else logits, on(m["drafts"]),
                           {"verify_query_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": width}, on(m["accept_u"]),
                           on(m["sample_u"]), draft_logits=draft_logits if draft_logits is not None else on(q),
                           temperature=t if isinstance(t, float) else t.to(dev))
    # (a temperature is an fp32 number, as the kernel gets it)
    tokens, accepted, probs = orc.verify(m["logits"].double().numpy(), m["drafts"].numpy(), lens, m["accept_u"].numpy(), m["sample_u"].numpy(),
                                         None if q is None else q.double().numpy(), np.float32(temperature), width)
    assert np.allclose(r.accept_probs.cpu().double().numpy(), probs, rtol=PROB_TOL, atol=1e-40)
    assert r.num_accepted.cpu().tolist() == accepted.tolist()
    assert r.tokens.cpu().tolist() == tokens.tolist()
    return r


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("lens,V", [([1], 7), ([2], 1), ([5], 1000), ([3, 1, 4, 2], 513), ([9, 2, 9, 5, 1], 8192), ([4, 4], 8193), ([2, 3], 32768),
                                    ([3], 50257), ([6, 3, 1, 2] * 20, 333), ([1] * 70, 257), ([2, 1], 131072), ([70, 1, 2], 64)])
def test_against_the_definition(dev, lens, V, with_q, dtype):
    check(dev, make(lens, V, dtype, seed=V, with_q=with_q))


@pytest.mark.parametrize("with_q", [True, False])
def test_temperatures_of_the_sequences(dev, with_q):
    lens = [5, 3, 1, 4, 2, 6, 3]
    m = make(lens, 3001, "fp16", seed=4, with_q=with_q)
    r = check(dev, m, [0.0, 1.0, 0.0, 0.3, 100.0, 1e-6, 0.0])
    assert (r.num_accepted.cpu() <= torch.tensor(lens) - 1).all()
    check(dev, m, 0.0)
    check(dev, m, 1.7)


def test_greedy_takes_the_lowest_of_equals(dev):
    m = make([3, 2, 1], 20000, "bf16", seed=1)
    m["logits"][:, 150] = m["logits"][:, 19000] = m["logits"][:, 9000] = 30.0
    m["drafts"][:] = torch.tensor([150, 9000, 150])
    r = check(dev, m, 0.0)
    assert r.tokens[0].tolist() == [150, 150, -1] and r.num_accepted.tolist() == [1, 1, 0]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masked_rows(dev, dtype):
    """-inf, NaN and +inf entries, rows that leave one token or none, the type's lowest value as a mask."""
    lens = [3, 2, 4, 2, 2, 2, 3]
    m = make(lens, 9000, dtype, seed=2)
    x, q = m["logits"], m["draft_logits"]
    low = torch.finfo(DT[dtype]).min
    x[:, 1::2] = -float("inf")                       # half of every row
    x[0, 4] = x[1, 4] = float("nan")
    x[3, :] = -float("inf")                          # no token at all
    x[5, :] = float("nan")
    x[6] = -float("inf")
    x[6, 8998] = -3.0                                # one token, in the last block
    x[9, 10] = x[9, 8200] = float("inf")
    x[11, :] = low                                   # all equal: uniform
    x[13, 4500:] = low
    q[2, :] = -float("inf")                          # the draft model's row is empty
    q[4, 7] = float("inf")
    for t in (0.8, 0.0):
        check(dev, m, t)
    m["accept_u"][:] = 0.999999                      # most drafts refused
    check(dev, m)
    m["accept_u"][:] = 0.0
    m["sample_u"][:] = 0.0
    check(dev, m)
    m["sample_u"][:] = 1.0 - 2.0 ** -24
    check(dev, m)


@pytest.mark.parametrize("dtype,bits,raw", [("fp32", 0x7fa00000, torch.int32), ("bf16", 0x7f81, torch.int16), ("fp16", 0x7d01, torch.int16)])
@pytest.mark.parametrize("with_q", [True, False])
def test_signalling_nan_counts_as_nothing(dev, dtype, bits, raw, with_q):
    m = make([3, 2, 1], 2000, dtype, seed=31, with_q=with_q)
    for t in (m["logits"], m["draft_logits"]):
        if t is not None:
            t.view(raw)[:, 5::7] = bits
            assert torch.isnan(t[:, 5::7]).all()
    m["logits"].view(raw)[5, 700:1999] = bits
    for u in (0.3, 0.999999):
        m["accept_u"][:] = u
        check(dev, m)
    check(dev, m, 0.0)


def test_drafts_outside_the_vocabulary_and_equal_models(dev):
    m = make([4, 4, 2], 700, "fp32", seed=3)
    m["drafts"][1], m["drafts"][4], m["drafts"][6] = 700, -1, 2 ** 40
    check(dev, m)
    m = make([6, 6], 700, "fp32", seed=5, near=0.0)       # q is p: every draft is kept
    r = check(dev, m)
    assert r.num_accepted.tolist() == [5, 5]
    for with_q in (True, False):
        m = make([3], 50, "fp32", seed=6, with_q=with_q)
        m["logits"][:] = -20.0
        m["logits"][:, 3] = 20.0
        m["drafts"][:] = 3
        check(dev, m)


def test_empty_sequences_and_wider_tokens(dev):
    m = make([0, 3, 0, 1, 2, 0], 1200, "bf16", seed=8)
    r = check(dev, m, width=5)
    assert r.tokens[0].tolist() == [-1] * 5 and r.tokens[5].tolist() == [-1] * 5


def test_no_rows_at_all(dev):
    none = torch.zeros(0, device=dev)
    ctx = {"verify_query_lens": torch.zeros(2, dtype=torch.int32, device=dev), "max_query_len": 0}
    r = odsd.verify_drafts(torch.zeros(0, 10, device=dev), None, ctx, None, torch.rand(2, device=dev))
    assert r.tokens.shape == (2, 0) and r.num_accepted.tolist() == [0, 0] and r.accept_probs.numel() == 0
    ctx["max_query_len"] = 3
    r = odsd.verify_drafts(torch.zeros(0, 10, device=dev), none.long(), ctx, none, torch.rand(2, device=dev))
    assert r.tokens.tolist() == [[-1] * 3] * 2 and r.num_accepted.tolist() == [0, 0]


def test_infinite_temperature_is_uniform(dev):
    x = torch.randn(5, 40, device=dev)
    x[:, ::4] = -float("inf")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999], device=dev)
    r = odsd.verify_drafts(x, None, {}, None, u, temperature=torch.full((5,), float("inf"), device=dev))
    free = [i for i in range(40) if i % 4]
    assert r.tokens[:, 0].tolist() == [free[int(v * 30)] for v in (0.0, 0.25, 0.5, 0.75, 0.999)]
    assert torch.equal(odsd.verify_drafts(x, None, {}, None, u, temperature=float("inf")).tokens, r.tokens)


def test_longer_sequences_than_stated(dev):
    """max_query_len below a length: its first rows are verified, as far as they go; nothing is written elsewhere."""
    m = make([5, 3], 400, "fp32", seed=9)
    ctx = {"verify_query_lens": torch.tensor([5, 3], dtype=torch.int32, device=dev), "max_query_len": 3}
    r = odsd.verify_drafts(m["logits"].to(dev), m["drafts"].to(dev), ctx, m["accept_u"].to(dev), m["sample_u"].to(dev), draft_logits=m["draft_logits"].to(dev))
    assert r.tokens.shape == (2, 3) and r.accept_probs[2:4].tolist() == [0.0, 0.0]
    full = make([5, 3], 400, "fp32", seed=9)
    w = orc.verify(full["logits"].double().numpy()[5:], full["drafts"].numpy()[4:], [3], full["accept_u"].numpy()[4:], full["sample_u"].numpy()[1:],
                   full["draft_logits"].double().numpy()[4:])
    assert r.tokens[1].tolist() == w[0][0].tolist()


@pytest.mark.parametrize("lens", [[2 ** 30] * 5, [2 ** 31 - 1, 2 ** 31 - 1, 1, 4], [3, 2 ** 31 - 1, 2 ** 31 - 1, 5]])
def test_lengths_that_do_not_belong_to_the_rows(dev, lens):
    """Lengths on the device are not checked; the first sequence's rows are verified as far as there are any, nobody else's are
    taken for it, and sums of lengths past 31 bits find no row."""
    m = make([4, 4], 300, "fp32", seed=14)
    ctx = {"verify_query_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": 3}
    su = torch.rand(len(lens), device=dev)
    for q in (m["draft_logits"].to(dev), None):
        r = odsd.verify_drafts(m["logits"].to(dev), m["drafts"].to(dev), ctx, m["accept_u"].to(dev), su, draft_logits=q,
                               temperature=torch.full((len(lens),), 0.8, device=dev))
        tokens = r.tokens.cpu()
        assert (tokens >= -1).all() and (tokens < 300).all() and tokens[0, 0] >= 0 and (r.num_accepted <= 2).all()
        if lens[0] > 3:
            assert (tokens[1] == -1).all()


def test_two_calls_at_once(dev):
    """Calls on two streams have workspaces of their own."""
    ms = [make([4, 2, 5], 70000, "bf16", seed=s) for s in (41, 42)]
    args = [{k: v.to(dev) for k, v in m.items() if k != "lens"} for m in ms]
    ctx = {"verify_query_lens": torch.tensor([4, 2, 5], dtype=torch.int32, device=dev), "max_query_len": 5}
    call = lambda a: odsd.verify_drafts(a["logits"], a["drafts"], ctx, a["accept_u"], a["sample_u"], draft_logits=a["draft_logits"], temperature=0.8)  # noqa: E731
    alone = [call(a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in ms], [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(args[i]))
    torch.cuda.synchronize()
    for want, rs in zip(alone, got):
        for r in rs:
            assert torch.equal(r.tokens, want.tokens) and torch.equal(r.accept_probs, want.accept_probs)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("pad,offset", [(0, 1), (5, 0), (8, 0), (7, 3)])
def test_strided_and_unaligned_rows(dev, dtype, pad, offset):
    m = make([3, 2, 4], 2049, dtype, seed=11)
    views = []
    for t in (m["logits"], m["draft_logits"]):
        buf = torch.full((t.shape[0] * (2049 + pad) + offset + 8,), float("nan"), dtype=t.dtype, device=dev)
        v = torch.as_strided(buf, t.shape, (2049 + pad, 1), offset)
        v.copy_(t)
        views.append(v)
    check(dev, m, 0.8, None, *views)


def test_sampling_of_a_decode_step(dev):
    """No drafts and a decode context: one token per row; the shares of many draws are the probabilities."""
    g = torch.Generator().manual_seed(0)
    row = torch.randn(1, 50, generator=g)
    n = 4096
    u = ((torch.arange(n) + 0.5) / n)
    r = odsd.verify_drafts(row.expand(n, 50).contiguous().to(dev), None, {}, None, u.to(dev), temperature=0.9)
    p = orc.distribution(row[0].double().numpy(), np.float32(0.9))
    share = np.bincount(r.tokens[:, 0].cpu().numpy(), minlength=50) / n
    assert np.abs(share - p).max() <= 1.0 / n + 1e-9 and r.accept_probs.numel() == 0 and not r.num_accepted.any()
    assert odsd.verify_drafts(row[:0].to(dev), None, {}, None, u[:0].to(dev)).tokens.shape == (0, 1)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_sampling_with_temperatures_masks_and_empty_rows(dev, dtype):
    g = torch.Generator().manual_seed(3)
    n, V = 37, 5001
    x = (torch.randn(n, V, generator=g) * 3).to(DT[dtype])
    x[:, 2::3] = -float("inf")
    x[4] = -float("inf")
    x[5] = float("nan")
    x[6, 100] = x[6, 4000] = float("inf")
    x[7, 50] = x[7, 4500] = 40.0
    x[8, :] = torch.finfo(DT[dtype]).min
    x[9, 10] = float("nan")
    t = torch.rand(n, generator=g) * 2
    t[::4] = 0.0
    t[7], t[30], t[31], t[33] = 0.0, 1e-35, 1e35, 3e38
    u = torch.rand(n, generator=g)
    u[10], u[11] = 0.0, 1.0 - 2.0 ** -24
    r = odsd.verify_drafts(x.to(dev), None, {}, None, u.to(dev), temperature=t.to(dev))
    want, _, _ = orc.verify(x.double().numpy(), None, [1] * n, None, u.numpy(), None, t.double().numpy())
    assert r.tokens.cpu().tolist() == want.tolist() and not r.num_accepted.any()


def test_extreme_temperatures_with_drafts(dev):
    lens = [3, 2, 4, 2, 3]
    m = make(lens, 2000, "fp32", seed=21)
    m["logits"][0, 5] = m["draft_logits"][1, 7] = -float("inf")
    check(dev, m, [1e-35, 1e35, 3e38, 1e-44, 50.0])


def test_all_tokens_alike(dev):
    """Rows whose logits are all equal, or equal but one: every rounding of the statistics falls the same way."""
    for V in (131072, 100003):
        m = make([3, 2], V, "fp32", seed=22)
        m["logits"][:] = 1.37
        m["draft_logits"][:] = -0.61
        m["logits"][1, 17] = 12.9
        m["draft_logits"][1, 5] = 13.3
        check(dev, m, 0.77)


def test_many_sequences(dev):
    check(dev, make([2, 1, 3] * 300, 40, "fp32", seed=13))


def test_graph_and_repeats(dev):
    lens = [4, 2, 5]
    m = make(lens, 40000, "bf16", seed=7)
    x, q, d, au, su = (m[k].to(dev) for k in ("logits", "draft_logits", "drafts", "accept_u", "sample_u"))
    ctx = {"verify_query_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_query_len": 5}
    call = lambda: odsd.verify_drafts(x, d, ctx, au, su, draft_logits=q, temperature=0.8)  # noqa: E731
    first = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        again = call()
        for a, b in ((out.tokens, again.tokens), (out.num_accepted, again.num_accepted), (out.accept_probs, again.accept_probs)):
            assert torch.equal(a, b), i
        if i == 0:
            assert torch.equal(first.tokens, again.tokens) and torch.equal(first.accept_probs, again.accept_probs)
        x.add_(torch.randn_like(x))
        au.uniform_()
        su.uniform_()


def test_refusals(dev):
    m = make([3, 2], 100, "bf16")
    x, q, d, au, su = (m[k].to(dev) for k in ("logits", "draft_logits", "drafts", "accept_u", "sample_u"))
    ctx = {"verify_query_lens": torch.tensor([3, 2], dtype=torch.int32, device=dev), "max_query_len": 3}
    ok = odsd.verify_drafts(x, d.to(torch.int32), ctx, au, su, draft_logits=q)
    assert ok.tokens.shape == (2, 3)
    # lengths on the host; [4, 1] are as many rows and drafts as [3, 2]
    assert odsd.verify_drafts(x, d, {"verify_query_lens": torch.tensor([4, 1])}, au, su).tokens.shape == (2, 5)
    for call in (lambda: odsd.verify_drafts(x.double(), d, ctx, au, su), lambda: odsd.verify_drafts(x, d, ctx, au.double(), su),
                 lambda: odsd.verify_drafts(x, d, ctx, au, su.half())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: odsd.verify_drafts(x, d, {}, au, su), lambda: odsd.verify_drafts(x, d, ctx, None, su), lambda: odsd.verify_drafts(x, d, ctx, au[:2], su),
                 lambda: odsd.verify_drafts(x, d, ctx, au, su[:1]), lambda: odsd.verify_drafts(x, d, ctx, au, su, draft_logits=q[:2]),
                 lambda: odsd.verify_drafts(x, d, ctx, au, su, draft_logits=q.float()), lambda: odsd.verify_drafts(x, d, ctx, au, su, temperature=-1.0),
                 lambda: odsd.verify_drafts(x, d, ctx, au, su, temperature=torch.ones(3, device=dev)),
                 lambda: odsd.verify_drafts(x, None, {}, None, su), lambda: odsd.verify_drafts(x, d, {"verify_query_lens": torch.tensor([4, 2])}, au, su),
                 lambda: odsd.verify_drafts(x, d, {"verify_query_lens": torch.tensor([5, 0])}, au, su),
                 lambda: odsd.verify_drafts(x, d, {"verify_query_lens": torch.tensor([3, 2]), "max_query_len": 2}, au, su)):
        with pytest.raises(ValueError):
            call()
