"""The 8-bit cache's operators as a server uses them together: prompts stored, a fork, a verify step -- store, attention, head, adjustment, verification --,
what was not kept taken back, compaction; and the same step captured into a graph and replayed beside eager calls."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import ops
from oracle import cache_oracle as corc
from oracle import dense_oracle as dorc

pytestmark = pytest.mark.gpu
HQ, H, D, BS, V = 8, 2, 64, 16, 500


def test_a_verify_step_between_fork_and_compaction(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    cache = odsd.KVCacheFP8.zeros(40, H, BS, D, dev)
    pool = odsd.BlockPool(40, BS, [cache])
    mirror = [t.cpu().numpy() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales.double())]
    seqs = {i: odsd.SequenceSlots(BS) for i in range(3)}

    def store(key, value, slots, src=None):
        odsd.store_kvcache_fp8(key, value, cache, slots, src)
        corc.store(key.double().cpu().numpy(), value.double().cpu().numpy(), *mirror, slots.tolist(), None if src is None else src.tolist())

    pool.append(list(seqs.values()), [37, 16, 5])
    context = odsd.build_prefill_context(seqs, [0, 1, 2], dev)
    store(randn(58, H, D).to(torch.bfloat16), randn(58, H, D).to(torch.bfloat16), context["slot_mapping"])
    seqs[3] = pool.fork(seqs[0])
    for s in seqs.values():
        s.draft_start_num_tokens = s.num_tokens
    before = {i: list(s.block_table) for i, s in seqs.items()}
    pool.append(list(seqs.values()), [3, 2, 0, 1])
    for i, s in seqs.items():                       # the books' copies, in the mirror too
        for old, new in zip(before[i], s.block_table):
            if old != new:
                for m in mirror:
                    m[new] = m[old]
    context = odsd.build_verify_context(seqs, [0, 1, 2, 3], dev)
    n = 4 + 3 + 2 + 0 + 1
    key, value, q = randn(n, H, D).to(torch.bfloat16), randn(n, H, D).to(torch.bfloat16) * 20, randn(n, HQ, D).to(torch.bfloat16)
    store(key, value, context["slot_mapping"], context["verify_q_indices"])
    assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), mirror[0]) and np.array_equal(cache.v.view(torch.uint8).cpu().numpy(), mirror[1])
    assert np.array_equal(cache.scales.double().cpu().numpy(), mirror[2])
    hidden = odsd.attention_for_context(q, None, None, cache, None, context, H, BS)
    lens, q_lens = context["context_lens"].tolist(), context["verify_query_lens"].tolist()
    want, mag, top = corc.attend(q.double().cpu().numpy(), *mirror, context["block_tables"].cpu().numpy(), lens, q_lens, D ** -0.5)
    u = 2.0 ** -8
    limit = 2 * (u + 2 * (D + 8) * 2.0 ** -24 * (top[..., None] + 1) + 70 * 2.0 ** -24) * mag + u * np.abs(want)
    assert (np.abs(hidden.double().cpu().numpy() - want) <= limit).all()
    head = (randn(V, HQ * D) * 0.05).to(torch.bfloat16)
    logits = ops.linear(hidden.flatten(1), head, out_dtype=torch.float32)
    drafts = torch.randint(0, V, (6,), generator=g, device=dev)
    tokens = torch.randint(0, V, (4, 60), generator=g, device=dev)
    token_lens = [37, 16, 5, 37]
    mask = torch.randint(-2 ** 31, 2 ** 31, (2, 16), generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    mask_rows = torch.tensor([0, -1, 1, 0, -1, -1, 1, 0, 1, 1], dtype=torch.int32, device=dev)
    accept, draw = torch.rand(6, generator=g, device=dev), torch.rand(4, generator=g, device=dev)
    raw = logits.double().cpu().numpy()
    adjusted = odsd.adjust_logits(logits, context, tokens=tokens, token_lens=torch.tensor(token_lens), draft_tokens=drafts, repetition=1.5, frequency=0.25,
                                  mask=mask, mask_rows=mask_rows, out=logits)
    assert adjusted is logits
    want, mag = corc.adjust(raw, q_lens, tokens.tolist(), token_lens, None, drafts.tolist(), [1.5] * 4, [0.25] * 4, [0.0] * 4, None, mask.cpu().numpy(), mask_rows.tolist())
    assert np.array_equal(np.isinf(adjusted.cpu().numpy()), np.isinf(want)) and np.isinf(want).any()
    fine = np.isfinite(want)
    assert (np.abs(adjusted.double().cpu().numpy()[fine] - want[fine]) <= 6 * 2.0 ** -24 * mag[fine]).all()
    r = odsd.verify_drafts(adjusted, drafts, context, accept, draw, temperature=0.7)
    temperature = float(torch.tensor(0.7))
    tokens_want, kept, _ = dorc.verify(adjusted.double().cpu().numpy(), drafts.cpu().numpy(), q_lens, accept.cpu().numpy(), draw.cpu().numpy(), None, temperature, 4)
    assert r.tokens.tolist() == tokens_want.tolist() and r.num_accepted.tolist() == list(kept)
    for i, k in enumerate(r.num_accepted.tolist()):
        pool.truncate(seqs[i], seqs[i].draft_start_num_tokens + k)
    pool.free(seqs.pop(0))
    left = list(seqs)
    context = odsd.build_decode_context(seqs, left, dev)
    q = randn(3, HQ, D).to(torch.float16)
    one = odsd.paged_attention_fp8(q, cache, context)
    pool.compact(list(seqs.values()), context["block_tables"])
    assert context["block_tables"].tolist() == odsd.build_decode_context(seqs, left, dev)["block_tables"].tolist()
    assert torch.equal(odsd.paged_attention_fp8(q, cache, context), one)


def test_captured_and_replayed(dev):
    """two graphs over the same cache; their inputs, lengths and slots change between the replays, eager calls run in between"""
    g = torch.Generator(device=dev).manual_seed(1)
    nb, S, ql, n = 30, 3, 3, 9
    cache = odsd.KVCacheFP8.zeros(nb, H, BS, D, dev)
    key, value = (torch.zeros(n, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    q = torch.zeros(n, HQ, D, dtype=torch.bfloat16, device=dev)
    slots = torch.full((n,), -1, dtype=torch.int32, device=dev)
    tables = torch.arange(S * 8, dtype=torch.int32, device=dev).view(S, 8)
    lens = torch.full((S,), ql, dtype=torch.int32, device=dev)
    context = {"block_tables": tables, "context_lens": lens, "verify_query_lens": torch.full((S,), ql, dtype=torch.int32, device=dev), "max_query_len": ql}
    head = (torch.randn(V, HQ * D, generator=g, device=dev) * 0.05).to(torch.bfloat16)
    drafts, tokens = torch.zeros(6, dtype=torch.int64, device=dev), torch.zeros(S, 20, dtype=torch.int64, device=dev)
    token_lens = torch.zeros(S, dtype=torch.int32, device=dev)
    mask = torch.full((n, 16), -1, dtype=torch.int32, device=dev)

    def step(c):
        odsd.store_kvcache_fp8(key, value, c, slots)
        hidden = odsd.paged_attention_fp8(q, c, context)
        logits = ops.linear(hidden.flatten(1), head, out_dtype=torch.float32)
        out = odsd.adjust_logits(logits, context, tokens=tokens, token_lens=token_lens, draft_tokens=drafts, repetition=1.3, presence=0.5, mask=mask)
        odsd.copy_cache_blocks([c], [2, 9], [28, 29])
        return hidden, out

    step(odsd.KVCacheFP8(cache.k.clone(), cache.v.clone(), cache.scales.clone()))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache)
        graphs.append((graph, out))
    eager = odsd.KVCacheFP8(cache.k.clone(), cache.v.clone(), cache.scales.clone())
    at = 0
    for i in range(8):
        for t in (key, value, q):
            t.normal_(generator=g).mul_(1.0 + i)
        pos = torch.arange(at, at + ql, device=dev)
        slots.copy_((tables[:, pos // BS] * BS + pos % BS).flatten().to(torch.int32))
        lens.fill_(at + ql)
        drafts.random_(0, V, generator=g)
        tokens.random_(0, V, generator=g)
        token_lens.random_(0, 21, generator=g)
        mask.random_(-2 ** 31, 2 ** 31 - 1, generator=g)
        at += ql if i != 4 else 0                   # (one step is taken again)
        graph, got = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(cache.k.view(torch.uint8), eager.k.view(torch.uint8)) and torch.equal(cache.v.view(torch.uint8), eager.v.view(torch.uint8))
        assert torch.equal(cache.scales, eager.scales)


def test_on_another_stream(dev):
    """inputs made on one stream, the calls on another that waits for it"""
    side = torch.cuda.Stream()
    cache = odsd.KVCacheFP8.zeros(300, H, BS, D, dev)
    twin = odsd.KVCacheFP8.zeros(300, H, BS, D, dev)
    tables = torch.arange(300, dtype=torch.int32, device=dev).view(2, 150)
    key = torch.randn(4000, H, D, device=dev).to(torch.bfloat16)
    slots = torch.arange(4000, dtype=torch.int32, device=dev)
    q = torch.randn(2, HQ, D, device=dev).to(torch.bfloat16)
    context = {"block_tables": tables, "context_lens": torch.tensor([2400, 1600], dtype=torch.int32, device=dev)}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        odsd.store_kvcache_fp8(key, key, cache, slots)
        odsd.copy_cache_blocks([cache], [0, 1], [280, 281])
        a = odsd.paged_attention_fp8(q, cache, context)
        b = odsd.adjust_logits(a.flatten(1).float(), {}, repetition=2.0, tokens=slots.view(2, 2000))
    side.synchronize()
    odsd.store_kvcache_fp8(key, key, twin, slots)
    odsd.copy_cache_blocks([twin], [0, 1], [280, 281])
    want = odsd.paged_attention_fp8(q, twin, context)
    assert torch.equal(a, want) and torch.equal(b, odsd.adjust_logits(want.flatten(1).float(), {}, repetition=2.0, tokens=slots.view(2, 2000)))
    assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8)) and torch.equal(cache.scales, twin.scales)


def test_two_at_once(dev):
    """the same calls on two streams, neither waiting for the other: every one has its own workspace"""
    g = torch.Generator(device=dev).manual_seed(4)
    n, new = 3, 6000
    key = torch.randn(2, new, H, D, generator=g, device=dev).to(torch.bfloat16)
    slots = torch.stack([torch.randperm(400 * BS, generator=g, device=dev)[:new].to(torch.int32) for _ in range(2)])
    tables = torch.arange(375, dtype=torch.int32, device=dev).view(n, 125)
    q = torch.randn(2, n, HQ, D, generator=g, device=dev).to(torch.bfloat16)
    logits = torch.randn(2, n, 5000, generator=g, device=dev)
    tokens = torch.randint(0, 5000, (2, n, 700), generator=g, device=dev)
    context = {"block_tables": tables, "context_lens": torch.tensor([2000, 1500, 7], dtype=torch.int32, device=dev)}

    def step(i, cache):
        odsd.store_kvcache_fp8(key[i], key[i], cache, slots[i])
        odsd.copy_cache_blocks([cache], [0, 1, 2], [397, 398, 399])
        return odsd.paged_attention_fp8(q[i], cache, context), odsd.adjust_logits(logits[i], {}, tokens=tokens[i], repetition=1.5, frequency=0.25)

    caches = [[odsd.KVCacheFP8.zeros(400, H, BS, D, dev) for _ in range(2)] for _ in range(2)]
    want = [step(i, caches[0][i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i, caches[1][i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(caches[0][i].k.view(torch.uint8), caches[1][i].k.view(torch.uint8)) and torch.equal(caches[0][i].scales, caches[1][i].scales)
        for a, x in got[i]:
            assert torch.equal(torch.isnan(a), torch.isnan(want[i][0])) and torch.equal(a.nan_to_num(), want[i][0].nan_to_num()) and torch.equal(x, want[i][1])
