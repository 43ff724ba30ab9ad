"""paged_attention_fp8 against the oracle in 64 bits, on the values that the cache stands for.

Error bound of an output, from the arithmetic: each weight is rounded to q's type (half a step, u = eps / 2, relative), the result once more
(u |out|); scores are fp32 sums of D products, off by at most (D + 8) 2^-24 of the sum of the products' magnitudes (with the scale's own
roundings), which changes a weight by that much relatively, in numerator and denominator (twice); exp2 and the sums of up to L weights add less
than (L / 16 + 64) 2^-24.  fp16 outputs below 2^-14 have steps of 2^-24."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def make(dev, H, D, bs, lens, seed, spare=3, extra=0, spread=0):
    """(cache, tables): random codes, NaN wherever no sequence has a key; `extra` more columns of -1; scales 2^-8 .. 2^-8 + spread"""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + spare
    order = np.random.default_rng(seed).permutation(nb)
    cache = odsd.KVCacheFP8.zeros(nb, H, bs, D, dev)
    cache.k.copy_((torch.randn(nb, H, bs, D, generator=g, device=dev) * 60).clamp(-448, 448))
    cache.v.copy_((torch.randn(nb, H, D, bs, generator=g, device=dev) * 60).clamp(-448, 448))
    cache.scales.copy_(torch.exp2(-6.0 + torch.randint(0, spread + 1, (nb, H, 2), generator=g, device=dev).float()))
    tables = torch.full((len(lens), max(max(need), 1) + extra), -1, dtype=torch.int32)
    used = torch.zeros(nb, bs, dtype=torch.bool)
    at = 0
    for i, (n, b) in enumerate(zip(lens, need)):
        tables[i, :b] = torch.tensor(order[at:at + b].astype(np.int32))
        for j in range(b):
            used[order[at + j], :min(bs, n - j * bs)] = True
        at += b
    free = ~used.to(dev)
    cache.k.view(torch.uint8).masked_fill_(free[:, None, :, None], 0x7f)
    cache.v.view(torch.uint8).masked_fill_(free[:, None, None, :], 0xff)
    return cache, tables.to(dev)


def expected(q, cache, tables, lens, q_lens, scale):
    return orc.attend(q.double().cpu().numpy(), cache.k.view(torch.uint8).cpu().numpy(), cache.v.view(torch.uint8).cpu().numpy(),
                      cache.scales.double().cpu().numpy(), tables.cpu().numpy(), lens, q_lens, scale)


def bound(out, mag, top, dtype, D, L):
    u = torch.finfo(dtype).eps / 2
    weights = u + 2 * (D + 8) * 2.0 ** -24 * (top[..., None] + 1) + (L / 16 + 64) * 2.0 ** -24
    return 2 * weights * mag + u * np.abs(out) + (2.0 ** -24 if dtype == torch.float16 else 1e-30)


def check(dev, heads, H, D, bs, lens, q_lens, dtype, seed=0, context_more=None, explicit=True, rows_behind=0, scale=None, **how):
    cache, tables = make(dev, H, D, bs, lens, seed, **how)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    n = sum(q_lens)
    q = torch.randn(n + rows_behind, heads, D, generator=g, device=dev).to(dtype)
    ctx = {"block_tables": tables, "context_lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if explicit:
        ctx["verify_query_lens"] = torch.tensor(q_lens, dtype=torch.int32, device=dev)
    ctx.update(context_more or {})
    got = odsd.paged_attention_fp8(q, cache, ctx, scale)
    torch.cuda.synchronize()
    want, mag, top = expected(q[:n], cache, tables, lens, q_lens, D ** -0.5 if scale is None else scale)
    assert got.shape == q.shape and got.dtype == dtype
    off = np.abs(got[:n].double().cpu().numpy() - want)
    limit = bound(want, mag, top, dtype, D, max(lens))
    worst = np.nanmax(off / limit)
    assert np.array_equal(np.isnan(off), np.isnan(want)) and worst <= 1, worst
    return got, q, cache, ctx


HEADS = [(32, 4, 128), (8, 8, 64), (14, 2, 64), (8, 1, 128), (28, 4, 128), (6, 3, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, H, D", HEADS)
@pytest.mark.parametrize("bs", [16, 48, 64, 256])
def test_decode(dev, dtype, heads, H, D, bs):
    """one query a sequence, lengths round every border of a group, a tile, a step and a block"""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300, 513]
    check(dev, heads, H, D, bs, lens, [1] * len(lens), dtype, explicit=False, spread=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, H, D", HEADS)
@pytest.mark.parametrize("bs", [16, 32, 128])
@pytest.mark.parametrize("most", [2, 5, 9, 40])
def test_verify_and_chunks(dev, dtype, heads, H, D, bs, most):
    """several queries a sequence: 16, 32, 64 rows and more of them; sequences that are all query, free places"""
    rng = np.random.default_rng(most)
    q_lens = [int(n) for n in rng.integers(1, most + 1, 7)] + [most, 0, 1]
    lens = [int(n) + q for n, q in zip((0, 3, 61, 64, 190, 255, 320, 777, 0, 0), q_lens)]
    lens[8], lens[9] = 30, 0                       # keys without a query; a query without keys
    check(dev, heads, H, D, bs, lens, q_lens, dtype, seed=most, context_more={"max_query_len": most}, spread=2)


@pytest.mark.parametrize("heads, H, D, q, L, bs", [(32, 4, 128, 1, 9000, 256), (8, 2, 64, 1, 20001, 16), (32, 8, 128, 6, 5003, 64),
                                                  (16, 2, 128, 8, 6007, 48), (8, 1, 128, 100, 3001, 256), (4, 4, 64, 300, 1777, 32),
                                                  (16, 1, 128, 8, 9001, 64), (8, 1, 64, 4, 30000, 256), (3, 1, 128, 1, 40000, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_sequences_are_shared_out(dev, heads, H, D, q, L, bs, dtype):
    """units are cut into pieces whose results are joined; short sequences beside them"""
    lens, q_lens = [q, L, 0, q + 40, 511], [q, q, 1, q, min(q, 511)]
    check(dev, heads, H, D, bs, lens, q_lens, dtype, seed=3, context_more={"max_query_len": q}, spread=4)


def test_bound_from_the_tokens(dev):
    """no max_query_len: as many queries as there are tokens are allowed for"""
    check(dev, 8, 2, 64, 32, [100, 40, 700], [3, 4, 2], torch.bfloat16)
    check(dev, 8, 2, 64, 32, [100, 40, 700], [3, 4, 2], torch.bfloat16, context_more={"max_query_len": 64})
    check(dev, 8, 2, 64, 32, [100, 40, 700], [3, 4, 2], torch.bfloat16, extra=200)         # tables far longer than the contexts


@pytest.mark.parametrize("n_seqs, heads, H, D, q, lens", [
    (32, 4, 4, 64, 1, (2048, 1, 2033)), (32, 4, 4, 64, 1, (2064, 0, 700)), (64, 4, 4, 64, 1, (4096, 5)), (64, 4, 4, 64, 1, (4112, 16)),
    (32, 8, 4, 128, 1, (1024, 17)), (32, 8, 4, 128, 1, (1040, 1000)), (1, 8, 4, 128, 1, (512,)), (1, 8, 4, 128, 1, (528,)), (1, 8, 1, 64, 1, (1040,)),
    (12, 28, 4, 64, 3, (576, 60)), (12, 28, 4, 64, 3, (592, 3)), (16, 16, 4, 64, 9, (768, 9)), (16, 16, 4, 64, 9, (784, 500)),
    (4, 64, 4, 64, 16, (512, 100)), (4, 64, 4, 64, 16, (528, 528))])
def test_whole_and_split_units(dev, n_seqs, heads, H, D, q, lens):
    """tables just within and just past the length up to which units are not split, for every number of rows"""
    lens = [lens[i % len(lens)] for i in range(n_seqs)]
    check(dev, heads, H, D, 16, lens, [q] * n_seqs, torch.bfloat16, explicit=q > 1, context_more={"max_query_len": q})


def test_many_sequences(dev):
    rng = np.random.default_rng(7)
    lens = [int(n) for n in rng.integers(0, 700, 700)]
    check(dev, 4, 2, 64, 32, lens, [1] * 700, torch.float16, explicit=False)
    lens = [int(n) + 3 for n in rng.integers(0, 90, 300)]
    check(dev, 32, 4, 64, 16, lens, [3] * 300, torch.bfloat16, context_more={"max_query_len": 3})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_far_apart(dev, dtype):
    """blocks whose scales of V are 2^40 apart, which fp16 weights could not hold side by side"""
    cache, tables = make(dev, 2, 64, 16, [300, 40], 5)
    g = torch.Generator(device=dev).manual_seed(1)
    cache.scales[..., 1] = torch.exp2(torch.randint(-30, 11, cache.scales[..., 1].shape, generator=g, device=dev).float())
    q = torch.randn(2, 4, 64, generator=g, device=dev).to(dtype)
    if dtype == torch.float16:                     # (the result has to fit)
        cache.scales[..., 1] *= 2.0 ** -15
    ctx = {"block_tables": tables, "context_lens": torch.tensor([300, 40], dtype=torch.int32, device=dev)}
    got = odsd.paged_attention_fp8(q, cache, ctx).double().cpu().numpy()
    want, mag, top = expected(q, cache, tables, [300, 40], [1, 1], 64 ** -0.5)
    assert (np.abs(got - want) <= bound(want, mag, top, dtype, 64, 300)).all()


def test_sharp_and_flat_scores(dev):
    check(dev, 8, 2, 128, 64, [900, 1300], [2, 3], torch.bfloat16, scale=3.0, context_more={"max_query_len": 3})
    check(dev, 8, 2, 128, 64, [900, 1300], [2, 3], torch.float16, scale=1e-6, context_more={"max_query_len": 3})


@pytest.mark.parametrize("q_len, heads", [(4, 4), (4, 16), (5, 64)])
@pytest.mark.parametrize("at", [0, 1, 3])
def test_nan_reaches_the_rows_that_attend_it(dev, q_len, heads, at):
    """a NaN in K takes the whole row, in V its dimension; queries in front of it are untouched"""
    H, D, bs, L = 2, 64, 32, 200
    for name in ("k", "v"):
        cache, tables = make(dev, H, D, bs, [L], 2)
        pos = L - q_len + at                       # the key of query `at`
        block, token = int(tables[0, pos // bs]), pos % bs
        codes = getattr(cache, name).view(torch.uint8)
        if name == "k":
            codes[block, 1, token, 7] = 0x7f
        else:
            codes[block, 1, 7, token] = 0xff
        q = torch.randn(q_len, heads, D, generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(torch.bfloat16)
        ctx = {"block_tables": tables, "context_lens": torch.tensor([L], dtype=torch.int32, device=dev), "max_query_len": q_len,
               "verify_query_lens": torch.tensor([q_len], dtype=torch.int32, device=dev)}
        got = torch.isnan(odsd.paged_attention_fp8(q, cache, ctx)).view(q_len, H, heads // H, D)
        want = torch.zeros_like(got)
        if name == "k":
            want[at:, 1] = True
        else:
            want[at:, 1, :, 7] = True
        assert bool((got == want).all())


def test_odd_lengths_and_tables(dev):
    """table entries that name no block read block 0, rows behind the last sequence's are nobody's, the same call gives the same bits"""
    cache, tables = make(dev, 2, 64, 16, [100, 80], 2, spare=0)
    cache.k.view(torch.uint8).masked_fill_(torch.isnan(cache.k.float()), 1)
    cache.v.view(torch.uint8).masked_fill_(torch.isnan(cache.v.float()), 1)
    tables[0, 3], tables[1, 1] = -7, 1 << 30
    q = torch.randn(2, 4, 64, generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(torch.float16)
    ctx = {"block_tables": tables, "context_lens": torch.tensor([100, 80], dtype=torch.int32, device=dev)}
    got = odsd.paged_attention_fp8(q, cache, ctx)
    want, mag, top = expected(q, cache, tables, [100, 80], [1, 1], 64 ** -0.5)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound(want, mag, top, torch.float16, 64, 100)).all()
    a = check(dev, 32, 4, 128, 64, [3000, 5], [8, 2], torch.bfloat16, rows_behind=6, context_more={"max_query_len": 8})
    assert torch.equal(odsd.paged_attention_fp8(*a[1:])[:10], a[0][:10])


@pytest.mark.parametrize("L, blocks", [(100, 2), (3000, 5), (70000, 200), (1 << 30, 40)])
@pytest.mark.parametrize("q_len, heads", [(1, 2), (3, 2), (6, 8), (9, 16)])
def test_a_context_past_its_table(dev, L, blocks, q_len, heads):
    """positions that the table has no entry for are not attended: every row sees the keys of the table's entries (-1 reads block 0)"""
    bs, D = 16, 64
    cache, tables = make(dev, 2, D, bs, [blocks * bs, 40], 4)
    q = torch.randn(q_len + 1, heads, D, generator=torch.Generator(device=dev).manual_seed(5), device=dev).to(torch.bfloat16)
    ctx = {"block_tables": tables, "context_lens": torch.tensor([L, 40], dtype=torch.int32, device=dev), "max_query_len": q_len,
           "verify_query_lens": torch.tensor([q_len, 1], dtype=torch.int32, device=dev)}
    got = odsd.paged_attention_fp8(q, cache, ctx).double().cpu().numpy()
    width = tables.shape[1] * bs
    ends = [min(L - q_len + 1 + j, width) for j in range(q_len)] + [40]
    rows = tables[[0] * q_len + [1]]
    want, mag, top = expected(q, cache, rows, ends, [1] * (q_len + 1), D ** -0.5)
    off = np.abs(got - want)
    assert np.array_equal(np.isnan(off), np.isnan(want)) and not (off > bound(want, mag, top, torch.bfloat16, D, width)).any()


@pytest.mark.parametrize("L", [300, 6000])
@pytest.mark.parametrize("heads, most", [(2, 4), (8, 8), (32, 8)])
@pytest.mark.parametrize("told", [[3, 9, 4], [3, 1 << 30, 1 << 30], [3, -2, 7]])
def test_query_lengths_past_the_rows(dev, L, heads, most, told):
    """q and out have 5 rows: nothing behind them is touched, and the first sequence, whose length is right, has its results"""
    D, n = 64, 5
    cache, tables = make(dev, 2, D, 64, [L, L, L], 6)
    q = torch.randn(40, heads, D, generator=torch.Generator(device=dev).manual_seed(7), device=dev).to(torch.bfloat16)
    out = torch.full((40, heads, D), 7.0, dtype=torch.bfloat16, device=dev)
    lens, q_lens = (torch.tensor(t, dtype=torch.int32, device=dev) for t in ([L] * 3, told))
    lib = odsd._lib.load()
    size = lib.odsd_paged_attention_fp8_workspace_bytes(3, most, heads, 2, D, 64, tables.shape[1])
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    rc = lib.odsd_paged_attention_fp8(q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.scales.data_ptr(), tables.data_ptr(),
                                      lens.data_ptr(), q_lens.data_ptr(), n, 3, most, heads, 2, D, 64, tables.shape[1], cache.k.shape[0],
                                      D ** -0.5, odsd._lib.DT_BF16, out.data_ptr(), ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and bool((out[n:] == 7.0).all())
    want, mag, top = expected(q[:3], cache, tables[:1], [L], [3], D ** -0.5)
    assert (np.abs(out[:3].double().cpu().numpy() - want) <= bound(want, mag, top, torch.bfloat16, D, L)).all()


def test_a_cache_past_32_bits(dev):
    """blocks whose bytes begin beyond 2^32"""
    H, D, bs = 8, 128, 256
    nb = (1 << 32) // (H * D * bs) + 40
    cache = odsd.KVCacheFP8.zeros(nb, H, bs, D, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    key, value = (torch.randn(400, H, D, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    blocks = [nb - 1, nb - 20]
    slots = torch.tensor([blocks[p // bs] * bs + p % bs for p in range(400)], dtype=torch.int32, device=dev)
    odsd.store_kvcache_fp8(key, value, cache, slots)
    tables = torch.tensor([blocks], dtype=torch.int32, device=dev)
    q = torch.randn(1, 32, D, generator=g, device=dev).to(torch.bfloat16)
    got = odsd.paged_attention_fp8(q, cache, {"block_tables": tables, "context_lens": torch.tensor([400], dtype=torch.int32, device=dev)})
    few = odsd.KVCacheFP8(cache.k[blocks[::-1]], cache.v[blocks[::-1]], cache.scales[blocks[::-1]])
    want, mag, top = expected(q, few, torch.tensor([[1, 0]]), [400], [1], D ** -0.5)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound(want, mag, top, torch.bfloat16, D, 400)).all()


def test_refusals(dev):
    cache, tables = make(dev, 2, 64, 16, [30, 20], 1)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    lens = torch.tensor([30, 20], dtype=torch.int32, device=dev)
    ctx = {"block_tables": tables, "context_lens": lens}
    f = odsd.paged_attention_fp8
    for error, call in ((TypeError, lambda: f(q.float(), cache, ctx)), (ValueError, lambda: f(q[:, :3], cache, ctx)),
                        (ValueError, lambda: f(q[..., :32], cache, ctx)), (ValueError, lambda: f(q[:1], cache, ctx)),
                        (ValueError, lambda: f(q, cache, {**ctx, "verify_query_lens": lens[:1]})),
                        (ValueError, lambda: f(q, cache, {**ctx, "verify_query_lens": torch.tensor([2, 1], dtype=torch.int32)})),
                        (ValueError, lambda: f(q, cache, {**ctx, "verify_query_lens": torch.tensor([2, 0], dtype=torch.int32)}, None, 1)),
                        (ValueError, lambda: f(q, cache, {**ctx, "block_tables": tables[:1]})),
                        (RuntimeError, lambda: f(q, odsd.KVCacheFP8(cache.k.cpu(), cache.v, cache.scales), ctx)),
                        (odsd._lib.OdsdError, lambda: f(q, cache, ctx, 0.0)), (odsd._lib.OdsdError, lambda: f(q, cache, ctx, float("nan"))),
                        (ValueError, lambda: odsd.attention_for_context(q, None, None, cache, cache, ctx, 2, 16)),
                        (ValueError, lambda: odsd.attention_for_context(q, None, None, cache, None, ctx, 2, 32))):
        with pytest.raises(error):
            call()
    assert f(q[:0], cache, {"block_tables": tables[:0], "context_lens": lens[:0]}).shape == (0, 4, 64)
    assert not f(q, cache, {"block_tables": tables[:, :0], "context_lens": torch.zeros_like(lens)}).any()
    assert torch.equal(odsd.attention_for_context(q, None, None, cache, None, ctx, 2, 16), f(q, cache, ctx))
