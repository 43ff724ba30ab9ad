"""store_kvcache_fp8 against the oracle: every code and every scale of the cache, bit for bit (scales are powers of two, so all
arithmetic on the way to a rounding is exact)."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def filled(dev, nb, H, bs, D, seed):
    """A cache in which earlier rows stand, some blocks empty with whatever bytes are there."""
    g = torch.Generator(device=dev).manual_seed(seed)
    cache = odsd.KVCacheFP8.zeros(nb, H, bs, D, dev)
    cache.k.view(torch.uint8).random_(0, 256, generator=g)
    cache.v.view(torch.uint8).random_(0, 256, generator=g)
    cache.scales.copy_(torch.exp2(torch.randint(-12, 3, (nb, H, 2), generator=g, device=dev).float()))
    cache.scales[::5] = 0
    return cache


def as_numpy(cache):
    return cache.k.view(torch.uint8).cpu().numpy().copy(), cache.v.view(torch.uint8).cpu().numpy().copy(), cache.scales.double().cpu().numpy()


def check(cache, key, value, slots, src=None):
    k, v, s = as_numpy(cache)
    odsd.store_kvcache_fp8(key, value, cache, slots, src)
    torch.cuda.synchronize()
    orc.store(key.double().cpu().numpy(), value.double().cpu().numpy(), k, v, s, slots.tolist(), None if src is None else src.tolist())
    gk, gv, gs = as_numpy(cache)
    assert np.array_equal(gs, s)
    # (which sign a NaN has is not said)
    assert np.array_equal(orc.E4M3[gk], orc.E4M3[k], equal_nan=True) and np.array_equal(orc.E4M3[gv], orc.E4M3[v], equal_nan=True)


def rows(dev, n, H, D, dtype, seed, gain=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(n, H, D, generator=g, device=dev) * gain).to(dtype) for _ in range(2)]


def places(blocks, starts, lens, bs):
    """Slots of sequences whose blocks are given out in the order of `blocks`."""
    blocks, out = iter(blocks), []
    for first, n in zip(starts, lens):
        table = {}
        for p in range(first, first + n):
            b = table.setdefault(p // bs, None)
            if b is None:
                b = table[p // bs] = next(blocks)
            out.append(b * bs + p % bs)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H, D, bs", [(4, 128, 256), (2, 64, 16), (1, 128, 48), (8, 64, 64), (3, 128, 1024), (16, 64, 32)])
@pytest.mark.parametrize("starts, lens", [((777,), (1,)), ((0, 0, 0), (300, 1, 17)), ((5, 31, 64, 100), (7, 3, 64, 9)), (tuple(range(3, 43)), (1,) * 40)])
@pytest.mark.parametrize("gain", [1.0, 300.0])
def test_sequences(dev, dtype, H, D, bs, starts, lens, gain):
    """decode, prompts, verify across blocks; with the larger rows every scale rises"""
    need = sum((f + n - 1) // bs - f // bs + 1 for f, n in zip(starts, lens))
    order = np.random.default_rng(need).permutation(need + 3)
    cache = filled(dev, need + 3, H, bs, D, bs)
    slots = torch.tensor(places(order.tolist(), starts, lens, bs), dtype=torch.int32, device=dev)
    check(cache, *rows(dev, len(slots), H, D, dtype, 1, gain), slots)
    check(cache, *rows(dev, len(slots), H, D, dtype, 2, 0.1), slots)           # scales that stay where they are, unless a block starts anew


@pytest.mark.parametrize("N", [1, 50, 700, 5000])
def test_rows_in_any_order(dev, N):
    """no two neighbours of a block, free places, slots and rows that do not exist, slots named twice"""
    H, D, bs, nb = 2, 64, 32, 60
    rng = np.random.default_rng(N)
    n = max(N // 2, 1)
    slots = torch.tensor(rng.integers(-3, nb * bs + 40, N), dtype=torch.int32, device=dev)
    src = torch.tensor(rng.integers(-2, n + 3, N), dtype=torch.int32, device=dev)
    check(filled(dev, nb, H, bs, D, N), *rows(dev, n, H, D, torch.bfloat16, N), slots, src)


@pytest.mark.parametrize("N", [300, 480, 4080, 20000])
def test_all_blocks_side_by_side(dev, N):
    """one token for every block in turn: every workgroup's entries are of other blocks"""
    H, D, bs = 1, 64, 32
    nb = 1 + N // bs
    i = torch.arange(N, device=dev)
    slots = (i % nb * bs + i // nb).to(torch.int32)
    slots = torch.where(i // nb < bs, slots, -1)
    check(filled(dev, nb, H, bs, D, 3), *rows(dev, N, H, D, torch.float16, 4), slots.to(torch.int32))


def test_a_long_prompt(dev):
    """more rows than a workgroup's list, blocks in no order"""
    H, D, bs, N = 1, 64, 16, 9001
    order = np.random.default_rng(5).permutation(600)
    slots = torch.tensor(places(order.tolist(), (3,), (N,), bs), dtype=torch.int32, device=dev)
    check(filled(dev, 600, H, bs, D, 5), *rows(dev, N, H, D, torch.bfloat16, 6), slots)


def test_skipped_rows(dev):
    H, D, bs = 4, 128, 256
    slots = torch.tensor([5, 6, -1, 7, 256 * 3 + 255, 9999, 0], dtype=torch.int32, device=dev)
    check(filled(dev, 4, H, bs, D, 1), *rows(dev, 7, H, D, torch.bfloat16, 8), slots)
    none = torch.full((7,), -1, dtype=torch.int32, device=dev)
    check(filled(dev, 4, H, bs, D, 1), *rows(dev, 7, H, D, torch.bfloat16, 8), none)
    check(filled(dev, 4, H, bs, D, 1), *rows(dev, 0, H, D, torch.bfloat16, 8), none[:0])


@pytest.mark.parametrize("how", ["fused", "misaligned", "transposed", "sliced"])
def test_strides(dev, how):
    n, H, D, bs = 37, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(2)
    if how == "fused":
        qkv = torch.randn(n, 3 * H * D, generator=g, device=dev).to(torch.bfloat16)
        key, value = qkv[:, H * D:2 * H * D].view(n, H, D), qkv[:, 2 * H * D:].view(n, H, D)
    elif how == "misaligned":
        flat = torch.randn(2, n * H * D + 3, generator=g, device=dev).to(torch.float16)
        key, value = flat[0, 1:1 + n * H * D].view(n, H, D), flat[1, 3:3 + n * H * D].view(n, H, D)
    elif how == "transposed":
        both = torch.randn(2, H, n, D, generator=g, device=dev).to(torch.bfloat16)
        key, value = both[0].transpose(0, 1), both[1].transpose(0, 1)
    else:
        both = torch.randn(2, n, H, 2 * D, generator=g, device=dev).to(torch.float16)
        key, value = both[0, ..., ::2], both[1, ..., 1::2]
    slots = torch.arange(9, 9 + n, dtype=torch.int32, device=dev)
    check(filled(dev, 5, H, bs, D, 1), key, value, slots)


def test_numbers_at_the_edges(dev):
    """infinities, NaN, zeros of both signs, the largest and the smallest numbers of the type, values on the border between two scales"""
    H, D, bs = 1, 64, 16
    for dtype in (torch.bfloat16, torch.float16):
        top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        for values in ([0.0, -0.0], [float("inf"), 1.0], [float("-inf"), float("nan"), 3.0], [float("nan")], [float("inf")], [top, -top, 1.0],
                       [tiny, -tiny], [448.0], [449.0 if dtype == torch.float16 else 450.0], [1.75, 1.0], [1.7578125, -0.3], [3.5, 2.0 ** -10, 2.0 ** -12]):
            x = torch.tensor(values, dtype=dtype, device=dev).repeat(200)[:3 * H * D].view(3, H, D)
            for slots in ([0, 1, 2], [5, 6, 7]):
                check(filled(dev, 5, H, bs, D, 3), x, x.flip(0), torch.tensor(slots, dtype=torch.int32, device=dev))
                check(filled(dev, 6, H, bs, D, 3), x, x.flip(0), torch.tensor([s + 80 for s in slots], dtype=torch.int32, device=dev))


def test_what_is_read_back(dev):
    """codes times scale are within half a step of what was stored: 2^-4 of the value, or of the smallest normal number 2^-6 scale"""
    cache = odsd.KVCacheFP8.zeros(3, 2, 64, 128, dev)
    key, value = rows(dev, 100, 2, 128, torch.bfloat16, 9)
    slots = torch.arange(64, 164, dtype=torch.int32, device=dev)
    odsd.store_kvcache_fp8(key, value, cache, slots)
    k = (cache.k.float() * cache.scales[..., 0, None, None]).transpose(1, 2).flatten(0, 1)[64:164]
    v = (cache.v.float() * cache.scales[..., 1, None, None]).permute(0, 3, 1, 2).flatten(0, 1)[64:164]
    for got, want, w in ((k, key, 0), (v, value, 1)):
        scale = cache.scales[:, :, w].repeat_interleave(64, 0)[64:164, :, None]
        assert bool(((got - want.float()).abs() <= 2.0 ** -4 * torch.maximum(want.float().abs(), 2.0 ** -6 * scale)).all())
    assert bool((cache.scales[0] == 0).all())


def test_refusals(dev):
    cache = odsd.KVCacheFP8.zeros(4, 2, 16, 64, dev)
    key, value = rows(dev, 3, 2, 64, torch.bfloat16, 1)
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    C8 = odsd.KVCacheFP8
    for error, call in ((ValueError, lambda: odsd.store_kvcache_fp8(key, value[:2], cache, slots)),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key, value, cache, slots[:2])),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key, value, cache, slots, slots[:2])),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key[:, :1], value[:, :1], cache, slots)),
                        (TypeError, lambda: odsd.store_kvcache_fp8(key.float(), value.float(), cache, slots)),
                        (TypeError, lambda: odsd.store_kvcache_fp8(key, value.half(), cache, slots)),
                        (RuntimeError, lambda: odsd.store_kvcache_fp8(key, value.cpu(), cache, slots)),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key, value, C8(cache.k, cache.v, cache.scales[:3]), slots)),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key, value, C8(cache.k, cache.k, cache.scales), slots)),
                        (TypeError, lambda: odsd.store_kvcache_fp8(key, value, C8(cache.k.view(torch.uint8), cache.v, cache.scales), slots)),
                        (ValueError, lambda: odsd.store_kvcache_fp8(key, value, C8(cache.k[None], cache.v[None], cache.scales[None]), slots)),
                        (odsd._lib.OdsdError, lambda: odsd.store_kvcache_fp8(
                            key, value, C8(cache.k.view(4, 2, 8, 128)[..., :64].contiguous(), cache.v.view(4, 2, 64, 16)[..., :8].contiguous(), cache.scales), slots))):
        with pytest.raises(error):
            call()
    assert not cache.k.view(torch.uint8).any() and not cache.scales.any()
