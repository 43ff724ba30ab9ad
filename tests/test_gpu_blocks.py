"""copy_cache_blocks and BlockPool on the GPU: every byte of the caches, copied or not."""
import pytest
import torch

import on_device_sd_amd as odsd

pytestmark = pytest.mark.gpu


def some_bytes(dev, shape, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, shape[:-1] + (shape[-1] * size,), generator=g, device=dev, dtype=torch.uint8).view(dtype)


def as_bytes(t):
    return t.contiguous().view(torch.uint8).clone()


def check(caches, src, dst, block_dim, tables=None, give=None):
    before = [as_bytes(c) for c in caches]
    names = None if tables is None else tables.cpu()
    odsd.copy_cache_blocks(give or caches, src, dst, block_dim, tables)
    torch.cuda.synchronize()
    src, dst = [int(b) for b in src], [int(b) for b in dst]
    for c, want in zip(caches, before):
        if block_dim:
            want[:, dst] = want[:, src]
        else:
            want[dst] = want[src]
        assert torch.equal(as_bytes(c), want)
    if tables is not None:
        moved = dict(zip(src, dst))
        assert tables.flatten().tolist() == [moved.get(b, b) for b in names.flatten().tolist()]


@pytest.mark.parametrize("pairs", [1, 7, 200, 384, 385, 900])
@pytest.mark.parametrize("row, dtype", [(512, torch.bfloat16), (1, torch.float32), (3, torch.int8), (5, torch.float16), (4100, torch.bfloat16), (9000, torch.uint8),
                                        (8191, torch.uint8), (8194, torch.uint8)])
def test_sizes(dev, pairs, row, dtype):
    """blocks from 3 bytes to several workgroups, any alignment, more pairs than a launch has"""
    nb = 2 * pairs + 5
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(pairs))
    caches = [some_bytes(dev, (nb, row), dtype, 1), some_bytes(dev, (nb, 2, row), dtype, 2)]
    check(caches, order[:pairs].tolist(), order[pairs:2 * pairs].to(torch.int32), 0)


@pytest.mark.parametrize("layers", [1, 3, 48])
def test_a_models_cache(dev, layers):
    """all layers of an 8-bit cache, block tables behind it"""
    nb, pairs = 50, 20
    cache = odsd.KVCacheFP8.zeros(nb, 2, 16, 64, dev, layers=layers)
    for t in (cache.k, cache.v, cache.scales):
        t.view(torch.uint8).random_(0, 256)
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(layers))
    tables = torch.randint(-1, nb, (7, 33), dtype=torch.int32, device=dev)
    check([cache.k, cache.v, cache.scales], order[:pairs], order[pairs:2 * pairs], 1, tables, give=[cache])
    layer = cache.layer(layers - 1)
    check([layer.k, layer.v, layer.scales], [3], [4], 0, give=[layer])


def test_more_tensors_than_a_launch_has(dev):
    caches = [some_bytes(dev, (9, 16 + i), torch.uint8, i) for i in range(37)]
    tables = torch.arange(-1, 9, dtype=torch.int32, device=dev)
    check(caches, [8, 0], [1, 2], 0, tables)


def test_one_source_for_several(dev):
    check([some_bytes(dev, (9, 4, 128), torch.bfloat16, 1)], [3, 3, 5], [0, 1, 2], 0)
    check([some_bytes(dev, (2, 9, 4, 128), torch.bfloat16, 1)], [], [], 1)


def test_views_off_alignment(dev):
    flat = some_bytes(dev, (9 * 32 + 7,), torch.uint8, 1)
    for at in (1, 2, 4, 7):
        check([flat[at:at + 9 * 32].view(9, 32)], [0, 1], [7, 8], 0)


def test_refusals(dev):
    c = some_bytes(dev, (9, 4, 128), torch.bfloat16, 1)
    before = as_bytes(c)
    t = torch.zeros(4, dtype=torch.int32, device=dev)
    f = odsd.copy_cache_blocks
    for error, call in ((ValueError, lambda: f([c], [0, 1], [2])), (ValueError, lambda: f([c], [0], [9])), (ValueError, lambda: f([c], [-1], [2])),
                        (ValueError, lambda: f([c], [0, 1], [2, 2])), (ValueError, lambda: f([c], [0, 1], [1, 2])), (ValueError, lambda: f([c], [3], [3])),
                        (ValueError, lambda: f([], [0], [1])), (ValueError, lambda: f([c, c[:8]], [0], [1])), (ValueError, lambda: f([c.transpose(1, 2)], [0], [1])),
                        (ValueError, lambda: f([c], [0], [1], 2)), (ValueError, lambda: f([c], [0, 0], [1, 2], 0, t)), (ValueError, lambda: f([c], [0], [1], 0, t.long())),
                        (TypeError, lambda: f([c], t[:1], [1])), (TypeError, lambda: f([c], torch.tensor([0.0]), [1])), (RuntimeError, lambda: f([c, c.cpu()], [0], [1]))):
        with pytest.raises(error):
            call()
    assert torch.equal(as_bytes(c), before)


def test_pool_copies_on_write_and_compacts(dev):
    """what the sequences' slots hold stays what was written there"""
    nb, bs, H, D, L = 24, 16, 2, 64, 3
    cache = odsd.KVCacheFP8.zeros(nb, H, bs, D, dev, layers=L)
    pool = odsd.BlockPool(nb, bs, [cache], block_dim=1)
    g = torch.Generator(device=dev).manual_seed(1)

    def write(seqs, counts):
        pool.append(seqs, counts)
        slots = torch.tensor([x for s, c in zip(seqs, counts) for x in s.get_slot_mapping(s.num_tokens - c, c)], dtype=torch.int32, device=dev)
        for i in range(L):
            key, value = (torch.randn(len(slots), H, D, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
            odsd.store_kvcache_fp8(key, value, cache.layer(i), slots)

    def read(seq):
        at = torch.tensor(seq.get_slot_mapping(0, seq.num_tokens), device=dev)
        k = cache.k.float() * cache.scales[..., 0, None, None]
        v = cache.v.float() * cache.scales[..., 1, None, None]
        return k[:, at // bs, :, at % bs].clone(), v[:, at // bs, :, :, at % bs].clone()

    def same(a, b):
        return all(torch.equal(x, y) for x, y in zip(a, b))

    a, b = odsd.SequenceSlots(bs), odsd.SequenceSlots(bs)
    write([b, a], [33, 41])
    f = pool.fork(a)
    was_a, was_b = read(a), read(b)
    assert same(read(f), was_a)
    write([a, f], [1, 2])
    keep = lambda r, n: (r[0][:n], r[1][:n])  # noqa: E731
    # (the copy's new row may have raised the scale of the block, so rows there are compared up to its last step)
    for got in (read(a), read(f)):
        assert same(keep(got, 32), keep(was_a, 32)) and all(torch.allclose(x[32:41], y[32:], rtol=2 ** -3, atol=2.0 ** -9) for x, y in zip(got, was_a))
    assert same(read(b), was_b)
    pool.free(b)
    tables = torch.tensor([s.get_block_table(6) for s in (a, f)], dtype=torch.int32, device=dev)
    now = read(a), read(f)
    assert pool.compact([a, f], tables)
    assert same(read(a), now[0]) and same(read(f), now[1]) and max(a.block_table + f.block_table) == nb - pool.num_free - 1
    assert tables.tolist() == [s.get_block_table(6) for s in (a, f)]
