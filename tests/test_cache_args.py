"""Refusals of the 8-bit cache, block copies and logit adjustment that need no GPU: status codes before anything is launched, errors
for CPU tensors; and the books that a pool of blocks keeps."""
import random

import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import _lib

P = 1 << 20


def test_store_status_codes():
    lib = _lib.load()
    f = lambda N=4, n=4, H=2, D=64, bs=16, nb=8, dt=1, key=P, val=P, k=P, v=P, sc=P, slots=P, src=None, st=128, ws=P, b=1 << 30: \
        lib.odsd_kv_store_fp8(key, st, D, val, st, D, k, v, sc, slots, src, N, n, H, D, bs, nb, dt, ws, b, None)  # noqa: E731
    assert f(N=-1) == f(n=-1) == f(H=0) == f(D=0) == f(bs=0) == f(bs=24) == f(nb=-1) == f(N=3) == 2
    assert f(dt=0) == f(dt=3) == 7
    assert f(D=96) == f(bs=1040) == f(nb=1 << 27) == f(nb=1 << 26, H=64) == f(N=1 << 29, n=1 << 29) == 3
    assert f(key=None) == f(val=None) == f(k=None) == f(v=None) == f(sc=None) == f(slots=None) == 1
    assert f(k=P + 8) == f(v=P + 1) == f(sc=P + 4) == f(key=P + 1) == 4
    many = dict(N=5000, n=5000)
    assert f(ws=None, **many) == 1 and f(ws=P + 2, **many) == 4 and f(b=256, **many) == 5
    size = lib.odsd_kv_store_fp8_workspace_bytes
    assert size(0) == size(4096) == 256 and size(4097) > 256 and size(-1) == size(1 << 29) == 0
    assert f(N=0, n=0, key=None) == f(nb=0, k=None) == f(N=0, src=P, key=None) == 0


def test_attention_status_codes():
    lib = _lib.load()
    f = lambda S=2, mq=3, H=8, KV=2, D=64, bs=16, mb=4, nb=8, scale=0.1, dt=1, q=P, k=P, v=P, sc=P, bt=P, cl=P, out=P, ws=P, n=1 << 30, T=6: \
        lib.odsd_paged_attention_fp8(q, k, v, sc, bt, cl, None, T, S, mq, H, KV, D, bs, mb, nb, scale, dt, out, ws, n, None)  # noqa: E731
    assert f(T=-1) == f(S=-1) == f(mq=0) == f(H=7) == f(KV=0) == f(bs=8) == f(mb=0) == f(nb=0) == f(scale=0.0) == f(scale=float("nan")) == f(scale=float("inf")) == 2
    assert f(dt=0) == f(dt=5) == 7
    assert f(D=96) == f(bs=1040) == f(nb=1 << 30) == f(mq=1 << 21) == f(S=1 << 28) == f(S=1 << 20, mq=1024) == 3
    assert f(q=None) == f(k=None) == f(v=None) == f(sc=None) == f(bt=None) == f(cl=None) == f(out=None) == f(mb=400, ws=None) == 1
    assert f(q=P + 8) == f(k=P + 8) == f(v=P + 8) == f(sc=P + 4) == f(out=P + 4) == f(mb=400, ws=P + 8) == 4
    assert f(mb=400, n=16) == 5
    assert f(S=0, q=None) == f(T=0, q=None) == 0 and f(S=0, D=96) == 3
    size = lib.odsd_paged_attention_fp8_workspace_bytes
    assert size(2, 3, 8, 2, 64, 16, 4) == 256 and size(2, 3, 8, 2, 64, 16, 400) > 256
    assert size(2, 3, 8, 2, 96, 16, 4) == size(2, 3, 8, 2, 64, 24, 4) == size(0, 3, 8, 2, 64, 16, 4) == size(1 << 28, 3, 8, 2, 64, 16, 4) == 0


def test_copy_status_codes():
    import ctypes as C
    lib = _lib.load()

    def f(tensors=(P,), bytes_=(64,), step=(640,), layers=(1,), n=None, src=(1,), dst=(2,), nb=10, bt=None, ne=0, pairs=None):
        k = len(tensors)
        a = lambda t, v: None if v is None else (t * len(v))(*v)  # noqa: E731
        return lib.odsd_copy_blocks(a(C.c_void_p, tensors), a(C.c_int64, bytes_), a(C.c_int64, step), a(C.c_int32, layers), k if n is None else n,
                                    a(C.c_int32, src), a(C.c_int32, dst), len(src or dst or ()) if pairs is None else pairs, nb, bt, ne, None)
    assert f(n=-1) == f(pairs=-1) == f(nb=-1) == f(ne=-1) == f(bytes_=(0,)) == f(layers=(-1,)) == f(layers=(2,), step=(639,)) == 2
    assert f(src=(10,)) == f(src=(-1,)) == f(dst=(10,)) == f(dst=(-1,)) == 2
    assert f(n=17) == f(bytes_=(1 << 31,)) == f(ne=1 << 32, bt=P) == 3
    assert f(src=None) == f(dst=None) == f(bytes_=None) == f(tensors=(None,)) == 1
    assert f(pairs=0) == f(n=0) == 0


def test_adjust_status_codes():
    lib = _lib.load()

    def f(x=P, ld=100, out=P, ldo=100, dt=0, rows=6, V=100, ql=P, S=2, tok=P, tb=8, ts=5, mt=5, dr=P, nd=4, r=1.0, fr=0.0, pr=0.0, bt=P, bv=P, nb=3,
          mask=P, ms=4, nm=6):
        return lib.odsd_adjust_logits(x, ld, out, ldo, dt, rows, V, ql, S, tok, tb, ts, mt, None, None, dr, nd, None, r, None, fr, None, pr, bt, bv, nb,
                                      mask, ms, nm, None, None)
    nan = float("nan")
    assert f(rows=-1) == f(V=0) == f(S=-1) == f(mt=-1) == f(nd=-1) == f(nb=-1) == f(nm=-1) == f(ld=99) == f(ldo=99) == f(ts=4) == f(ms=3) == 2
    assert f(ql=None) == f(r=0.0) == f(r=nan) == f(r=-1.0) == f(r=float("inf")) == f(fr=nan) == f(pr=float("inf")) == 2
    assert f(dt=3) == f(tb=2) == 7
    assert f(S=1 << 23, V=65536, ld=65536, ldo=65536, ms=2048) == 3
    assert f(x=None) == f(out=None) == f(dr=None) == f(bt=None) == f(bv=None) == 1
    assert f(x=P + 2) == f(out=P + 1, dt=1) == f(tok=P + 4) == f(dr=P + 4) == f(mask=P + 2) == 4
    assert f(rows=0, x=None) == f(S=0, x=None) == 0


def test_cpu_tensors_are_refused():
    cache = odsd.KVCacheFP8.zeros(4, 2, 16, 64, device="cpu")
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    context = {"block_tables": torch.zeros(2, 1, dtype=torch.int32), "context_lens": torch.ones(2, dtype=torch.int32)}
    for call in (lambda: odsd.store_kvcache_fp8(x, x, cache, torch.zeros(2, dtype=torch.int32)),
                 lambda: odsd.paged_attention_fp8(x, cache, context),
                 lambda: odsd.attention_for_context(x, x, x, cache, None, context, 2, 16),
                 lambda: odsd.copy_cache_blocks([cache], [0], [1]),
                 lambda: odsd.adjust_logits(torch.zeros(2, 9), {})):
        with pytest.raises(RuntimeError):
            call()
    for bad in ((4, 2, 24, 64), (4, 2, 16, 96), (4, 2, 2048, 64)):
        with pytest.raises(ValueError):
            odsd.KVCacheFP8.zeros(*bad, device="cpu")


# ---- the pool's books (no caches: nothing is copied) ---------------------------------------------------
def _tokens(pool, seq):
    assert len(seq.block_table) == -(-seq.num_tokens // pool.block_size)
    return [seq.block_table[p // pool.block_size] * pool.block_size + p % pool.block_size for p in range(seq.num_tokens)]


def test_pool_fork_writes_and_frees():
    pool = odsd.BlockPool(8, 4)
    a = odsd.SequenceSlots(4)
    pool.append([a], [6])
    assert a.block_table == [0, 1] and pool.num_free == 6
    b = pool.fork(a)
    assert b.block_table == a.block_table and b.block_table is not a.block_table and pool.holders[:2] == [2, 2] and pool.num_free == 6
    pool.append([a, b], [1, 1])                  # the first to write gets a copy, the other keeps the block
    assert a.block_table == [0, 2] and b.block_table == [0, 1] and pool.holders[:3] == [2, 1, 1]
    pool.append([a], [2])
    assert a.block_table == [0, 2, 3] and a.num_tokens == 9
    c = pool.fork(a)
    pool.append([c], [0])                        # nothing is written, nothing is copied
    assert c.block_table == a.block_table
    pool.truncate(a, 7)
    assert a.block_table == [0, 2] and pool.holders[3] == 1
    pool.free(c)
    assert pool.holders == [2, 1, 1, 0, 0, 0, 0, 0] and c.block_table == [] and c.num_tokens == 0
    full = odsd.SequenceSlots(4)
    pool.append([full], [4])
    twin = pool.fork(full)
    pool.append([full, twin], [1, 1])            # a full block is never written again: it stays shared
    assert full.block_table[0] == twin.block_table[0] and full.block_table[1] != twin.block_table[1]


def test_pool_refusals_change_nothing():
    pool = odsd.BlockPool(3, 4)
    a = odsd.SequenceSlots(4)
    pool.append([a], [7])
    b = pool.fork(a)
    before = (list(pool.holders), pool.num_free, list(a.block_table), a.num_tokens)
    with pytest.raises(RuntimeError):
        pool.append([a, b], [5, 1])              # a copy and a new block: one is free
    for call in (lambda: pool.append([a], [-1]), lambda: pool.append([a, a], [1, 1]), lambda: pool.append([a], [1, 2]),
                 lambda: pool.append([odsd.SequenceSlots(8)], [1]), lambda: pool.truncate(a, 8), lambda: pool.truncate(a, -1),
                 lambda: pool.fork(odsd.SequenceSlots(4, [2], 3)), lambda: pool.compact([a]),
                 lambda: pool.append([odsd.SequenceSlots(4, [0], 9)], [1])):
        with pytest.raises(ValueError):
            call()
    assert before == (list(pool.holders), pool.num_free, list(a.block_table), a.num_tokens)
    pool.append([a], [1])
    assert a.block_table == [0, 2] and b.block_table == [0, 1]


def test_pool_compacts():
    pool = odsd.BlockPool(10, 4)
    seqs = [odsd.SequenceSlots(4) for _ in range(4)]
    pool.append(seqs, [8, 9, 4, 5])
    assert pool.num_free == 2
    seqs.append(pool.fork(seqs[1]))
    pool.free(seqs.pop(0))
    pool.free(seqs.pop(1))
    moved = pool.compact(seqs)
    held = {b for s in seqs for b in s.block_table}
    assert held == set(range(pool.num_blocks - pool.num_free)) and all(old not in held for old in moved)
    assert sorted(pool._free) == list(range(len(held), 10)) and pool.compact(seqs) == {}
    new = odsd.SequenceSlots(4)
    pool.append([new], [1])
    assert new.block_table == [len(held)]


def test_pool_random_walk():
    """what any two sequences share is what they shared when one was forked off the other"""
    rng = random.Random(4)
    pool, live, text = odsd.BlockPool(40, 4), [], {}
    store = {}                                   # slot -> token written there
    for step in range(600):
        do = rng.random()
        if do < 0.15 or not live:
            live.append(odsd.SequenceSlots(4))
            text[id(live[-1])] = []
        elif do < 0.6:
            some = rng.sample(live, rng.randint(1, len(live)))
            counts = [rng.randint(0, 5) for _ in some]
            tables = {id(s): list(s.block_table) for s in some}
            before = {id(s): _tokens(pool, s) for s in some}
            try:
                pool.append(some, counts)
            except RuntimeError:
                assert all(tables[id(s)] == s.block_table for s in some)
                pool.free(live.pop(rng.randrange(len(live))))
                continue
            for s in some:                       # the copies that the pool would make
                for old, new in zip(before[id(s)], _tokens(pool, s)):
                    store[new] = text[id(s)][_tokens(pool, s).index(new)]
            for s, c in zip(some, counts):
                for slot in _tokens(pool, s)[s.num_tokens - c:]:
                    store[slot] = step * 100 + rng.randint(0, 99)
                    text[id(s)].append(store[slot])
        elif do < 0.75:
            s = rng.choice(live)
            live.append(pool.fork(s))
            text[id(live[-1])] = list(text[id(s)])
        elif do < 0.85:
            s = rng.choice(live)
            n = rng.randint(0, s.num_tokens)
            pool.truncate(s, n)
            del text[id(s)][n:]
        elif do < 0.92:
            i = rng.randrange(len(live))
            pool.free(live.pop(i))
        else:
            moved = pool.compact(live)
            for old, new in moved.items():
                for o in range(4):
                    store[4 * new + o] = store.pop(4 * old + o, None)
        for s in live:
            assert [store[x] for x in _tokens(pool, s)] == text[id(s)]
        assert pool.num_free == pool.holders.count(0) == len(pool._free)
        assert sum(pool.holders) == sum(len(s.block_table) for s in live)


def test_rows_half_alike():
    from on_device_sd_amd.verify import _half_alike
    buf = torch.zeros(20, 50)
    a = buf[:8, :20]
    for b, alike in ((a, False), (buf[8:16, :20], False), (buf[:8, 20:40], False), (buf[:8, 30:], False), (buf[1:9, :20], True), (buf[:8, 19:39], True),
                     (buf[:8, 10:30], True), (buf.view(-1)[:160].view(8, 20), True), (buf[::2][:8, :20], True), (torch.zeros(8, 20), False),
                     (buf.view(-1)[800:960].view(8, 20), False), (buf.view(-1)[35:435].view(8, 50)[:, :20], True)):
        assert _half_alike(a, b) == alike == _half_alike(b, a), (b.shape, b.stride(), b.storage_offset())
    assert not _half_alike(buf[:1, :20], buf[:1, 20:40]) and _half_alike(buf[:1, :20], buf[:1, 1:21]) and not _half_alike(a[:0], buf[:0, 1:21])
