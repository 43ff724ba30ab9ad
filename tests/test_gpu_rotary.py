"""apply_rotary and rotary_store_kvcache against 64 bits.

Tolerance, derived: the angle's fraction of a turn is rounded to fp32 (at most 2^-26 turns, 9.4e-8 radians), sin and cos are a
few ulp off, then a handful of fp32 roundings: 2^-20 (|x1| + |x2|) covers them (9.5e-7); the norm's scale adds 2^-21 of the
value, contained in it.  The output is rounded once: half a step of its type."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import dense_oracle as orc

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def check(got, want, size, dtype):
    e = torch.finfo(DT[dtype]).eps / 2
    inner = 2.0 ** -20 * size
    tol = inner + e * (np.abs(want) + inner) + 2.0 ** -25
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), f"error {err.max():.3e}, {(err / tol).max():.2f} of the tolerance"


def inputs(n, H, KV, D, R, dtype, axes=1, norm=False, seed=0, far=131072, pos_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, (H + 2 * KV) * D, generator=g).to(DT[dtype])
    pos = torch.randint(0, far, (axes, n), generator=g, dtype=pos_dtype)
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(DT[dtype]) for _ in range(2)) if norm else (None, None)
    return qkv, pos if axes > 1 else pos[0], inv, qw, kw


def heads(qkv, H, KV, D):
    n = qkv.shape[0]
    return qkv[:, :H * D].view(n, H, D), qkv[:, H * D:(H + KV) * D].view(n, KV, D), qkv[:, (H + KV) * D:].view(n, KV, D)


def np64(t):
    return None if t is None else t.double().cpu().numpy()


@pytest.mark.parametrize("n,H,KV,D,R,axes,sections,interleaved,norm", [
    (1, 32, 4, 128, 128, 1, None, False, True), (8, 32, 4, 128, 128, 1, None, False, False), (7, 14, 2, 64, 64, 1, None, True, True),
    (33, 14, 2, 64, 32, 1, None, True, False), (5, 3, 1, 128, 64, 1, None, False, True), (130, 32, 8, 128, 128, 3, (16, 24, 24), False, True),
    (19, 16, 16, 64, 64, 2, (8, 24), True, False), (12, 4, 4, 80, 80, 4, (10, 0, 10, 20), False, True), (9, 2, 1, 96, 48, 1, None, False, True),
    (6, 2, 2, 20, 12, 1, None, False, True), (6, 2, 1, 30, 30, 2, (7, 8), True, True), (4, 1, 1, 2, 2, 1, None, False, False),
    (3, 2, 1, 256, 256, 1, None, False, True), (3, 2, 1, 258, 130, 1, None, False, True), (2, 1, 1, 1024, 1024, 1, None, True, True),
    (1025, 8, 1, 64, 64, 3, (12, 10, 10), False, False)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_against_64_bits(dev, n, H, KV, D, R, axes, sections, interleaved, norm, dtype):
    qkv, pos, inv, qw, kw = inputs(n, H, KV, D, R, dtype, axes, norm, seed=n)
    q, k, _ = heads(qkv.to(dev), H, KV, D)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    qo, ko = odsd.apply_rotary(q, k, pos.to(dev), inv.to(dev), sections=sections, interleaved=interleaved, q_weight=on(qw), k_weight=on(kw))
    assert qo.is_contiguous() and ko.is_contiguous() and qo.dtype == q.dtype
    check(qo, *orc.rotary(np64(q), np64(pos), np64(inv), sections, interleaved, np64(qw)), dtype)
    check(ko, *orc.rotary(np64(k), np64(pos), np64(inv), sections, interleaved, np64(kw)), dtype)


@pytest.mark.parametrize("far", [1 << 20, 1 << 30])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_far_positions(dev, far, pos_dtype):
    """An angle of 2^30 radians in fp64 keeps 2^-23 of its own: the oracle's fp64 product is off by as much, 1.2e-7."""
    qkv, pos, inv, _, _ = inputs(40, 4, 2, 64, 64, "fp16", seed=3, far=far, pos_dtype=pos_dtype)
    pos[0], pos[1] = 0, far - 1
    q, k, _ = heads(qkv.to(dev), 4, 2, 64)
    qo, ko = odsd.apply_rotary(q, k, pos.to(dev), inv.to(dev))
    check(qo, *orc.rotary(np64(q), np64(pos), np64(inv)), "fp16")
    assert torch.equal(qo[0], q[0]) and torch.equal(ko[0], k[0])         # position 0 turns nothing
    neg = -pos.to(dev)
    qn, _ = odsd.apply_rotary(qo, ko, neg, inv.to(dev))
    assert (qn.float() - q.float()).abs().max() < 4 * 2.0 ** -11 * q.float().abs().max()


@pytest.mark.parametrize("n,H,KV,D,skip,dtype", [(1, 32, 4, 128, 0, "bf16"), (40, 32, 4, 128, 5, "bf16"), (63, 14, 2, 64, 9, "fp16"),
                                                 (300, 8, 1, 64, 0, "fp16"), (10, 2, 2, 20, 2, "bf16")])
@pytest.mark.parametrize("norm", [False, True])
def test_store(dev, n, H, KV, D, skip, dtype, norm):
    """Stored rows are apply_rotary's keys and the step's values, bit for bit, in their slots; every other slot stays."""
    qkv, pos, inv, qw, kw = inputs(n, H, KV, D, D, dtype, norm=norm, seed=n)
    qkv, pos, inv = qkv.to(dev), pos.to(dev), inv.to(dev)
    qw, kw = (None, None) if qw is None else (qw.to(dev), kw.to(dev))
    q, k, v = heads(qkv, H, KV, D)
    qo, ko = odsd.apply_rotary(q, k, pos, inv, q_weight=qw, k_weight=kw)
    slots_n = n + 37
    g = torch.Generator(device=dev).manual_seed(n)
    kc = torch.randn(slots_n, KV * D, generator=g, device=dev).to(DT[dtype])
    vc = torch.randn(slots_n, KV * D, generator=g, device=dev).to(DT[dtype])
    src = None
    rows = torch.arange(n, device=dev)
    if skip:
        rows = rows[rows % skip != 0]
        src = rows.to(torch.int32)
    slots = torch.randperm(slots_n, generator=g, device=dev)[:rows.numel()].to(torch.int32)
    want_k, want_v = kc.clone(), vc.clone()
    keep = torch.ones_like(rows, dtype=torch.bool)
    if rows.numel() > 4:
        slots[1], slots[3] = -1, slots_n          # no slot, and one past the cache
        keep[1] = keep[3] = False
    want_k[slots[keep].long()] = ko[rows[keep]].flatten(1)
    want_v[slots[keep].long()] = v[rows[keep]].flatten(1)
    version = kc._version
    q2 = odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, vc, slots, src, q_weight=qw, k_weight=kw)
    assert torch.equal(q2, qo) and torch.equal(kc, want_k) and torch.equal(vc, want_v) and kc._version > version
    if not skip:
        q3, k3 = odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, vc, slots, q_weight=qw, k_weight=kw, want_k=True)
        assert torch.equal(q3, qo) and torch.equal(k3, ko) and torch.equal(kc, want_k)


def test_rows_without_a_token(dev):
    """An index outside the step is not read: its slot stays as it was."""
    qkv, pos, inv, _, _ = inputs(6, 2, 1, 64, 64, "bf16")
    q, k, v = heads(qkv.to(dev), 2, 1, 64)
    kc, vc = torch.zeros(8, 64, device=dev).bfloat16(), torch.zeros(8, 64, device=dev).bfloat16()
    src = torch.tensor([0, -1, 6, 5], dtype=torch.int32, device=dev)
    odsd.rotary_store_kvcache(q, k, v, pos.to(dev), inv.to(dev), kc, vc, torch.tensor([0, 1, 2, 3], device=dev), src)
    assert vc[0].any() and vc[3].any() and not vc[1].any() and not vc[2].any() and not kc[1:3].any() and not kc[4:].any()
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    before = kc.clone()
    odsd.rotary_store_kvcache(q, k, v, pos.to(dev), inv.to(dev), kc, vc, none, none)        # nothing to store
    assert torch.equal(kc, before)


@pytest.mark.parametrize("D", [64, 20])
def test_one_token_in_several_slots(dev, D):
    """src_index names a token twice: both slots get its rows."""
    qkv, pos, inv, _, _ = inputs(6, 2, 2, D, D, "bf16")
    q, k, v = heads(qkv.to(dev), 2, 2, D)
    _, ko = odsd.apply_rotary(q, k, pos.to(dev), inv.to(dev))
    kc, vc = torch.zeros(9, 2 * D, device=dev).bfloat16(), torch.zeros(9, 2 * D, device=dev).bfloat16()
    src = torch.tensor([3, 0, 3, 3, 5, 0, 1, 2], dtype=torch.int32, device=dev)
    slots = torch.tensor([8, 1, 0, 3, 4, 5, 6, 7], dtype=torch.int32, device=dev)
    odsd.rotary_store_kvcache(q, k, v, pos.to(dev), inv.to(dev), kc, vc, slots, src)
    assert torch.equal(kc[slots.long()], ko[src.long()].flatten(1)) and torch.equal(vc[slots.long()], v[src.long()].flatten(1))
    assert not kc[2].any() and not vc[2].any()


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_unaligned_views(dev, offset):
    H, KV, D, n = 4, 2, 64, 11
    qkv, pos, inv, qw, kw = inputs(n, H, KV, D, D, "bf16", norm=True, seed=5)
    width = (H + 2 * KV) * D
    buf = torch.zeros(n, width + offset + 3, dtype=torch.bfloat16, device=dev)
    buf[:, offset:offset + width] = qkv.to(dev)
    odd = buf[:, offset:offset + width]
    q, k, v = (odd[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    a = odsd.apply_rotary(q, k, pos.to(dev), inv.to(dev), q_weight=qw.to(dev), k_weight=kw.to(dev))
    check(a[0], *orc.rotary(np64(q), np64(pos), np64(inv), weight=np64(qw)), "bf16")
    check(a[1], *orc.rotary(np64(k), np64(pos), np64(inv), weight=np64(kw)), "bf16")
    # heads in front of tokens
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(odsd.apply_rotary(qt, k, pos.to(dev), inv.to(dev))[0], odsd.apply_rotary(q.contiguous(), k, pos.to(dev), inv.to(dev))[0])
    # positions of every second token
    wide = torch.stack([pos, pos], 1).flatten().to(dev)
    assert torch.equal(odsd.apply_rotary(q, k, wide[::2], inv.to(dev))[0], odsd.apply_rotary(q, k, pos.to(dev), inv.to(dev))[0])


def test_graph(dev):
    qkv, pos, inv, qw, kw = inputs(24, 8, 2, 64, 64, "bf16", norm=True)
    qkv, pos, inv, qw, kw = (t.to(dev) for t in (qkv, pos, inv, qw, kw))
    q, k, v = heads(qkv, 8, 2, 64)
    kc, vc = torch.zeros(64, 128, device=dev).bfloat16(), torch.zeros(64, 128, device=dev).bfloat16()
    slots = torch.arange(24, device=dev, dtype=torch.int32)
    odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, vc, slots, q_weight=qw, k_weight=kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, vc, slots, q_weight=qw, k_weight=kw)
    for i in range(3):
        qkv.normal_()
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        k1 = kc.clone()
        want = odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, vc, slots, q_weight=qw, k_weight=kw)
        assert torch.equal(out, want) and torch.equal(k1, kc), i


def test_no_tokens_and_refusals(dev):
    qkv, pos, inv, qw, _ = inputs(4, 2, 1, 64, 64, "bf16", norm=True)
    q, k, v = heads(qkv.to(dev), 2, 1, 64)
    pos, inv = pos.to(dev), inv.to(dev)
    a, b = odsd.apply_rotary(q[:0], k[:0], pos[:0], inv)
    assert a.shape == (0, 2, 64) and b.shape == (0, 1, 64)
    kc = torch.zeros(8, 64, device=dev).bfloat16()
    slots = torch.zeros(4, dtype=torch.int32, device=dev)
    for call in (lambda: odsd.apply_rotary(q.float(), k.float(), pos, inv), lambda: odsd.apply_rotary(q, k, pos, inv.float()),
                 lambda: odsd.apply_rotary(q, k, pos.float(), inv)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: odsd.apply_rotary(q, k[:3], pos, inv), lambda: odsd.apply_rotary(q, k, pos[:3], inv),
                 lambda: odsd.apply_rotary(q, k, torch.stack([pos, pos]), inv), lambda: odsd.apply_rotary(q, k, torch.stack([pos, pos]), inv, sections=(16, 15)),
                 lambda: odsd.apply_rotary(q, k, pos, torch.cat([inv, inv])), lambda: odsd.apply_rotary(q, k, pos, inv, q_weight=qw.to(dev)[:32]),
                 lambda: odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, kc, slots[:3]), lambda: odsd.rotary_store_kvcache(q, k, v, pos, inv, kc.float(), kc, slots),
                 lambda: odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, kc[:, :32], slots), lambda: odsd.rotary_store_kvcache(q, k, v, pos, inv, kc, kc, slots, slots, want_k=True)):
        with pytest.raises(ValueError):
            call()
