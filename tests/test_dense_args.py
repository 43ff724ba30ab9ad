"""Refusals of the dense entry points that need no GPU: status codes before anything is launched, errors for CPU tensors."""
import ctypes as C

import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import _lib, ops

P = 1 << 20


def test_linear_status_codes():
    lib = _lib.load()
    f = lambda M=4, N=16, K=64, ldx=64, ldw=64, ldr=16, ldo=16, x=P, w=P, res=None, out=P, dt=1, odt=1, act=0, ws=P, nb=1 << 30: \
        lib.odsd_linear(x, ldx, w, ldw, None, res, ldr, out, ldo, M, N, K, dt, odt, act, ws, nb, None)  # noqa: E731
    assert f(M=-1) == f(N=0) == f(K=0) == f(ldx=63) == f(ldw=63) == f(ldo=15) == f(res=P, ldr=15) == 2
    assert f(dt=0) == f(dt=9) == f(odt=2) == f(odt=9) == 7
    assert f(act=5) == f(act=-1) == 3 and f(M=5_000_000) == 3
    assert f(x=None) == f(w=None) == f(out=None) == 1
    split = dict(M=40, N=512, K=8192, ldx=8192, ldw=8192, ldo=512)             # parts of K: a workspace is needed
    assert lib.odsd_linear_workspace_bytes(40, 512, 8192) > 256 and f(ws=None, **split) == 1 and f(nb=256, **split) == 5
    assert f(x=P + 1) == f(out=P + 1) == f(odt=0, out=P + 2) == f(ws=P + 8) == 4
    assert f(M=0, x=None, out=None) == 0
    assert lib.odsd_linear_workspace_bytes(4, 16, 0) == 0 and lib.odsd_linear_workspace_bytes(4, 16, 64) >= 256


def test_rotary_status_codes():
    lib = _lib.load()
    def f(n=4, H=4, KV=2, D=64, R=64, dt=1, pb=8, axes=1, sec=None, q=P, q_out=P, k_out=P, kc=None, vc=None, slots=None, src=None,
          ns=0, v=P, pos=P, inv=P):
        s = None if sec is None else (C.c_int32 * len(sec))(*sec)
        return lib.odsd_rotary(q, H * D, D, P, KV * D, D, v, KV * D, D, n, H, KV, D, R, 0, dt, pos, pb, axes, n, s, inv, None, None,
                               1e-6, q_out, k_out, kc, vc, slots, src, ns, 64, None)
    assert f(n=-1) == f(H=0) == f(R=66) == f(R=3) == f(D=65) == f(axes=0) == 2
    assert f(axes=2) == f(axes=2, sec=(16, 17)) == f(axes=2, sec=(16, 15)) == f(axes=2, sec=(33, -1)) == 2
    assert f(axes=5, sec=(32, 0, 0, 0, 0)) == 3 and f(D=2048, R=64) == 3
    assert f(dt=0) == f(pb=2) == 7
    assert f(q=None) == f(q_out=None) == f(pos=None) == f(inv=None) == f(k_out=None) == 1
    assert f(kc=P, slots=P, ns=4) == f(kc=P, vc=P, ns=4) == f(kc=P, vc=P, v=None, slots=P, ns=4) == 1
    assert f(kc=P, vc=P, slots=P, ns=3) == f(ns=4) == 2                # rows and tokens differ without an index; nothing to store to
    assert f(kc=P, vc=P, slots=P, src=P, ns=3) == 3                    # every key is wanted, but only some are computed
    assert f(q=P + 1) == f(pos=P + 4) == f(inv=P + 4) == 4
    assert f(n=0, q=None) == 0


def test_verify_status_codes():
    lib = _lib.load()
    f = lambda S=2, mq=3, rows=6, nd=4, V=100, ld=100, dl=None, ldd=100, dt=0, dr=P, ql=P, t=None, ta=1.0, au=P, su=P, tok=P, ws=P, nb=1 << 30, x=P: \
        lib.odsd_verify_drafts(x, ld, dl, ldd, dt, dr, ql, t, ta, au, su, S, mq, rows, nd, V, tok, P, P, ws, nb, None)  # noqa: E731
    assert f(S=-1) == f(V=0) == f(ld=99) == f(dl=P, ldd=99) == f(ta=-1.0) == f(ta=float("nan")) == 2
    assert f(dt=3) == 7 and f(S=70000) == 3
    assert f(x=None) == f(dr=None) == f(ql=None) == f(au=None) == f(su=None) == f(tok=None) == f(ws=None) == 1
    assert f(x=P + 2) == f(ws=P + 4) == f(dt=1, x=P + 1) == 4
    assert f(nb=16) == 5
    assert f(S=0) == f(mq=0) == 0
    ws = lib.odsd_verify_workspace_bytes
    assert ws(2, 3, 6, 4, 100, 1) >= 256 and ws(2, 3, 6, 4, 0, 1) == 0 and ws(2, 3, 6, 4, 2 ** 31 - 1, 1) == 0
    assert ws(64, 9, 576, 512, 131072, 1) > ws(64, 9, 576, 512, 131072, 0)


def test_launches_of_too_many_threads_are_refused():
    """2^32 threads and more, before anything is launched."""
    lib = _lib.load()
    n = 1 << 26
    assert lib.odsd_linear_workspace_bytes(1, n, 64) == 0
    assert lib.odsd_linear(P, 64, P, 64, None, None, n, P, n, 1, n, 64, 1, 1, 0, P, 1 << 30, None) == 3
    for n, heads in ((1 << 24, 4), (4, 1 << 27)):
        assert lib.odsd_rotary(P, heads * 20, 20, P, 40, 20, P, 40, 20, n, heads, 2, 20, 20, 0, 1, P, 8, 1, n, None, P, None, None, 1e-6, P, P,
                               None, None, None, None, 0, 64, None) == 3
    assert lib.odsd_verify_workspace_bytes(2, 3, 1 << 24, 4, 100, 0) == 0
    assert lib.odsd_verify_workspace_bytes(2, 3, 1 << 20, 4, 131072, 0) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    f = torch.zeros(32, dtype=torch.float64)
    for call in (lambda: ops.linear(x, x), lambda: odsd.apply_rotary(q, q, torch.zeros(2, dtype=torch.int64), f),
                 lambda: odsd.verify_drafts(x, None, {}, None, torch.zeros(2))):
        with pytest.raises(RuntimeError):
            call()
