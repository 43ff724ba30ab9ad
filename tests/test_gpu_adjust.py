"""adjust_logits against the oracle in 64 bits.  At most 6 roundings of fp32 on the way, each half a step of the largest magnitude there, and
one to the logits' type."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def check(dev, lens, V, dtype, history=50, bias=0, mask=None, seed=0, token_dtype=torch.int64, padded=0, penalties="tensor", stride=0, in_place=False,
          context=True, wild=False):
    rng = np.random.default_rng(seed)
    S, n = len(lens), sum(lens)
    rows = n + padded
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn(rows, V + stride, generator=g, device=dev) * 4).to(dtype)[:, :V]
    lo, hi = (-3, V + 9) if wild else (0, V)
    word = lambda *shape: np.where(rng.random(shape) < 0.5, rng.integers(lo, hi, shape), rng.integers(0, min(V, 7), shape))  # noqa: E731
    tokens, drafts = word(S, history), word(sum(max(k - 1, 0) for k in lens))
    token_lens = rng.integers(0, history + 1, S)
    prompt_lens = rng.integers(0, history + 1, S) * (token_lens > 0)
    r, f, p = 1 + rng.random(S).astype(np.float32), rng.normal(size=S).astype(np.float32), rng.normal(size=S).astype(np.float32)
    if penalties == "number":
        r, f, p = np.full(S, 1.25, np.float32), np.full(S, 0.5, np.float32), np.full(S, -0.25, np.float32)
    bt, bv = word(S, bias), (rng.normal(size=(S, bias)) * 5).astype(np.float32)
    if bias:
        bt[:, bias // 2] = -1
    words = (V + 31) // 32
    masks = {"rows": rng.integers(-2 ** 31, 2 ** 31, (rows, words + 2)), "shared": rng.integers(-2 ** 31, 2 ** 31, (3, words)),
             "none": np.zeros((rows, words), np.int64)}.get(mask)
    mask_rows = rng.integers(-2, 5, rows) if mask == "shared" else None
    dv = lambda a, t: torch.tensor(a, dtype=t, device=dev)  # noqa: E731
    ctx = {"verify_query_lens": dv(lens, torch.int32), "max_query_len": max(lens)} if context else {}
    want, mag = orc.adjust(logits.double().cpu().numpy(), lens, tokens.tolist(), token_lens.tolist(), prompt_lens.tolist(), drafts.tolist(),
                           r.astype(np.float64), f.astype(np.float64), p.astype(np.float64), [list(zip(a, b)) for a, b in zip(bt.tolist(), bv.tolist())],
                           masks, mask_rows)
    out = logits if in_place else None
    given = torch.full((rows, V), 7.0, dtype=dtype, device=dev) if padded and not in_place else out
    keep = logits.clone()
    setting = (lambda a: float(a[0])) if penalties == "number" else (lambda a: dv(a, torch.float32))
    got = odsd.adjust_logits(logits, ctx, tokens=dv(tokens, token_dtype), token_lens=dv(token_lens, torch.int32), prompt_lens=dv(prompt_lens, torch.int32),
                             draft_tokens=dv(drafts, torch.int64) if context else None, repetition=setting(r), frequency=setting(f), presence=setting(p),
                             bias_tokens=dv(bt, torch.int32) if bias else None, bias_values=dv(bv, torch.float32) if bias else None,
                             mask=None if masks is None else dv(masks, torch.int64).to(torch.int32),
                             mask_rows=None if mask_rows is None else dv(mask_rows, torch.int32), out=given)
    torch.cuda.synchronize()
    assert got.dtype == dtype and got.shape == (rows, V)
    assert torch.equal(logits, keep) or in_place
    if padded:
        assert torch.equal(got[n:], keep[n:] if in_place else torch.full_like(keep[n:], 7.0))
    x, want, mag = got[:n].double().cpu().numpy(), want[:n], mag[:n]
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    fine = np.isfinite(want)
    assert np.array_equal(x[~fine], want[~fine], equal_nan=True)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    x, want, fp32 = x[fine], want[fine], 6 * 2.0 ** -24 * mag[fine]
    assert (np.abs(x - want) <= fp32 + u * (np.abs(want) + fp32) + tiny).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 31, 1000, 8192, 8193, 50257])
@pytest.mark.parametrize("lens", [[1], [5], [1, 3, 0, 9, 2]])
def test_all_of_it(dev, dtype, V, lens):
    check(dev, lens, V, dtype, history=300, bias=min(V, 9), mask="rows", seed=V)


@pytest.mark.parametrize("mask", [None, "rows", "shared", "none"])
@pytest.mark.parametrize("bias", [0, 1, 600])
def test_parts(dev, mask, bias):
    check(dev, [4, 1, 6], 3001, torch.bfloat16, bias=bias, mask=mask, seed=bias)
    check(dev, [4, 1, 6], 3001, torch.float32, bias=bias, mask=mask, seed=bias, penalties="number", in_place=True)


@pytest.mark.parametrize("history", [0, 1, 5000, 70000])
def test_histories(dev, history):
    """counts beyond what 16 bits hold, no token at all"""
    check(dev, [3, 2], 2000, torch.float32, history=history, seed=history)
    check(dev, [3, 2], 2000, torch.float32, history=history, seed=history, token_dtype=torch.int32, wild=True, bias=3)


@pytest.mark.parametrize("stride", [0, 1, 8, 13])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_apart(dev, stride, dtype):
    check(dev, [4, 1, 6], 4099, dtype, stride=stride, bias=5, mask="rows")
    check(dev, [4, 1, 6], 4096, dtype, stride=stride, bias=5, mask="rows", in_place=True)


def test_padded_and_plain_batches(dev):
    check(dev, [1, 0, 1, 1, 0], 700, torch.float16, padded=2, mask="rows")
    check(dev, [3, 0, 2], 700, torch.float16, padded=4, in_place=True, bias=2)
    check(dev, [1] * 6, 700, torch.bfloat16, context=False)
    check(dev, [2] * 300, 97, torch.float32, bias=4)
    check(dev, [1] * 64, 131072, torch.bfloat16, history=2000)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("mask", [None, "shared"])
@pytest.mark.parametrize("in_place", [False, True])
def test_many_rows_of_a_sequence(dev, dtype, mask, in_place):
    """more rows than are looked up at a time, with drafts that repeat; few and many tokens that have occurred"""
    check(dev, [130, 1, 65, 64], 1500, dtype, history=40, mask=mask, bias=3, in_place=in_place)
    check(dev, [129, 66], 9000, dtype, history=6000, mask=mask, bias=700, in_place=in_place, token_dtype=torch.int32)


def test_query_lengths_past_the_rows(dev):
    """rows and drafts past those that there are stay out of it, whatever the lengths say, and the first sequence has its own"""
    V, i32 = 300, lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    all_ = torch.randn(12, V, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    x = all_[:4]
    tokens = torch.randint(0, V, (3, 50), generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    drafts = torch.arange(2, device=dev)
    want = odsd.adjust_logits(x[:2], {"verify_query_lens": i32(2)}, tokens=tokens[:1], draft_tokens=drafts[:1], repetition=2.0, frequency=0.5)
    for told in ((2, 7, 3), (2, 2 ** 31 - 1, 2 ** 31 - 1), (2, -5, 9)):
        out = torch.full((12, V), 7.0, device=dev)
        got = odsd.adjust_logits(x, {"verify_query_lens": i32(*told)}, tokens=tokens, draft_tokens=drafts, repetition=2.0, frequency=0.5, out=out[:4])
        torch.cuda.synchronize()
        assert torch.equal(got[:2], want) and bool((out[4:] == 7.0).all())


def test_special_numbers(dev):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 3.0, nan]], device=dev)
    mask = torch.tensor([[0b0111111]], dtype=torch.int32, device=dev)
    got = odsd.adjust_logits(x, {}, tokens=torch.arange(7, device=dev)[None], repetition=2.0, mask=mask)[0].tolist()
    assert got[0] == inf and got[1] == -inf and got[2] != got[2] and got[3:6] == [0.0, 0.0, 1.5] and got[6] == -inf
    same = odsd.adjust_logits(x, {})
    assert torch.equal(same.view(torch.int32), x.view(torch.int32)) and same.data_ptr() != x.data_ptr()
    assert odsd.adjust_logits(x[:0], {}).shape == (0, 7)


def test_refusals(dev):
    x = torch.zeros(3, 40, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    ctx = {"verify_query_lens": i32(2, 1), "max_query_len": 2}
    f = odsd.adjust_logits
    for error, call in ((TypeError, lambda: f(x.double(), {})), (ValueError, lambda: f(x[0], {})), (ValueError, lambda: f(x, {}, draft_tokens=i32(1))),
                        (ValueError, lambda: f(x, {"verify_query_lens": torch.tensor([2, 2], dtype=torch.int32)})),
                        (ValueError, lambda: f(x, {"verify_query_lens": torch.tensor([2, 1], dtype=torch.int32)}, draft_tokens=i32(1, 2))),
                        (ValueError, lambda: f(x, ctx, tokens=i32(1, 2, 3)[None])), (TypeError, lambda: f(x, ctx, tokens=torch.zeros(2, 3, device=dev))),
                        (ValueError, lambda: f(x, ctx, token_lens=i32(1, 1))), (ValueError, lambda: f(x, ctx, tokens=torch.zeros(2, 3, dtype=torch.int32, device=dev), token_lens=i32(1))),
                        (ValueError, lambda: f(x, ctx, repetition=0.0)), (ValueError, lambda: f(x, ctx, repetition=float("nan"))), (ValueError, lambda: f(x, ctx, frequency=float("inf"))),
                        (ValueError, lambda: f(x, ctx, repetition=torch.ones(3, device=dev))), (ValueError, lambda: f(x, ctx, presence=torch.ones(2, device=dev).double())),
                        (ValueError, lambda: f(x, ctx, bias_tokens=i32(1, 2)[:, None])), (ValueError, lambda: f(x, ctx, bias_tokens=i32(1)[None], bias_values=torch.ones(1, 1, device=dev))),
                        (TypeError, lambda: f(x, ctx, bias_tokens=torch.zeros(2, 1, dtype=torch.int64, device=dev), bias_values=torch.ones(2, 1, device=dev))),
                        (ValueError, lambda: f(x, ctx, mask=i32(1, 2, 3)[:, None])), (ValueError, lambda: f(x, ctx, mask=i32(1, 2)[None])),
                        (ValueError, lambda: f(x, ctx, mask_rows=i32(0, 0, 0))), (ValueError, lambda: f(x, ctx, mask=i32(1, 2)[None], mask_rows=i32(0, 0))),
                        (ValueError, lambda: f(x, ctx, out=x[:2])), (ValueError, lambda: f(x, ctx, out=x.half())),
                        (ValueError, lambda: f(x, ctx, out=torch.zeros(40, 3, device=dev).t())), (RuntimeError, lambda: f(x, ctx, out=x.cpu()))):
        with pytest.raises(error):
            call()
