"""The 64-bit definitions of the dense operators, against properties they must have (CPU only)."""
import numpy as np
import pytest

from oracle import dense_oracle as orc


def test_verified_tokens_are_distributed_as_the_target():
    """What speculative sampling is for: the first token of a verified sequence follows p whatever q is.  Drafts drawn from q
    and both random numbers on a grid: the shares come out as p to the grid's width."""
    rng = np.random.default_rng(0)
    p_logits, q_logits = rng.normal(size=6), rng.normal(size=6)
    p, q = orc.distribution(p_logits, 0.7), orc.distribution(q_logits, 0.7)
    n = 40
    share = np.zeros(6)
    grid = (np.arange(n) + 0.5) / n
    logits = np.stack([p_logits, rng.normal(size=6)])
    for d in range(6):
        for u in grid:
            for r in grid:
                tok, acc, _ = orc.verify(logits, [d], [2], [u], [r], q_logits[None], 0.7)
                share[tok[0, 0]] += q[d] / (n * n)
    assert np.abs(share - p).max() < 3.0 / n


@pytest.mark.parametrize("r,want", [(0.0, 1), (0.2499, 1), (0.25, 3), (0.999, 3)])
def test_draw_takes_the_lowest_token_past_the_aim(r, want):
    assert orc.draw(np.array([0.0, 1.0, 0.0, 3.0, 0.0]), r) == want


def test_greedy_and_empty_rows():
    row = np.array([1.0, 5.0, 5.0, -np.inf])
    assert orc.distribution(row, 0.0).tolist() == [0.0, 1.0, 0.0, 0.0]
    assert orc.distribution(np.full(3, -np.inf), 1.0).sum() == 0
    assert orc.distribution(np.array([np.nan, 1.0]), 1.0).tolist() == [0.0, 1.0]
    tok, acc, a = orc.verify(np.stack([np.full(4, -np.inf), row]), [1], [2], [0.0], [0.5])
    assert tok.tolist() == [[-1, -1]] and acc.tolist() == [0] and a.tolist() == [0.0]


def test_rotary_keeps_lengths_and_turns_by_differences():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(2, 1, 16))
    f = 10000.0 ** (-np.arange(0, 8, 2) / 8)
    a, _ = orc.rotary(x, [5, 5], f)
    b, _ = orc.rotary(x, [1005, 1005], f)
    assert np.allclose((a * a).sum(-1), (x * x).sum(-1))
    assert np.allclose((a[0] * a[1]).sum(), (b[0] * b[1]).sum())          # only the difference of positions counts
    assert np.array_equal(a[..., 8:], x[..., 8:])
    c, _ = orc.rotary(x, [[5, 5], [5, 5]], f, sections=(1, 3))
    assert np.allclose(a, c)


def test_linear_epilogue_order():
    y, s, pre = orc.linear([[1.0, 2.0]], [[3.0, -4.0]], bias=[1.0], act="relu", residual=[[10.0]])
    assert y.tolist() == [[10.0]] and s.tolist() == [[11.0]] and pre.tolist() == [[-5.0]]
