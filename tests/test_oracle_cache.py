"""The 8-bit cache's oracle against torch's own conversion and against a second way of writing the definitions."""
import numpy as np
import torch

from oracle import cache_oracle as orc


def test_codes_are_torchs():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(every, orc.E4M3, equal_nan=True)
    rng = np.random.default_rng(0)
    half_way = (orc.E4M3[:126] + orc.E4M3[1:127]) / 2
    y = np.concatenate([rng.uniform(-448, 448, 20000), rng.normal(0, 0.01, 20000), half_way, -half_way, orc.E4M3[:127], [0.0, -0.0]]).astype(np.float32)
    assert np.array_equal(torch.tensor(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), orc.e4m3_codes(y))
    assert orc.e4m3_codes([np.inf, -np.inf, np.nan, 1e9]).tolist() == [126, 254, 127, 126]


def test_scales_are_the_smallest_that_fit():
    for e in range(-60, 100, 7):
        assert orc.block_scale(448 * 2.0 ** e) == 2.0 ** e and orc.block_scale(448.0001 * 2.0 ** e) == 2.0 ** (e + 1)
    assert orc.block_scale(0.0) == orc.block_scale(1e-30) == 2.0 ** -64


def test_a_scale_that_rises_changes_normal_codes_exactly():
    rng = np.random.default_rng(1)
    codes = orc.e4m3_codes(rng.uniform(1, 448, 1000))
    for k in (1, 3, 6):
        again = orc.e4m3_codes(orc.E4M3[codes] * 2.0 ** -k)
        assert np.array_equal(orc.E4M3[again] * 2.0 ** k, orc.E4M3[codes])


def test_attention_is_a_softmax():
    rng = np.random.default_rng(2)
    nb, H, bs, D, L, ql = 5, 2, 16, 64, 37, 3
    k, v = rng.integers(0, 127, (nb, H, bs, D)).astype(np.uint8), rng.integers(0, 127, (nb, H, D, bs)).astype(np.uint8)
    scales = 2.0 ** rng.integers(-9, -5, (nb, H, 2))
    q = rng.normal(size=(ql, 4, D))
    got, _, _ = orc.attend(q, k, v, scales, np.array([[3, 1, 4]]), [L], [ql], 0.1)
    kk, vv = (torch.tensor(t).repeat_interleave(2, 0) for t in orc.gathered(k, v, scales, [3, 1, 4], L))
    mask = torch.ones(ql, L, dtype=torch.bool).tril(L - ql)
    want = torch.nn.functional.scaled_dot_product_attention(torch.tensor(q).transpose(0, 1), kk, vv, attn_mask=mask, scale=0.1)
    assert np.allclose(got, want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-12)


def test_adjustment_by_hand():
    x = np.array([[2.0, -2.0, 4.0, 1.0], [2.0, -2.0, 4.0, 1.0]])
    got, _ = orc.adjust(x, [2], [[0, 1, 1, 9]], [4], [1], [2], [2.0], [0.5], [0.25], [[(3, 7.0), (3, 1.0)]], np.array([[0b1011], [-1]]))
    # the prompt is token 0; output 1 and 1; the draft in front of the second row is token 2
    assert got.tolist() == [[1.0, -4.0 - 1.25, -np.inf, 2.0], [1.0, -5.25, 2.0 - 0.75, 2.0]]
