"""Sizes at the ends of the dense operators' ranges: what a kernel could not count is refused before anything is launched."""
from on_device_sd_amd import _lib

P = 1 << 20                                     # an aligned address; every call here ends before anything could read it


def test_rotary_rows_of_values_that_31_bits_cannot_step_over():
    """A workgroup steps through a token's values 256 at a time: its counter passes the last by up to 255."""
    lib = _lib.load()
    for kv_heads, D in ((2 ** 30 - 1, 2), (2 ** 30 - 100, 2), ((2 ** 31 - 2) // 6, 6)):
        assert lib.odsd_rotary(P, D, D, P, kv_heads * D, D, P, kv_heads * D, D, 1, 1, kv_heads, D, D, 0, 1, P, 8, 1, 1, None, P, None, None, 1e-6, P,
                               None, P, P, P, None, 1, 64, None) == 3


def test_verify_token_rows_that_31_bits_cannot_step_over():
    lib = _lib.load()
    for longest in (2 ** 31 - 1, 2 ** 31 - 256):
        assert lib.odsd_verify_workspace_bytes(1, longest, 1, 0, 100, 0) == 0
        assert lib.odsd_verify_drafts(P, 100, None, 100, 0, None, None, None, 1.0, None, P, 1, longest, 1, 0, 100, P, P, None, P, 1 << 30, None) == 3
    assert lib.odsd_verify_workspace_bytes(1, 2 ** 31 - 257, 1, 0, 100, 0) >= 256


def test_linear_workspace_query_answers_0_where_the_call_refuses():
    lib = _lib.load()
    for M, N, K in ((64 * 65535 + 1, 16, 64), (5_000_000, 7, 9), (2 ** 31 - 1, 16, 64), (4, 2 ** 31 - 1, 64), (4, 2 ** 31 - 256, 8), (4, 16, 2 ** 31 - 1),
                    (100, 16, 2 ** 31 - 256)):
        assert lib.odsd_linear(P, K, P, K, None, None, N, P, N, M, N, K, 1, 1, 0, P, 1 << 40, None) == 3, (M, N, K)
        assert lib.odsd_linear_workspace_bytes(M, N, K) == 0, (M, N, K)
    assert lib.odsd_linear_workspace_bytes(64 * 65535, 16, 64) >= 256
