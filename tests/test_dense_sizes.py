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
