"""Which kernels the product's GPU tests run, asked of the library (no GPU): every combination of tile, parts of K, packed
columns and weights past the caches that a size can lead to has a shape in their lists, whatever the estimates behind the choice."""
import ctypes as C
import math
import random

from on_device_sd_amd import _lib
from tests.test_gpu_linear import SHAPES, TILES
from tests.test_gpu_linear_plans import PLANS

_plan = (C.c_int32 * 7)()


def plan(M, K, N, ldx=None, ldw=None, aligned=1):
    rc = _lib.load().odsd_linear_plan(M, N, K, ldx or K, ldw or K, aligned, _plan)
    return tuple(_plan) if rc == 0 else rc


def kind(p):
    return p[:4] + (p[4] > 1, p[5] > 0, p[6])


def _sizes(n):
    """Of two sorts: anything up to 8192 tokens, and weights of 96 MB and a little more in one pass, their rows whole lines."""
    rng = random.Random(20)
    log = lambda a, b: round(math.exp(rng.uniform(math.log(a), math.log(b))))  # noqa: E731
    for i in range(n):
        if i % 2:
            K = log(4, 144) * 64 - (rng.randrange(8) if rng.random() < 0.7 else 0)
            yield log(1, 192), K, int(((96 << 19) // ((K + 7) // 8 * 8) + 1) * rng.uniform(1, 1.3))
        else:
            M, K, N = log(1, 8192), log(8, 9216), log(16, 131072)
            yield M, K // 8 * 8 if rng.random() < 0.5 else K, N


def test_the_lists_cover_every_kernel():
    tested = {kind(plan(*s)) for s in SHAPES + TILES + PLANS}
    missing = {}
    for s in _sizes(400_000):
        k = kind(plan(*s))
        if k not in tested:
            missing.setdefault(k, s)
    assert not missing, f"(kernel, n, m, shares, parts, packed, past the caches): a shape that no list has: {missing}"
    assert len({k[:4] for k in tested if k[0] == 2}) == 10


def test_the_lists_of_one_kernel_each_are_of_several():
    """what the shapes that were added stand for"""
    kinds = [kind(plan(*s)) for s in PLANS]
    assert len(set(kinds)) == len(kinds)


def test_alignment_and_far_rows_change_the_plan():
    assert plan(100, 512, 512)[0] == 2 and plan(100, 512, 512, aligned=0)[:3] == (1, 64, 64)
    assert plan(100, 512, 512, ldx=513)[0] == plan(100, 512, 512, ldw=1 << 21)[0] == 1
    assert plan(3, 512, 512)[0] == plan(16, 512, 512, aligned=0)[0] == 0
    assert plan(300, 4097, 2000)[5] == 4104


def test_plan_refusals():
    for sizes in ((0, 8, 8), (4, 0, 8), (4, 8, 0), (-1, 8, 8)):
        assert plan(*sizes) == 2
    assert plan(4, 64, 64, ldx=63) == plan(4, 64, 64, ldw=63) == 2
    assert plan(5_000_000, 8, 8) == plan(4, 2 ** 31 - 1, 8) == plan(1, 64, 1 << 26) == 3
    assert _lib.load().odsd_linear_plan(4, 8, 8, 8, 8, 1, None) == 1


def test_a_plan_asks_for_the_workspace_that_the_query_answers():
    """256 where nothing is split or packed; else the parts' sums and the packed operands"""
    up = lambda b: (b + 255) // 256 * 256  # noqa: E731
    for M, K, N in SHAPES + TILES + PLANS:
        p = plan(M, K, N)
        sums = p[4] * M * ((N + 7) // 8 * 8) * 4 if p[4] > 1 else 0
        want = up(sums) + up(M * p[5] * 2) + up(N * p[5] * 2) if p[5] else sums
        assert _lib.load().odsd_linear_workspace_bytes(M, N, K) == max(want, 256), (M, K, N)
