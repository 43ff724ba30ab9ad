"""Kernels of ops.linear that the shapes of test_gpu_linear.py do not reach: packed columns and parts of K in every tile shape,
weights past the caches in each of them, packed too.  test_linear_plan.py checks on the CPU that the lists cover them."""
import pytest

from tests.test_gpu_linear import run

pytestmark = pytest.mark.gpu
# (M, K, N), small ones of their kind; nothing a multiple of a tile
PLANS = [(17, 9, 17), (5, 6208, 8109), (20, 913, 17), (17, 7741, 6500), (18, 3091, 18), (18, 2587, 18), (5, 3008, 16745), (5, 9088, 5585), (6, 5632, 8938),
         (773, 1102, 610), (22, 6139, 8221), (13, 8704, 16473), (331, 3876, 375), (65, 4928, 10217), (785, 1554, 1300), (259, 3916, 388), (65, 2752, 18298),
         (1189, 715, 1682), (115, 6779, 16771), (605, 5653, 804), (67, 8638, 5826), (136, 2944, 17124), (2340, 1135, 1823), (131, 2233, 22506),
         (130, 8064, 6243), (1287, 4737, 806), (129, 8319, 6055), (1615, 455, 2524), (585, 6483, 810), (66, 1472, 34196), (2286, 322, 3597),
         (144, 5628, 45978), (130, 5952, 8474), (1313, 6086, 1486), (129, 9212, 5509), (4465, 196, 2798), (1973, 8136, 1454), (2317, 7681, 1155), (17, 9105, 4172)]


@pytest.mark.parametrize("M,K,N", PLANS)
def test_every_kernel(dev, M, K, N):
    if M % 2:
        run(dev, M, K, N, "bf16", act="silu", seed=M)
    else:
        run(dev, M, K, N, "fp16", "fp32", act="relu", seed=M)
