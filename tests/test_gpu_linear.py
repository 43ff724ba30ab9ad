"""ops.linear against 64 bits, over the shapes, types, strides and epilogues where a product can go wrong.

Tolerance, derived: the sum takes one rounding (or truncation: a step, 2^-23) per matrix instruction of at least 16 products,
each of at most S = sum |x w|, and a few more where partial sums are joined: (K / 16 + 16) 2^-23 S.  An activation multiplies
an error by at most 1.13 (the slope of gelu and silu), adds 2e-5 of its value for 16-bit outputs (the hardware's exp2 of an
argument of up to 100) and 2^-20 for fp32.  The output is rounded once: half a step of its type."""
import numpy as np
import pytest
import torch

from on_device_sd_amd import ops
from oracle import dense_oracle as orc

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def tolerance(y, size, K, act, out):
    e = torch.finfo(DT[out]).eps / 2
    inner = 1.13 * (K / 16 + 16) * 2.0 ** -23 * (size + 1) + (2.0 ** -20 if out == "fp32" else 2e-5) * np.abs(y)
    small = torch.finfo(DT[out]).smallest_normal * e * 2
    return inner + e * (np.abs(y) + inner) + small


def run(dev, M, K, N, dtype="bf16", out=None, act=None, bias=True, residual=True, seed=0, pad=0, offset=0, scale=0.05):
    g = torch.Generator().manual_seed(seed)
    out = out or dtype
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731

    def matrix(rows, cols, t, mul=1.0):
        """rows `cols + pad` apart, the first `offset` elements into its memory, NaN around it"""
        buf = torch.full((rows * (cols + pad) + offset + 16,), float("nan"), dtype=DT[t])
        m = torch.as_strided(buf, (rows, cols), (cols + pad, 1), offset)
        m.copy_(rnd(rows, cols) * mul)
        d = buf.to(dev)
        return torch.as_strided(d, (rows, cols), (cols + pad, 1), offset), m.double().numpy()

    x, xh = matrix(M, K, dtype)
    w, wh = matrix(N, K, dtype, scale)
    b = (rnd(N) * 0.5).to(DT[dtype]) if bias else None
    r, rh = matrix(M, N, out) if residual else (None, None)
    y = ops.linear(x, w, None if b is None else b.to(dev), activation=act, residual=r, out_dtype=DT[out])
    want, size, _ = orc.linear(xh, wh, None if b is None else b.double().numpy(), act, rh)
    assert y.shape == (M, N) and y.dtype == DT[out]
    err = np.abs(y.double().cpu().numpy() - want)
    tol = tolerance(want, size, K, act, out)
    if residual:
        tol = tol + (torch.finfo(DT[out]).eps / 2 + 2.0 ** -23) * np.abs(rh)
    assert np.isfinite(err).all() and (err <= tol).all(), \
        f"M={M} K={K} N={N} {dtype}->{out} {act}: error {err.max():.3e}, {(err / tol).max():.2f} of the tolerance"


SHAPES = [(1, 2048, 4096), (1, 8, 1), (1, 1, 1), (2, 64, 16), (3, 100, 7), (5, 2048, 5120), (7, 2056, 130), (8, 4096, 2048), (15, 512, 333),
          (16, 1288, 1000), (17, 1288, 1001), (31, 640, 260), (33, 264, 515), (40, 2048, 512), (64, 2048, 1024), (64, 72, 40), (65, 512, 512),
          (100, 1000, 300), (128, 4096, 256), (129, 64, 129), (200, 512, 384), (256, 256, 256), (257, 1288, 513), (333, 1288, 2053),
          (512, 32, 512), (1000, 520, 1000), (1, 520, 40000), (20, 4096, 64), (300, 4104, 128), (700, 1536, 700),
          # the borders of the choice of kernels: tokens, rows of w, parts of K
          (4, 256, 300), (5, 256, 300), (16, 8200, 520), (33, 8192, 512), (64, 2048, 8192), (64, 2048, 8193), (48, 1032, 16384), (64, 1032, 16392),
          (32, 2056, 16640), (64, 520, 24576), (65, 4096, 512), (256, 2048, 2048), (128, 8192, 128), (2048, 256, 2048), (1500, 192, 5000)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_shapes(dev, M, K, N):
    run(dev, M, K, N, act="silu")


# every tile shape, in one part of K and in several, with edges that are no multiple of it
TILES = [(37, 72, 72), (18, 2168, 85), (67, 2888, 1173), (1341, 3008, 79), (19, 72, 65), (28, 6296, 5539), (14, 3800, 2822), (17, 2584, 1206),
         (24, 64, 16930), (33, 4368, 8795), (7, 5008, 4990), (8, 7536, 2495), (38, 72, 8198), (77, 3368, 1037), (33, 7872, 1034), (72, 72, 8460),
         (83, 4496, 4222), (198, 6072, 1032), (69, 8288, 1321), (134, 64, 9036), (218, 5216, 4446), (67, 5496, 4701), (143, 728, 17065),
         (139, 4152, 9634), (134, 4808, 6065), (2316, 7120, 194), (133, 64, 18196), (66, 5200, 9058), (229, 9016, 2126), (258, 80, 22286),
         (622, 64, 16930), (5433, 344, 2113), (35, 3392, 2317), (18, 72, 8309), (5, 6296, 4790), (17, 3736, 1080), (33, 7240, 4410),
         (35, 4648, 2232), (67, 392, 4290), (133, 6296, 1054), (72, 6056, 2231), (75, 3944, 1085), (151, 64, 8799), (65, 6592, 8199),
         (67, 6576, 4446), (143, 968, 18257), (134, 3688, 11100), (158, 5144, 5560), (478, 8920, 1122), (137, 72, 18111), (195, 6304, 4171),
         (133, 7600, 2787), (132, 4544, 5737), (404, 64, 22868), (140, 1104, 16903), (1353, 3872, 110), (111, 2880, 332), (6, 8888, 4382),
         (16, 9048, 4574), (4267, 6848, 153), (129, 4904, 8293), (17, 2592, 78)]


@pytest.mark.parametrize("M,K,N", TILES)
def test_tile_shapes(dev, M, K, N):
    run(dev, M, K, N, "fp16", act="relu")


@pytest.mark.parametrize("M,K,N", [(12, 8192, 8000), (20, 12288, 4300), (40, 2048, 25700), (60, 4096, 12900), (100, 2048, 25700), (120, 4096, 12900),
                                   (190, 2048, 25700), (190, 1024, 51300)])
def test_weights_of_more_than_96_mb_in_one_pass(dev, M, K, N):
    """they are read past the caches"""
    run(dev, M, K, N, "bf16", "fp32")


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("M,K,N", [(37, 136, 72), (19, 72, 65), (24, 72, 16930), (38, 72, 8198), (72, 72, 8460), (134, 64, 9036), (143, 728, 17065),
                                   (133, 64, 18196), (258, 80, 22286), (622, 64, 16930), (18, 72, 8309), (67, 392, 4290), (143, 968, 18257),
                                   (137, 72, 18111), (140, 1104, 16903)])
def test_tile_shapes_of_every_type(dev, M, K, N, dtype, out):
    run(dev, M, K, N, dtype, out, "gelu_tanh", seed=M)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M", [1, 24, 150, 600])
def test_types_and_activations(dev, M, act, dtype, out):
    run(dev, M, 512, 520, dtype, out, act, seed=M)
    run(dev, M, 256, 320, dtype, out, act, bias=False, residual=False, seed=M + 1, scale=0.4)


@pytest.mark.parametrize("M,K,N", [(1, 2049, 65), (4, 333, 100), (16, 1111, 514), (50, 777, 201), (130, 513, 260), (400, 1027, 300),
                                   (20, 3809, 700), (300, 2999, 520), (70, 2047, 9000), (257, 9, 257), (600, 4100, 1030)])
def test_odd_columns(dev, M, K, N):
    run(dev, M, K, N, "bf16")
    run(dev, M, K, N, "fp16", "fp32", "gelu")


@pytest.mark.parametrize("M", [1, 20, 90, 520])
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (3, 0), (1, 1), (0, 2), (0, 1), (64, 4)])
def test_strides_and_alignment(dev, M, pad, offset):
    run(dev, M, 264, 200, "bf16", "bf16", "relu", pad=pad, offset=offset)
    run(dev, M, 264, 200, "fp16", "fp32", None, pad=pad, offset=offset)


@pytest.mark.parametrize("M", [1, 30, 300])
def test_values_at_the_edges(dev, M):
    """Subnormals, the largest values of fp16, infinities and NaN reach their own outputs only."""
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, 256, generator=g).half()
    w = (torch.randn(200, 256, generator=g) * 0.05).half()
    x[0] *= 2.0 ** -14                       # products of subnormals
    w[3] = 0
    w[3, 5] = 60000.0                        # 60000 x: past fp16 for some rows, fine in fp32
    w[7, 9] = float("inf")
    w[8, 10] = float("nan")
    y = ops.linear(x.to(dev), w.to(dev), out_dtype=torch.float32).cpu().double()
    ref = x.double() @ w.double().t()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(y[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
    size = x.double().abs() @ w.double().abs().t()
    assert ((y - ref).abs()[fine] <= (32 * 2.0 ** -23 * size + 2.0 ** -24 * ref.abs())[fine]).all()
    ok = torch.ones(200, dtype=torch.bool)
    ok[7:9] = False
    assert torch.isfinite(y[:, ok]).all()


def test_same_bits_every_time_and_in_a_graph(dev):
    for M, K, N in [(1, 4096, 2048), (40, 2048, 512), (300, 1024, 256), (600, 512, 1024)]:
        g = torch.Generator(device=dev).manual_seed(1)
        x = torch.randn(M, K, generator=g, device=dev).bfloat16()
        w = torch.randn(N, K, generator=g, device=dev).bfloat16()
        y = ops.linear(x, w, activation="silu")
        for _ in range(3):
            assert torch.equal(ops.linear(x, w, activation="silu"), y)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.linear(x, w, activation="silu")
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            z = ops.linear(x, w, activation="silu")
        for k in range(3):
            x.normal_(generator=g)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(z, ops.linear(x, w, activation="silu")), (M, k)


def test_two_calls_at_once(dev):
    """Calls on two streams, of the forms with a workspace (parts of K; packed columns), have workspaces of their own."""
    for M, K, N in [(64, 8192, 2048), (300, 4097, 2000)]:
        g = torch.Generator(device=dev).manual_seed(9)
        xs = [torch.randn(M, K, generator=g, device=dev).bfloat16() for _ in range(2)]
        w = torch.randn(N, K, generator=g, device=dev).bfloat16()
        alone = [ops.linear(x, w) for x in xs]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
        for _ in range(8):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(ops.linear(xs[i], w))
        torch.cuda.synchronize()
        for want, ys in zip(alone, got):
            assert all(torch.equal(y, want) for y in ys)


def test_the_output_may_be_the_residual_of_the_next_call(dev):
    """Calls one after the other on one stream share freed workspaces in order: a chain equals its steps."""
    g = torch.Generator(device=dev).manual_seed(10)
    x = torch.randn(48, 8192, generator=g, device=dev).half()
    w = torch.randn(1024, 8192, generator=g, device=dev).half() / 90
    y = torch.zeros(48, 1024, device=dev).half()
    steps = []
    for _ in range(5):
        y = ops.linear(x, w, residual=y, activation="relu")
        steps.append(y)
    once = ops.linear(x, w, activation="relu", out_dtype=torch.float32)
    want = torch.zeros(48, 1024, device=dev).half()
    for y in steps:                                     # the sums of every call are the same bits; one rounding a call
        want = (once + want.float()).half()
        assert torch.equal(y, want)


def test_leading_dimensions_single_rows_and_empty(dev):
    w = torch.randn(24, 64, device=dev).half()
    x = torch.randn(2, 3, 64, device=dev).half()
    assert torch.equal(ops.linear(x, w).view(6, 24), ops.linear(x.view(6, 64), w))
    # one row is another kernel than six, with another order of the sum: both within the tolerance of the exact row
    one, of_six = ops.linear(x[0, 0], w), ops.linear(x.view(6, 64), w)[0]
    want, size, _ = orc.linear(x[0, :1].double().cpu().numpy(), w.double().cpu().numpy())
    for y in (one, of_six):
        assert y.shape == (24,) and (np.abs(y.double().cpu().numpy() - want[0]) <= tolerance(want, size, 64, None, "fp16")[0]).all()
    col = torch.randn(64, 1, device=dev).half()
    assert torch.equal(ops.linear(col.t(), w), ops.linear(col.t().clone(), w))       # one row, strides (1, 1)
    assert ops.linear(x[:, :0], w).shape == (2, 0, 24)
    assert torch.equal(ops.linear(x.transpose(0, 1), w), ops.linear(x.transpose(0, 1).contiguous(), w))
    assert torch.equal(ops.linear(x[0, :1].expand(5, 64), w), ops.linear(x[0, :1].repeat(5, 1), w))


def test_rows_far_apart(dev):
    """Rows 2^21 elements apart and more do not fit the tiles' 32-bit offsets: another kernel takes them."""
    g = torch.Generator(device=dev).manual_seed(2)
    far = torch.randn(70, 1 << 21, generator=g, device=dev, dtype=torch.float16)
    x, w = far[:, :256], torch.randn(96, 256, generator=g, device=dev).half()
    assert torch.equal(ops.linear(x[:3], w), ops.linear(x[:3].clone(), w))
    for a, b in ((x, w), (w, x)):
        y, z = ops.linear(a, b, out_dtype=torch.float32).double(), a.double() @ b.double().t()
        assert ((y - z).abs() <= 32 * 2.0 ** -23 * (a.double().abs() @ b.double().abs().t())).all()


def test_refusals(dev):
    x, w = torch.randn(4, 64, device=dev).half(), torch.randn(8, 64, device=dev).half()
    for bad in (lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.bfloat16()), lambda: ops.linear(x, w, w[0, :8].float()),
                lambda: ops.linear(x, w, out_dtype=torch.bfloat16)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.linear(x[:, :32], w), lambda: ops.linear(x[:, :0], w[:, :0]), lambda: ops.linear(x, w, x[0, :7]), lambda: ops.linear(x, w, activation="tanh"),
                lambda: ops.linear(x, w, residual=x[:, :7]), lambda: ops.linear(x, w, residual=x[:, :8].float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.linear(x, w.cpu())
