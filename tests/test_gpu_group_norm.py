"""Group norm with an activation against its definition in 64 bits.

The tolerance counts what the kernels round: the mean and the deviation (f32
sums of deviations from a value of the map, a few steps of 2^-24 each; 16 are
allowed, times how far such a step moves the value), the activation (its
argument's error through its slope, exponentials of arguments off by a step)
and half a step of the output's type."""

import numpy as np
import pytest

import eight_bits as E
from test_gpu_eight_bits import ACTS, cuda, strided

pytestmark = pytest.mark.gpu


def tolerance(want, reach, v_max, act, dtype):
    half = 2.0**-11 if dtype == np.float16 else 2.0**-24
    return (E.SLOPE[act] * 16 * 2.0**-24 * reach + (4 + v_max) * 2.0**-23 * np.abs(want) + half * np.abs(want)
            + (2.0**-25 if dtype == np.float16 else 0) + (4 * 2.0**-23 * v_max if act == "gelu" else 2.0**-23))


def features(rng, rows, c, dtype):
    return (rng.standard_normal((rows, c)) * (0.2 + rng.random(c)) + rng.standard_normal(c)).astype(dtype)


def run(ctx, x, images, groups, gamma, beta, act, out, extra=0, eps=1e-5):
    import ien
    import torch

    y = torch.full((x.shape[0], x.shape[1] + extra), 7.0, dtype=torch.float16 if out == np.float16 else torch.float32,
                   device="cuda")
    ien.group_norm(ctx, strided(x, extra), images, groups, None if gamma is None else cuda(gamma),
                   None if beta is None else cuda(beta), y[:, :x.shape[1]], eps=eps, act=ACTS[act])
    assert bool((y[:, x.shape[1]:] == 7.0).all())
    return y[:, :x.shape[1]].cpu().numpy()


def check(ctx, x, images, groups, gamma, beta, act, out, extra=0, eps=1e-5):
    want, reach = E.group_norm(x, images, groups, gamma, beta, eps, act)
    v, _ = E.group_norm(x, images, groups, gamma, beta, eps, "none")
    got = run(ctx, x, images, groups, gamma, beta, act, out, extra, eps).astype(np.float64)
    tol = tolerance(want, reach, np.abs(v), act, out)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


# One pixel, one channel, groups of odd sizes and of one channel, channels past a workgroup's
# lanes; images of one and many pixels; rows that are no whole vectors.
SHAPES = [(1, 1, 1, 1, 0), (1, 1, 8, 1, 0), (2, 7, 36, 3, 0), (1, 9, 36, 3, 4), (3, 50, 64, 32, 0), (1, 256, 512, 32, 0),
          (2, 1000, 40, 40, 8), (1, 4096, 128, 32, 0), (2, 333, 320, 32, 0), (1, 77, 1280, 32, 0), (1, 30, 2056, 8, 0),
          (1, 5, 8192, 64, 0), (4, 1, 24, 8, 0), (1, 10625, 384, 24, 128), (1, 60000, 4, 1, 0), (1, 2500, 35, 5, 0),
          (20, 64, 96, 8, 0), (1, 20000, 96, 32, 13), (1, 1024, 512, 32, 0), (2, 900, 640, 32, 0)]


@pytest.mark.parametrize("types", [(np.float16, np.float16), (np.float16, np.float32), (np.float32, np.float16),
                                   (np.float32, np.float32)])
@pytest.mark.parametrize("images,pixels,c,groups,extra", SHAPES)
def test_group_norm(ctx, images, pixels, c, groups, extra, types):
    rng = np.random.default_rng(pixels + c)
    x = features(rng, images * pixels, c, types[0])
    gamma, beta = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32), rng.standard_normal(c).astype(np.float32)
    check(ctx, x, images, groups, gamma, beta, "silu", types[1], extra)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("pixels", [16, 5000])
def test_group_norm_activations(ctx, act, pixels):
    rng = np.random.default_rng(1)
    x = features(rng, 2 * pixels, 192, np.float16)
    for gamma, beta in ((None, None), ((3 * rng.standard_normal(192)).astype(np.float32), None),
                        (None, rng.standard_normal(192).astype(np.float32))):
        check(ctx, x, 2, 16, gamma, beta, act, np.float32)


@pytest.mark.parametrize("pixels,c,groups", [(64, 64, 8), (6000, 64, 8)])
def test_group_norm_far_means(ctx, pixels, c, groups):
    """Means thousands of deviations away, constant groups, one far value."""
    rng = np.random.default_rng(2)
    x = (1000 + 0.25 * rng.standard_normal((pixels, c))).astype(np.float32)
    x[:, 8:16] = 3.5  # a group without spread: (x - m) is 0
    x[5, 17] = 4e5
    check(ctx, x, 1, groups, None, None, "none", np.float32)
    y = run(ctx, x, 1, groups, None, None, "none", np.float32)
    assert (y[:, 8:16] == 0).all()


@pytest.mark.parametrize("pixels", [100, 9000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_group_norm_nan_stays_in_its_group(ctx, pixels, bad):
    rng = np.random.default_rng(3)
    x = features(rng, 2 * pixels, 96, np.float16)
    clean, _ = E.group_norm(x, 2, 12, None, None, 1e-5, "relu")
    x[pixels + 3, 50] = bad
    y = run(ctx, x, 2, 12, None, None, "relu", np.float32)
    hit = np.zeros(y.shape, bool)
    hit[pixels:, 48:56] = True
    assert np.array_equal(np.isnan(y), hit)
    assert np.abs(y - clean)[~hit].max() < 1e-5


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("images,pixels,c,groups,extra", [(1, 1, 8, 1, 0), (2, 7, 36, 3, 0), (1, 256, 512, 32, 0), (2, 333, 320, 32, 8),
                                                          (1, 6144, 640, 32, 0), (1, 5000, 64, 32, 0), (3, 50, 200, 8, 3),
                                                          (1, 12, 8192, 64, 0), (1, 400, 128, 32, 0), (1, 3000, 384, 32, 0)])
def test_group_norm8_is_quantize8_of_the_result(ctx, images, pixels, c, groups, extra, dtype):
    """Bit for bit the 8-bit form of the f32 result."""
    import ien
    import torch

    rng = np.random.default_rng(c)
    x = strided(features(rng, images * pixels, c, dtype), extra)
    gamma, beta = cuda((1 + 0.3 * rng.standard_normal(c)).astype(np.float32)), cuda(rng.standard_normal(c).astype(np.float32))
    y = torch.empty(images * pixels, c, device="cuda")
    want, got = ien.Rows8(images * pixels, c), ien.Rows8(images * pixels, c)
    got.data.fill_(99)
    ien.group_norm(ctx, x, images, groups, gamma, beta, y, act=ien.ACT_SILU)
    ien.quantize8(ctx, y, want)
    ien.group_norm(ctx, x, images, groups, gamma, beta, got, act=ien.ACT_SILU)
    blocks = -(-c // 128)
    assert torch.equal(got.scales[:, :blocks], want.scales[:, :blocks])
    assert torch.equal(got.data, want.data)


def test_group_norm_in_place(ctx):
    import ien
    import torch

    for rows, c in ((300, 128), (40000, 64), (256, 36)):
        x = torch.randn(rows, c, device="cuda").half()
        y = torch.empty_like(x)
        ien.group_norm(ctx, x, 1, 4, None, None, y, act=ien.ACT_GELU)
        ien.group_norm(ctx, x, 1, 4, None, None, x, act=ien.ACT_GELU)
        assert torch.equal(x, y)


def test_group_norm_other_stream_and_graph(ctx):
    import ien
    import torch

    torch.cuda.synchronize()
    xs = [torch.randn(r, c, device="cuda").half() for r, c in ((256, 512), (30000, 128))]
    want = [torch.empty_like(x) for x in xs]
    for x, y in zip(xs, want):
        ien.group_norm(ctx, x, 1, 32, None, None, y, act=ien.ACT_SILU)
    torch.cuda.synchronize()
    other, L = torch.cuda.Stream(), ien.load()
    ys = [torch.zeros_like(x) for x in xs]
    torch.cuda.synchronize()
    try:
        ien.check(L.ien_set_stream(ctx.h, other.cuda_stream))
        for x, y in zip(xs, ys):
            ien.group_norm(ctx, x, 1, 32, None, None, y, act=ien.ACT_SILU)
        other.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(ys, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=other):
            for x, y in zip(xs, ys):
                ien.group_norm(ctx, x, 1, 32, None, None, y, act=ien.ACT_SILU)
    finally:
        ien.check(L.ien_set_stream(ctx.h, None))
    for _ in range(4):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(ys, want))
        z = torch.empty_like(ys[1])
        ien.group_norm(ctx, xs[1], 1, 32, None, None, z, act=ien.ACT_SILU)
        torch.cuda.synchronize()
        assert torch.equal(z, want[1])
