"""The residual block at changing sizes, in a captured graph, and on f32 maps."""

import numpy as np
import pytest

import eight_bits as E

pytestmark = pytest.mark.gpu

C, GROUPS = 64, 8


def parts(seed):
    rng = np.random.default_rng(seed)
    convs = [((rng.standard_normal((9 * C, C)) / np.sqrt(9 * C)).astype(np.float32), rng.standard_normal(C).astype(np.float32))
             for _ in range(2)]
    gains = [((1 + 0.2 * rng.standard_normal(C)).astype(np.float32), rng.standard_normal(C).astype(np.float32))
             for _ in range(2)]
    return rng, convs, gains


def block_of(ctx, convs, gains):
    import torch

    from residual_block import ResidualBlock8

    return ResidualBlock8(ctx, C, GROUPS, [tuple(torch.from_numpy(g).cuda() for g in p) for p in gains], convs)


def test_graph_at_one_size_and_runs_at_others(ctx):
    """Each replay equals the eager result, with eager runs of other sizes and
    new tensors between them."""
    import ien
    import torch

    rng, convs, gains = parts(1)
    block = block_of(ctx, convs, gains)
    sizes = [(20, 30), (40, 50), (10, 12)]
    xs = [torch.from_numpy(rng.standard_normal((h * w, C)).astype(np.float16)).cuda() for h, w in sizes]
    want = [block_of(ctx, convs, gains).run(x, 1, *s) for x, s in zip(xs, sizes)]
    y = torch.zeros_like(xs[0])
    block.run(xs[0], 1, *sizes[0], y)
    torch.cuda.synchronize()
    other, L = torch.cuda.Stream(), ien.load()
    try:
        ien.check(L.ien_set_stream(ctx.h, other.cuda_stream))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=other):
            block.run(xs[0], 1, *sizes[0], y)
    finally:
        ien.check(L.ien_set_stream(ctx.h, None))
    kept = []
    for _ in range(4):
        for x, s, w in zip(xs[1:], sizes[1:], want[1:]):
            assert torch.equal(block.run(x, 1, *s), w)
        kept += [torch.full((n, C), 3.0, dtype=torch.float16, device="cuda") for n in (120, 600, 2000)]
        kept += [torch.full((n, 128), 9, dtype=torch.uint8, device="cuda") for n in (120, 600, 2000)]
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0])
        assert torch.equal(block.run(xs[0], 1, *sizes[0]), want[0])
        assert all(bool((t == (3 if t.dtype == torch.float16 else 9)).all()) for t in kept)
    block.free()


@pytest.mark.parametrize("images,h,w", [(1, 9, 14), (2, 24, 20)])
def test_f32_maps(ctx, images, h, w):
    """As the f16 maps of test_gpu_residual_block: values next to a border of e4m3
    may fall on its other side, 2^-10 of the result's norm, and the map between
    the halves is f16, 2^-11."""
    import torch

    rng, convs, gains = parts(2)
    x = rng.standard_normal((images * h * w, C)).astype(np.float32)
    block = block_of(ctx, convs, gains)
    y = block.run(torch.from_numpy(x).cuda(), images, h, w)
    assert y.dtype == torch.float32

    def half(v, gain, conv):
        n, _ = E.group_norm(v, images, GROUPS, *gain, 1e-5, "silu")
        return E.patches(E.values(*E.quantize(n), C), images, h, w, 1) @ E.weights(conv[0], 9) + conv[1]

    want = x.astype(np.float64) + half(half(x, gains[0], convs[0]).astype(np.float16), gains[1], convs[1])
    assert np.linalg.norm(y.double().cpu().numpy() - want) <= (2.0**-11 + 2.0**-10) * np.linalg.norm(want)
    block.free()
