"""The norm, the router and the experts' products run together: the block of
expert_mlp.py against its steps in 64 bits, its command, and runs in a captured
graph, on other streams and of two contexts.

Values next to a border of e4m3 may fall on its other side (f32 sums), which moves
them by a sixteenth: the result is compared by its norm, 2^-10 for those, and 2^-11
each for the stream's, the parts' and the result's f16."""

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import cuda

pytestmark = pytest.mark.gpu


def weights_of(rng, c, hidden, experts, gated):
    n = hidden * (2 if gated else 1)
    f = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    return dict(gamma=1 + 0.2 * f(c), router=((f(c, experts) / np.sqrt(c)).astype(np.float16), 0.2 * f(experts)),
                first=(f(experts, c, n) / np.sqrt(c).astype(np.float32), 0.3 * f(experts, n)),
                second=(f(experts, hidden, c) / np.sqrt(hidden).astype(np.float32), 0.3 * f(experts, c)))


def block_of(ctx, w, c, top, gated, **kw):
    from expert_mlp import ExpertMlp8

    return ExpertMlp8(ctx, c, top, cuda(w["gamma"]), w["router"], w["first"], w["second"], gated=gated, **kw)


@pytest.mark.parametrize("tokens,c,hidden,experts,top,gated", [(1, 128, 64, 4, 2, True), (50, 96, 200, 8, 3, False), (333, 136, 256, 6, 2, True),
                                                             (1500, 64, 130, 2, 1, True), (700, 387, 100, 20, 4, False)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_block(ctx, tokens, c, hidden, experts, top, gated, dtype):
    import ien
    import torch

    rng = np.random.default_rng(tokens)
    w = weights_of(rng, c, hidden, experts, gated)
    act = "silu" if gated else "gelu"
    offset = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    how = dict(score=ien.SCORE_SIGMOID, bias=cuda(offset), scale=2.5)
    block = block_of(ctx, w, c, top, gated, act=ien.ACT_SILU if gated else ien.ACT_GELU, how=how)
    x, add = (rng.standard_normal((tokens, c)).astype(dtype) for _ in range(2))
    xt, at = cuda(x), cuda(add)
    y = block.run(xt, add=at)
    assert y.dtype == xt.dtype
    first = y.clone()
    assert torch.equal(block.run(xt, add=at, out=torch.empty_like(xt)), first)
    _, _, logits, routes, _, _ = block._work[tokens, xt.dtype]
    s = x.astype(np.float32) + add.astype(np.float32)
    n = X.rms_norm(s, w["gamma"], block.eps)
    # The router's product has f16 operands: its logits, and the choice of its own.
    want = n.astype(np.float16).astype(np.float64) @ w["router"][0].astype(np.float64) + w["router"][1]
    assert np.abs(logits.cpu().numpy() - want).max() <= 2.0**-9 * np.abs(n).max()
    index, weight = X.route(logits.cpu().numpy(), top, False, bias=offset, scale=2.5)
    assert np.array_equal(routes.index.cpu().numpy(), index)
    v, _ = X.products(E.values(*E.quantize(n), c), index, X.weights(w["first"][0]), w["first"][1].astype(np.float64), True)
    h = E.values(*E.quantize(X.gate(v, act, gated)), hidden)
    v, _ = X.products(h, index, X.weights(w["second"][0]), w["second"][1].astype(np.float64), False)
    want = s + X.combine(v, index, weight, experts)
    assert np.linalg.norm(first.double().cpu().numpy() - want) <= (2.0**-10 + 3 * 2.0**-11) * np.linalg.norm(want)
    # In place of the stream, and without a branch.
    whole = cuda((x + add).astype(dtype))
    other = block.run(whole.clone())
    assert torch.equal(block.run(whole, out=whole), other)
    assert block.run(xt[:0]).shape == (0, c)
    block.free()


def test_the_command(ctx, capsys):
    """Three operands in 8 bits in a row are off by at most a sixteenth of themselves, evenly spread: some 6%."""
    import expert_mlp
    import torch

    assert expert_mlp.main(500, 128, 96, 8, 2) < 0.1
    assert "us a block" in capsys.readouterr().out
    assert torch.cuda.current_stream() == ctx.stream  # (the command's own context left it as it was)


@pytest.mark.parametrize("sizes", [(24, 300, 7), (900, 30, 64)])
def test_graphs(ctx, sizes):
    """Two captured runs of other sizes and an eager one in turns: each replay equals the eager result, with new
    inputs in the captured tensors and other work between them."""
    import ien
    import torch

    rng = np.random.default_rng(3)
    w = weights_of(rng, 96, 160, 6, True)
    block, check = block_of(ctx, w, 96, 2, True), block_of(ctx, w, 96, 2, True)
    xs = [cuda(rng.standard_normal((t, 96)).astype(np.float16)) for t in sizes]
    ys = [torch.zeros_like(x) for x in xs]
    for x, y in zip(xs, ys):
        block.run(x, out=y)
    torch.cuda.synchronize()
    other, L, graphs = torch.cuda.Stream(), ien.load(), []
    try:
        ien.check(L.ien_set_stream(ctx.h, other.cuda_stream))
        for x, y in list(zip(xs, ys))[:2]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=other):
                block.run(x, out=y)
    finally:
        ien.check(L.ien_set_stream(ctx.h, None))
    for turn in range(4):
        for x in xs:
            x.copy_(cuda(rng.standard_normal(tuple(x.shape)).astype(np.float16)))
        want = [check.run(x) for x in xs]
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        block.run(xs[2], out=ys[2])
        torch.cuda.synchronize()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        for y, z in zip(ys, want):
            assert torch.equal(y, z)
    block.free()
    check.free()


def test_two_contexts_at_once():
    """Blocks of two contexts, each on its own stream, in flight together."""
    import ien
    import torch

    rng = np.random.default_rng(4)
    contexts = [ien.Context(0), ien.Context(0)]
    ws = [weights_of(rng, 128, 256, 8, True) for _ in contexts]
    blocks = [block_of(c, w, 128, 2, True) for c, w in zip(contexts, ws)]
    xs = [cuda(rng.standard_normal((2000, 128)).astype(np.float16)) for _ in contexts]
    want = []
    for b, x in zip(blocks, xs):
        want.append(b.run(x))
        torch.cuda.synchronize()
    ys = [torch.zeros_like(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, x, y in zip(blocks, xs, ys):
            b.run(x, out=y)
    torch.cuda.synchronize()
    for y, z in zip(ys, want):
        assert torch.equal(y, z)
    for b, c in zip(blocks, contexts):
        b.free()
        c.close()


def test_blocks_that_do_not_fit_are_refused(ctx):
    rng = np.random.default_rng(5)
    w = weights_of(rng, 64, 96, 4, True)
    with pytest.raises(ValueError):
        block_of(ctx, w, 64, 2, False)
    with pytest.raises(ValueError):
        block_of(ctx, dict(w, router=(w["router"][0][:, :3], None)), 64, 2, True)
