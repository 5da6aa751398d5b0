"""The second product with f32 products and a branch in a captured graph, and with products
that lie past 4 GiB: whole numbers, compared for equality."""

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import cuda, rows8_of
from test_gpu_experts8 import plan_of, routed, whole_weights
from test_gpu_experts8_parts import hidden_whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,top,c,n", [(3, 4, 2, 300, 70), (250, 3, 2, 200, 130)])
def test_captured(ctx, tokens, experts, top, c, n):
    """Replays with new rows, weights and addends in the captured tensors, eager work between them."""
    import ien
    import torch

    rng = np.random.default_rng(tokens)
    index = routed(rng, tokens, experts, top)
    w = whole_weights(rng, experts, c, n)
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, np.ones((tokens, top)), experts)
    q, parts = ien.Rows8(tokens * top, c), ien.expert_parts(routes, m, torch.float32)
    x, branch, out = (torch.zeros(tokens, n, dtype=t, device="cuda") for t in (torch.float16, torch.float32, torch.float16))
    call = lambda: ien.experts_out8(ctx, q, routes, m, parts, out, add=x, branch=branch)  # noqa: E731
    q.data.zero_()
    q.scales.fill_(127)
    call()
    torch.cuda.synchronize()
    other, L, graph = torch.cuda.Stream(), ien.load(), torch.cuda.CUDAGraph()
    try:
        ien.check(L.ien_set_stream(ctx.h, other.cuda_stream))
        with torch.cuda.graph(graph, stream=other):
            call()
    finally:
        ien.check(L.ien_set_stream(ctx.h, None))
    for _ in range(4):
        v, data, scales = hidden_whole(rng, tokens * top, c)
        weight = (2.0 ** rng.integers(-1, 2, (tokens, top))).astype(np.float32)
        a, b = rng.integers(-2048, 2049, (tokens, n)), rng.integers(-2048, 2049, (tokens, n))
        q.data.copy_(cuda(data))
        q.scales[:, :scales.shape[1]].copy_(cuda(scales))
        routes.weight.copy_(cuda(weight))
        x.copy_(cuda(a.astype(np.float16)))
        branch.copy_(cuda(b.astype(np.float32)))
        y, size = X.products(v[:int(X.plan(index, experts)[0][-1])], index, w.astype(np.float64), None, False)
        assert size.max() < 2**22
        want = (X.combine(y, index, weight, experts) + a + b).astype(np.float16)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
        call()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    m.free()


def test_products_past_4_gib(ctx):
    """Two experts, every token with both; rows of zeros but the first and the last tokens'."""
    import ien
    import torch

    rng = np.random.default_rng(10)
    tokens, c, n = 1 << 17, 64, 4400
    index = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(tokens, 1)
    routes = ien.Routes(tokens, 2, 2, index=index, weight=torch.tensor([[1.0, 0.5]], device="cuda").repeat(tokens, 1))
    ien.plan_routes(ctx, routes)
    w = whole_weights(rng, 2, c, n)
    m, h = ien.Experts8(ctx, w), ien.Rows8(2 * tokens, c)
    h.data.zero_()
    h.scales.fill_(127)
    v = rng.integers(-2, 3, (4, c)).astype(np.float64)
    rows = cuda(E.to_bytes(v))
    for place, row in zip((0, tokens - 1, tokens, 2 * tokens - 1), rows):  # (expert 0's first and last, expert 1's)
        h.data[place, :c] = row
    parts = ien.expert_parts(routes, m, torch.float32)
    assert parts.numel() * 4 > 2**32
    out, branch = torch.empty(tokens, n, dtype=torch.float16, device="cuda"), torch.zeros(tokens, n, dtype=torch.float16, device="cuda")
    branch[-1] = 3.0
    ien.experts_out8(ctx, h, routes, m, parts, out, branch=branch)
    first, last = (v[i] @ w[0].astype(np.float64) + 0.5 * (v[2 + i] @ w[1].astype(np.float64)) for i in (0, 1))
    assert np.array_equal(out[0].cpu().numpy(), first.astype(np.float16))
    assert np.array_equal(out[-1].cpu().numpy(), (last + 3.0).astype(np.float16))
    assert not bool(out[1:-1].any())
    m.free()
