"""The experts' second product with its products in f32 under f16 results, and with a
branch beside the residual.

Whole numbers as in test_gpu_experts8: sums in f32 are exact, so an f16 result is the
sum rounded once, compared for equality.  Real ones: f32 products as there (no
rounding of theirs to f16), and one rounding of the result, 2^-11."""

import ctypes

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import cuda, rows8_of, strided
from test_gpu_experts8 import plan_of, routed, whole_weights

pytestmark = pytest.mark.gpu

# tokens, experts, top, depth, outputs: few rows an expert (two depths), tiles of 64 and of 128 rows.
SIZES = [(3, 4, 2, 300, 70), (2, 3, 2, 2100, 37), (250, 3, 2, 200, 130), (1500, 2, 1, 140, 200), (33, 8, 3, 96, 129)]


def hidden_whole(rng, pairs, c):
    v = np.where(rng.random((pairs, c)) < min(1.0, 60 / c), rng.integers(-2, 3, (pairs, c)), 0).astype(np.float64)
    return v, E.to_bytes(np.concatenate([v, np.zeros((pairs, -c % 128))], 1)), np.full((pairs, -(-c // 128)), 127, np.uint8)


@pytest.mark.parametrize("tokens,experts,top,c,n", SIZES)
@pytest.mark.parametrize("exact", [True, False])
def test_products_past_f16(ctx, tokens, experts, top, c, n, exact):
    """Products of up to 2^18 under weights of 2^-8 and 2^-9: the results are f16's, the products are not."""
    import ien
    import torch

    rng = np.random.default_rng(tokens + n)
    v, data, scales = hidden_whole(rng, tokens * top, c)
    index, weight = routed(rng, tokens, experts, top), 2.0 ** rng.integers(-9, -7, (tokens, top))
    w = whole_weights(rng, experts, c, n) * 4096
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, experts)
    y, size = X.products(v[:int(X.plan(index, experts)[0][-1])], index, w.astype(np.float64), None, False)
    assert 65504 < size.max() < 2**24 and np.abs(y).max() > 65504
    want = X.combine(y, index, weight, experts)
    assert np.abs(want).max() < 65504
    out = torch.empty(tokens, n, dtype=torch.float16, device="cuda")
    ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, ien.expert_parts(routes, m, torch.float32), out, exact=exact)
    assert np.array_equal(out.cpu().numpy(), want.astype(np.float16))
    m.free()


@pytest.mark.parametrize("tokens,experts,top,c,n", SIZES)
@pytest.mark.parametrize("dtype,branch_dtype,parts", [(np.float16, np.float16, "f32"), (np.float16, np.float32, "f32"), (np.float16, np.float16, "f16"),
                                                      (np.float32, np.float16, "f32"), (np.float32, np.float32, "f32")])
@pytest.mark.parametrize("over", [None, "add", "branch", "alone"])
def test_a_branch(ctx, tokens, experts, top, c, n, dtype, branch_dtype, parts, over):
    """The residual's two addends: up to 2^13, so that their sum in f16 would be off by up to two.  In place of either; a
    branch without a residual."""
    import ien
    import torch

    if over == "branch" and dtype != branch_dtype:
        return  # (in place of rows of another type: not asked for)
    rng = np.random.default_rng(tokens + 5 * n)
    v, data, scales = hidden_whole(rng, tokens * top, c)
    index, weight = routed(rng, tokens, experts, top), 2.0 ** rng.integers(-1, 2, (tokens, top))
    w = whole_weights(rng, experts, c, n)
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, experts)
    y, size = X.products(v[:int(X.plan(index, experts)[0][-1])], index, w.astype(np.float64), None, False)
    assert size.max() <= 2048
    whole = lambda: rng.integers(-2048, 2049, (tokens, n)) * 2.0 ** rng.integers(0, 3, (tokens, n))  # noqa: E731
    a, b = whole().astype(dtype), whole().astype(branch_dtype)
    want = X.combine(y, index, weight, experts) + b.astype(np.float64) + (0 if over == "alone" else a.astype(np.float64))
    add, branch = strided(a, 3), strided(b, 2)
    out = {"add": add, "branch": branch}.get(over, strided(np.zeros((tokens, n), dtype), 5, 7.0))
    extra = out.stride(0) - n if tokens > 1 else 0
    products = ien.expert_parts(routes, m, torch.float16 if parts == "f16" else torch.float32)
    ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, products, out, add=None if over == "alone" else add, branch=branch)
    assert np.array_equal(out.cpu().numpy(), want.astype(dtype))
    if over in (None, "alone") and extra:
        assert bool((torch.as_strided(out, (tokens, n + extra), (n + extra, 1))[:, n:] == 7.0).all())
    m.free()


@pytest.mark.parametrize("tokens,experts,top,c,n", SIZES)
@pytest.mark.parametrize("exact", [True, False])
def test_f32_products_of_real_numbers(ctx, tokens, experts, top, c, n, exact):
    import ien
    import torch

    rng = np.random.default_rng(tokens * n + c)
    data, scales = E.quantize(rng.standard_normal((tokens * top, c)))
    index, weight = routed(rng, tokens, experts, top), rng.random((tokens, top)).astype(np.float32)
    w = (rng.standard_normal((experts, c, n)) / np.sqrt(c)).astype(np.float32)
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, experts)
    out = torch.empty(tokens, n, dtype=torch.float16, device="cuda")
    ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, ien.expert_parts(routes, m, torch.float32), out, exact=exact)
    y, size = X.products(E.values(data, scales, c), index, X.weights(w), None, False)
    off = (2.0**-23 * c if exact else 2.0**-10) * size + 2.0**-24 * np.abs(y)
    want, off = X.combine(y, index, weight, experts), X.combine(off, index, weight, experts)
    size = X.combine(np.abs(y), index, weight, experts)
    off = off + 2.0**-24 * (top + 1) * size
    assert (np.abs(out.cpu().numpy() - want) <= off + 2.0**-11 * (np.abs(want) + off) + 2.0**-25).all()
    m.free()


def test_the_entry_point_without_a_branch(ctx):
    """ien_experts_out8 is the other with products of the result's type."""
    import ien
    import torch

    rng = np.random.default_rng(11)
    v, data, scales = hidden_whole(rng, 80, 200)
    index, weight = routed(rng, 40, 4, 2), rng.random((40, 2)).astype(np.float32)
    m, routes = ien.Experts8(ctx, whole_weights(rng, 4, 200, 60)), plan_of(ctx, index, weight, 4)
    q = rows8_of(data, scales, 200)
    for dtype, kind in ((torch.float16, ien.OUT_F16), (torch.float32, ien.OUT_F32)):
        parts, add = ien.expert_parts(routes, m, dtype), torch.randn(40, 60, device="cuda").to(dtype)
        want, got = torch.empty(40, 60, dtype=dtype, device="cuda"), torch.empty(40, 60, dtype=dtype, device="cuda")
        ien.experts_out8(ctx, q, routes, m, parts, want, add=add)
        ien.check(ien.load().ien_experts_out8(ctx.h, q._at, routes._at, m.h, 0, parts.data_ptr(), add.data_ptr(), 60,
                                              ctypes.byref(ien.Output(got.data_ptr(), 60, ien.NHWC, kind))))
        assert torch.equal(got, want)
    m.free()


@pytest.mark.parametrize("tokens,c,hidden,experts,top,gated", [(1, 128, 64, 4, 2, True), (50, 96, 200, 8, 3, False), (333, 136, 256, 6, 2, True),
                                                             (700, 387, 100, 20, 4, False)])
def test_the_block_rounds_once(ctx, tokens, c, hidden, experts, top, gated):
    """An f16 stream and branch give what the same values in f32 give, rounded."""
    import torch

    from test_gpu_expert_mlp import block_of, weights_of

    rng = np.random.default_rng(tokens + 1)
    block = block_of(ctx, weights_of(rng, c, hidden, experts, gated), c, top, gated)
    x, add = (cuda(rng.standard_normal((tokens, c)).astype(np.float16)) for _ in range(2))
    for a in (add, None):
        want = block.run(x.float(), add=None if a is None else a.float())
        assert torch.equal(block.run(x, add=a), want.half())
        assert torch.equal(block.run(x.float(), add=a), want)
        for out in ("x", "add") if a is not None else ("x",):
            xt, at = x.clone(), None if a is None else a.clone()
            got = block.run(xt, add=at, out=xt if out == "x" else at)
            assert torch.equal(got, want.half())
    block.free()
