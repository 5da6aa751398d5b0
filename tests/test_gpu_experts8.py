"""The experts' products in 8 bits against their definitions in 64 bits.

Products of small whole numbers under power-of-two scales are exact in f32 whatever
the order of the sums: what they give is compared for equality, rows in 8 bits bit
for bit.  Of real numbers, a value before its rounding is off by one step of f32 for
each sum, 2^-23 k times the sum of the products' magnitudes, times the activation's
steepest slope (and, gated, the other factor); rounding to 8 bits moves it by half a
step, 2^-4 of it or 2^-10 of its block's scale; to f16 by 2^-11."""

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import ACTS, cuda, rows8_of, strided, whole_rows

pytestmark = pytest.mark.gpu


def routed(rng, tokens, experts, top, none=0.1, one=False):
    """Distinct random experts a token, some pairs without one; `one`: mostly the same expert."""
    index = np.argsort(rng.random((tokens, experts)), 1)[:, :top].astype(np.int32)
    if one:
        index[:, 0] = experts // 2
    index[rng.random((tokens, top)) < none] = -1
    return index


def plan_of(ctx, index, weight, experts):
    import ien

    r = ien.Routes(*index.shape[:1], experts, index.shape[1], index=cuda(index), weight=cuda(weight.astype(np.float32)))
    ien.plan_routes(ctx, r)
    return r


def whole_weights(rng, experts, c, n):
    return rng.integers(-3, 4, (experts, c, n)).astype(np.float32)


# tokens, experts, top, c, hidden: means of one row to thousands, odd and ragged sizes.
SIZES = [(1, 1, 1, 1, 1), (1, 64, 8, 128, 128), (3, 4, 2, 130, 40), (40, 8, 3, 96, 200), (33, 16, 16, 384, 129),
         (200, 3, 2, 257, 320), (500, 4, 1, 64, 384), (700, 2, 2, 512, 136), (1300, 2, 1, 96, 640), (2600, 5, 2, 40, 300)]


def hidden_rows(ctx, q, index, experts, m, outs, act, exact=True, extra=0):
    """experts_in8's rows as (bytes, scales) of the pairs with an expert; the others must stay."""
    import ien
    import torch

    tokens, top = index.shape
    routes = plan_of(ctx, index, np.ones(index.shape), experts)
    width, scale_width = 128 * -(-outs // 128), 4 * -(-outs // 512)
    data = torch.full((tokens * top, width + extra), 99, dtype=torch.uint8, device="cuda")
    scales = torch.full((tokens * top, scale_width + extra), 98, dtype=torch.uint8, device="cuda")
    h = ien.Rows8(tokens * top, outs, data=data[:, :width], scales=scales[:, :scale_width])
    ien.experts_in8(ctx, q, routes, m, h, act=act, exact=exact)
    some = int(X.plan(index, experts)[0][-1])
    data, scales, blocks = data.cpu().numpy(), scales.cpu().numpy(), -(-outs // 128)
    assert (data[some:] == 99).all() and (scales[some:] == 98).all()
    assert (data[:, width:] == 99).all() and (scales[:, blocks:] == 98).all()
    return data[:some, :width], scales[:some, :blocks]


@pytest.mark.parametrize("tokens,experts,top,c,hidden", SIZES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("gated", [False, True])
def test_in8_whole(ctx, tokens, experts, top, c, hidden, act, gated):
    import ien

    rng = np.random.default_rng(tokens + c + hidden)
    n = hidden * (2 if gated else 1)
    data, scales = whole_rows(rng, tokens, c)
    x, w = E.values(data, scales, c), whole_weights(rng, experts, c, n)
    b = rng.integers(-20, 20, (experts, n)).astype(np.float32)
    for one in (False, True):
        index = routed(rng, tokens, experts, top, one=one)
        m = ien.Experts8(ctx, w, b, gated=gated)
        got = hidden_rows(ctx, rows8_of(data, scales, c, 16), index, experts, m, hidden, ACTS[act], extra=16)
        v, size = X.products(x, index, w.astype(np.float64), b.astype(np.float64), True)
        v = X.gate(v, act, gated)
        # Whole numbers under 2^24 are f32's: every partial sum is at most `size`, a gated product |v|.
        assert size.size == 0 or (size.max() < 2**24 and np.abs(v).max() < 2**24)
        if not v.size:  # (the only pair has no expert: hidden_rows has seen that it stays)
            continue
        want = E.quantize(v)
        assert np.array_equal(got[1], want[1])
        v = E.values(*want, hidden)  # (a zero may be either one)
        assert np.array_equal(E.values(*got, hidden), v) and not E.E4M3[got[0]][:, hidden:].any()
        m.free()


@pytest.mark.parametrize("tokens,experts,top,c,hidden", SIZES[1:])
@pytest.mark.parametrize("act,gated", [("gelu", False), ("silu", True), ("sigmoid", False), ("sigmoid", True), ("gelu", True)])
@pytest.mark.parametrize("exact", [True, False])
def test_in8_real(ctx, tokens, experts, top, c, hidden, act, gated, exact):
    import ien

    rng = np.random.default_rng(tokens * c + hidden)
    n = hidden * (2 if gated else 1)
    data, scales = E.quantize(rng.standard_normal((tokens, c)))
    x, index = E.values(data, scales, c), routed(rng, tokens, experts, top)
    w = (rng.standard_normal((experts, c, n)) / np.sqrt(c)).astype(np.float32)
    b = rng.standard_normal((experts, n)).astype(np.float32)
    m = ien.Experts8(ctx, w, b, gated=gated)
    got = E.values(*hidden_rows(ctx, rows8_of(data, scales, c), index, experts, m, hidden, ACTS[act], exact), hidden)
    v, size = X.products(x, index, X.weights(w), b.astype(np.float64), True)
    off = (2.0**-23 * c if exact else 2.0**-10) * size + 2.0**-23 * np.abs(v)
    want = X.gate(v, act, gated)
    if gated:
        g = E.activate(v[:, :hidden], act)
        off = E.SLOPE[act] * off[:, :hidden] * (np.abs(v[:, hidden:]) + off[:, hidden:]) + np.abs(g) * off[:, hidden:]
    else:
        off = E.SLOPE[act] * off
    off += 2.0**-21 * np.abs(want)  # (the activation's own)
    _, e = E.quantize(np.abs(want) + off)
    unit = np.repeat(np.ldexp(1.0, e.astype(int) - 127), 128, 1)[:, :hidden]
    assert (np.abs(got - want) <= off + 2.0**-4 * (np.abs(want) + off) + 2.0**-10 * unit).all()
    m.free()


@pytest.mark.parametrize("tokens,experts,top,n,c", SIZES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("add", [None, "rows", "out"])
def test_out8_whole(ctx, tokens, experts, top, n, c, dtype, add):
    """Weights are powers of two, the products within f16's whole numbers."""
    import ien
    import torch

    rng = np.random.default_rng(tokens + 3 * c + n)
    v = np.where(rng.random((tokens * top, c)) < min(1.0, 60 / c), rng.integers(-2, 3, (tokens * top, c)), 0).astype(np.float64)
    data, scales = E.to_bytes(np.concatenate([v, np.zeros((tokens * top, -c % 128))], 1)), np.full((tokens * top, -(-c // 128)), 127, np.uint8)
    index, weight = routed(rng, tokens, experts, top), 2.0 ** rng.integers(-3, 2, (tokens, top))
    w, b = whole_weights(rng, experts, c, n), rng.integers(-9, 9, (experts, n)).astype(np.float32)
    m, routes = ien.Experts8(ctx, w, b), plan_of(ctx, index, weight, experts)
    some = int(X.plan(index, experts)[0][-1])
    data[some:], scales[some:] = 127, 255  # rows without an expert: NaN, never read
    y, size = X.products(v[:some], index, w.astype(np.float64), b.astype(np.float64), False)
    assert size.size == 0 or size.max() <= 2048
    want = X.combine(y, index, weight, experts)
    old = rng.integers(-50, 50, (tokens, n)).astype(dtype)
    if add:
        want = want + old
    out = strided(old if add == "out" else np.zeros((tokens, n), dtype), 5, 7.0)
    parts = ien.expert_parts(routes, m, out.dtype)
    for _ in range(2):
        if add == "out":
            out.copy_(cuda(old))
        ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, parts, out, add={None: None, "rows": strided(old, 3), "out": out}[add])
        assert np.array_equal(out.cpu().numpy(), want.astype(dtype))
    assert bool((torch.as_strided(out, (tokens, n + 5), (n + 5, 1))[:, n:] == 7.0).all())
    m.free()


@pytest.mark.parametrize("tokens,experts,top,n,c", SIZES[2:])
@pytest.mark.parametrize("dtype,exact", [(np.float16, True), (np.float16, False), (np.float32, True)])
def test_out8_real(ctx, tokens, experts, top, n, c, dtype, exact):
    import ien

    rng = np.random.default_rng(tokens * n + c)
    x = rng.standard_normal((tokens * top, c))
    data, scales = E.quantize(x)
    index, weight = routed(rng, tokens, experts, top), rng.random((tokens, top)).astype(np.float32)
    w = (rng.standard_normal((experts, c, n)) / np.sqrt(c)).astype(np.float32)
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, experts)
    out = strided(np.zeros((tokens, n), dtype), 0)
    ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, ien.expert_parts(routes, m, out.dtype), out, exact=exact)
    y, size = X.products(E.values(data, scales, c), index, X.weights(w), None, False)
    half = 2.0**-11 if dtype == np.float16 else 2.0**-24
    off = (2.0**-23 * c if exact else 2.0**-10) * size + half * np.abs(y) + 2.0**-25
    want, off = X.combine(y, index, weight, experts), X.combine(off, index, weight, experts)
    size = X.combine(np.abs(y), index, weight, experts)
    assert (np.abs(out.cpu().numpy() - want) <= off + 2.0**-24 * (top + 1) * size + half * (np.abs(want) + off) + 2.0**-25).all()
    m.free()


def test_weights_of_every_kind(ctx):
    """f16 and f32, torch and numpy, without biases: the same experts."""
    import ien
    import torch

    rng = np.random.default_rng(5)
    w = (rng.standard_normal((3, 200, 64)) / 8).astype(np.float16)
    data, scales = E.quantize(rng.standard_normal((50, 200)))
    index = routed(rng, 50, 3, 2)
    got = []
    for t in (w, w.astype(np.float32), cuda(w), cuda(w).float().transpose(1, 2).contiguous().transpose(1, 2)):
        m = ien.Experts8(ctx, t, gated=True)
        got.append(hidden_rows(ctx, rows8_of(data, scales, 200), index, 3, m, 32, ien.ACT_SILU))
        m.free()
    for g in got[1:]:
        assert np.array_equal(g[0], got[0][0]) and np.array_equal(g[1], got[0][1])
    torch.cuda.synchronize()


def test_an_unplanned_routing_does_nothing(ctx):
    import ien
    import torch

    rng = np.random.default_rng(6)
    m = ien.Experts8(ctx, whole_weights(rng, 2, 64, 64))
    q, h, routes = ien.Rows8(9, 64), ien.Rows8(18, 64), ien.Routes(9, 2, 2)
    q.data.zero_(), q.scales.fill_(127)
    h.data.fill_(99)
    ien.experts_in8(ctx, q, routes, m, h)
    assert bool((h.data == 99).all())
    torch.cuda.synchronize()
    m.free()


@pytest.mark.parametrize("tokens,experts,top", [(3, 4, 1), (90, 3, 2), (1400, 2, 1), (5000, 2, 1)])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_and_outputs_that_are_not_finite(ctx, tokens, experts, top, gated):
    """A NaN in a token's row makes that token's rows NaN and no others; an infinite output is NaN and does not count
    into its block's scale."""
    import ien

    rng = np.random.default_rng(tokens)
    c, outs = 200, 300
    n = outs * (2 if gated else 1)
    data, scales = whole_rows(rng, tokens, c)
    w, b = whole_weights(rng, experts, c, n), rng.integers(1, 9, (experts, n)).astype(np.float32)
    b[:, 130] = np.inf
    if gated:
        w[:, :, outs + 130] = 0  # (the factor of that gate is its bias, 1 .. 8)
    index = np.stack([(np.arange(tokens) + k) % experts for k in range(top)], 1).astype(np.int32)
    bad = tokens // 2
    m = ien.Experts8(ctx, w, b, gated=gated)
    clean = hidden_rows(ctx, rows8_of(data, scales, c), index, experts, m, outs, ien.ACT_RELU)
    v, _ = X.products(E.values(data, scales, c), index, w.astype(np.float64), np.where(np.isinf(b), 0, b).astype(np.float64), True)
    v = X.gate(v, "relu", gated)
    v[:, 130] = np.nan  # (infinite before its rounding)
    want = E.quantize(v)
    assert np.array_equal(clean[1], want[1])
    got, ref = E.values(*clean, outs), E.values(*want, outs)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[~np.isnan(ref)], ref[~np.isnan(ref)])
    broken = data.copy()
    broken[bad, 7] = 127
    again = hidden_rows(ctx, rows8_of(broken, scales, c), index, experts, m, outs, ien.ACT_RELU)
    _, order = X.plan(index, experts)
    its = order // top == bad
    assert its.sum() == top and np.isnan(E.values(again[0][its], again[1][its], outs)).all()
    assert np.array_equal(again[0][~its], clean[0][~its]) and np.array_equal(again[1][~its], clean[1][~its])
    m.free()


def test_an_expert_twice_and_far_values(ctx):
    """The same expert in two of a token's slots; products past f16 in f32 results."""
    import ien
    import torch

    rng = np.random.default_rng(7)
    index = np.array([[1, 1], [0, 1], [1, 0]], np.int32)
    v = rng.integers(-2, 3, (6, 64)).astype(np.float64) * 64
    data, scales = E.to_bytes(np.concatenate([v, np.zeros((6, 64))], 1)), np.full((6, 1), 127, np.uint8)
    w = whole_weights(rng, 2, 64, 24) * 4096
    weight = np.array([[0.5, 0.25], [2, 1], [1, 4]])
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, 2)
    out = torch.empty(3, 24, device="cuda")
    ien.experts_out8(ctx, rows8_of(data, scales, 64), routes, m, ien.expert_parts(routes, m, out.dtype), out)
    y, size = X.products(v, index, w.astype(np.float64), None, False)
    assert size.max() / (64 * 4096) < 2**24 and size.max() > 65504
    assert np.array_equal(out.cpu().numpy(), X.combine(y, index, weight, 2).astype(np.float32))
    m.free()
