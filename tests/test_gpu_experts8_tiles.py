"""Every tile of the experts' products, with whole numbers (equality, see
test_gpu_experts8), and rows that lie past 4 GiB."""

import ctypes

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from internal import _function
from test_gpu_eight_bits import cuda, rows8_of, whole_rows
from test_gpu_experts8 import hidden_rows, plan_of, routed, whole_weights

pytestmark = pytest.mark.gpu

CUS = 256


def in_choice(*a):
    return _function("_ZN3ien17experts_in_choiceEilllii", ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int,
                     ctypes.c_int)(*a)


def out_choice(*a):
    return _function("_ZN3ien18experts_out_choiceElli", ctypes.c_long, ctypes.c_long, ctypes.c_int)(*a)


# tokens, experts, top, c, outputs, gated, the tile
IN = [(6, 3, 2, 200, 130, 1, 0), (150, 3, 1, 130, 200, 1, 1), (1000, 2, 2, 300, 1100, 1, 2), (9000, 4, 2, 520, 1500, 1, 3),
      (3, 4, 1, 200, 130, 0, 0), (200, 3, 2, 130, 200, 0, 1), (1700, 2, 1, 200, 400, 0, 2)]


def test_the_sizes_reach_every_tile(ctx):
    for tokens, experts, top, c, outs, gated, tile in IN:
        npad = 256 * -(-outs // 128) if gated else 128 * -(-outs // 128)
        assert in_choice(CUS, tokens * top, experts, npad, -(-c // 128), gated) == tile, (tokens, outs)


@pytest.mark.parametrize("tokens,experts,top,c,outs,gated,tile", IN)
@pytest.mark.parametrize("fast", [False, True])
def test_in8(ctx, tokens, experts, top, c, outs, gated, tile, fast):
    """Random loads, all tokens with one expert, and none.  (Operands within 4 and 3 under scales of 1 and 2: aligned eights
    of products under 2^13 of the largest's last bit lose nothing in the coarser sums either.)"""
    import ien

    rng = np.random.default_rng(tokens)
    n = outs * (1 + gated)
    data, scales = whole_rows(rng, tokens, c)
    w, b = whole_weights(rng, experts, c, n), rng.integers(-9, 9, (experts, n)).astype(np.float32)
    m, x, q = ien.Experts8(ctx, w, b, gated=bool(gated)), E.values(data, scales, c), rows8_of(data, scales, c)
    loads = [routed(rng, tokens, experts, top), np.full((tokens, top), -1, np.int32), np.full((tokens, top), -1, np.int32)]
    loads[1][:, 0] = experts - 1
    for index in loads:
        got = hidden_rows(ctx, q, index, experts, m, outs, ien.ACT_RELU, exact=not fast)
        v, size = X.products(x, index, w.astype(np.float64), b.astype(np.float64), True)
        v = X.gate(v, "relu", gated)
        if not v.size:
            continue
        assert size.max() < 2**24 and np.abs(v).max() < 2**24
        want = E.quantize(v)
        assert np.array_equal(got[1], want[1]) and np.array_equal(E.values(*got, outs), E.values(*want, outs))
    m.free()


# tokens, experts, top, depth, outputs, the tile
OUT = [(3, 4, 2, 300, 70, 0), (250, 3, 2, 200, 130, 1), (1500, 2, 1, 140, 200, 2), (2, 3, 2, 2100, 37, 3)]


@pytest.mark.parametrize("tokens,experts,top,c,n,tile", OUT)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("fast", [False, True])
def test_out8(ctx, tokens, experts, top, c, n, tile, dtype, fast):
    import ien
    import torch

    assert out_choice(tokens * top, experts, -(-c // 128)) == tile
    rng = np.random.default_rng(tokens)
    pairs = tokens * top
    v = np.where(rng.random((pairs, c)) < min(1.0, 60 / c), rng.integers(-2, 3, (pairs, c)), 0).astype(np.float64)
    data = E.to_bytes(np.concatenate([v, np.zeros((pairs, -c % 128))], 1))
    scales = np.full((pairs, -(-c // 128)), 127, np.uint8)
    index, weight = routed(rng, tokens, experts, top), 2.0 ** rng.integers(-3, 2, (tokens, top))
    w = whole_weights(rng, experts, c, n)
    m, routes = ien.Experts8(ctx, w), plan_of(ctx, index, weight, experts)
    out = torch.empty(tokens, n, dtype=cuda(np.zeros(1, dtype)).dtype, device="cuda")
    ien.experts_out8(ctx, rows8_of(data, scales, c), routes, m, ien.expert_parts(routes, m, out.dtype), out, exact=not fast)
    y, size = X.products(v[:int(X.plan(index, experts)[0][-1])], index, w.astype(np.float64), None, False)
    assert size.max() <= 2048  # (f16's whole numbers)
    assert np.array_equal(out.cpu().numpy(), X.combine(y, index, weight, experts).astype(dtype))
    m.free()


def test_rows_past_32_bits(ctx):
    """4.6 GB of hidden rows, a stream 65536 apart, logits 16384 apart: the last tokens as the first."""
    import ien
    import torch

    rng = np.random.default_rng(9)
    tokens, c, experts = 1 << 17, 64, 2
    wide = torch.zeros(tokens, 20000, dtype=torch.float16, device="cuda")
    part = rng.standard_normal((256, c)).astype(np.float16)
    wide[:256, :c] = wide[-256:, :c] = cuda(part)
    y = torch.empty(tokens, c, dtype=torch.float16, device="cuda")
    ien.rms_norm(ctx, wide[:, :c], None, y, total=wide[:, 8192:8192 + c])
    assert torch.equal(y[:256], y[-256:]) and torch.equal(wide[-256:, 8192:8192 + c], wide[-256:, :c]) and bool(y[-1].any())
    routes = ien.Routes(tokens, experts, 1)
    wide[:, :2] = 0
    wide[-256:, :2] = wide[:256, :2] = cuda(part[:, :2])
    ien.route(ctx, wide[:, :2], routes)
    assert torch.equal(routes.index[:256], routes.index[-256:]) and len(set(routes.index[-256:, 0].tolist())) == 2
    del wide
    hidden = 35000
    h = ien.Rows8(tokens, hidden)
    assert h.data.numel() > 2**32
    h.data.zero_()
    h.scales.fill_(127)
    order = routes.order.long()
    rows = cuda(E.to_bytes(rng.integers(-1, 2, (1, hidden)).astype(np.float64)))
    h.data[-1, :hidden] = rows[0]
    w = whole_weights(rng, experts, hidden, 16)
    m = ien.Experts8(ctx, w)
    out = torch.empty(tokens, 16, dtype=torch.float32, device="cuda")
    ien.experts_out8(ctx, h, routes, m, ien.expert_parts(routes, m, out.dtype), out)
    last = int(order[-1])
    e = int(routes.index[last, 0])
    want = E.E4M3[rows[0].cpu().numpy()] @ w[e].astype(np.float64)
    assert np.array_equal(out[last].cpu().numpy(), (want * float(routes.weight[last, 0])).astype(np.float32))
    out[last] = 0
    assert not bool(out.any())
    m.free()
