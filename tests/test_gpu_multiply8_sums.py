"""How exactly the 8-bit products add: in f32 unless the caller asks otherwise.

A product and its opposite with a small one between them, neighbours in one
block of 128: their sum is the small product, which f32 holds beside 2^16 down to
2^-7.  All values are powers of two, so nothing rounds."""

import numpy as np
import pytest

import eight_bits as E
from test_gpu_eight_bits import rows8_of

pytestmark = pytest.mark.gpu


def cancelling(rows, taps, k, n, at, t):
    """Rows and weights whose products at `at` and its neighbours are 2^16, 1/4 and
    -2^16, at tap t."""
    x, w = np.zeros((rows, k), np.float32), np.zeros((taps * k, n), np.float32)
    x[:, at:at + 3] = 256, 0.25, 256
    w[t * k + at:t * k + at + 3] = np.array([256, 1, -256], np.float32)[:, None]
    return x, w


# (rows, k, n): a small tile, its depth in splits, a middle tile, the largest one.
@pytest.mark.parametrize("rows,k,n", [(5, 128, 72), (3, 9000, 24), (4096, 384, 136), (16384, 256, 2048)])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_small_products_beside_large_ones(ctx, rows, k, n, dtype):
    import ien
    import torch

    for at in (0, 4, 101):
        x, w = cancelling(rows, 1, k, n, at, 0)
        m = ien.Matrix8(ctx, w)
        y = torch.full((rows, n), 9.0, dtype=getattr(torch, dtype), device="cuda")
        ien.multiply8(ctx, rows8_of(*E.quantize(x), k), m, y)
        assert bool((y == 0.25).all())
        m.free()


def test_small_products_of_a_map(ctx):
    import ien
    import torch

    x, w = cancelling(2 * 8 * 24, 9, 128, 40, 17, 4)
    y = torch.full((2 * 8 * 24, 40), 9.0, dtype=torch.float16, device="cuda")
    ien.conv8(ctx, rows8_of(*E.quantize(x), 128), 2, 8, 24, ien.Matrix8(ctx, w, taps=9), y)
    assert bool((y == 0.25).all())


def exponents(data, scales):
    """The powers of two of bytes under their scales, [rows, k]: at least -6 before the scale."""
    e = np.maximum(np.frexp(np.nan_to_num(E.E4M3[data]))[1] - 1, -6)
    e = np.where(E.E4M3[data] == 0, -6, e)
    return e + np.repeat(scales.astype(int) - 127, 128, 1)


@pytest.mark.parametrize("rows,k,n", [(1, 128, 24), (37, 1152, 72), (300, 512, 136), (4096, 256, 136)])
def test_fast_sums(ctx, rows, k, n):
    """exact=False, where neighbours cancel and values lie far apart: each eight
    products are off by at most 8 times 2^-13 of the largest one's power of two, the
    sums by a step of f32 each, the result by half a step of f16."""
    import ien
    import torch

    rng = np.random.default_rng(rows + k)
    x = (rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-9, 9, (rows, k))).astype(np.float32)
    w = (rng.standard_normal((k, n)) * 2.0 ** rng.integers(-4, 4, (k, n))).astype(np.float32)
    x[:, 1::2] = x[:, ::2] * (1 + 2.0**-4 * rng.standard_normal((rows, k // 2)))
    w[1::2] = -w[::2]
    data, scales = E.quantize(x)
    m = ien.Matrix8(ctx, w)
    y = torch.full((rows, n), 9.0, dtype=torch.float16, device="cuda")
    ien.multiply8(ctx, rows8_of(data, scales, k), m, y, exact=False)
    wdata, wscales = E.quantize(np.ascontiguousarray(w.T))
    x8, w8 = E.values(data, scales, k), E.values(wdata, wscales, k).T
    want = x8 @ w8
    ex, ew = exponents(data, scales).reshape(rows, -1, 8), exponents(wdata, wscales).reshape(n, -1, 8)
    off = np.zeros((rows, n))
    for g in range(k // 8):
        off += 2.0 ** (ex[:, None, g] + ew[None, :, g]).max(2)
    tol = 8 * 2.0**-13 * off + (k + 2) * 2.0**-23 * (np.abs(x8) @ np.abs(w8)) + 2.0**-11 * np.abs(want) + 2.0**-25
    with np.errstate(over="ignore"):
        assert (np.abs(want) + tol < 65504).all()
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
