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
