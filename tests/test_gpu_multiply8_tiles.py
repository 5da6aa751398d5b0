"""Every tile of the 8-bit products at its edges, and exact sums into f16.

Products of whole numbers as in test_gpu_eight_bits: equal whatever the order
of the sums."""

import numpy as np
import pytest

import eight_bits as E
from test_gpu_eight_bits import check_whole, rows8_of, whole_rows, whole_weights

pytestmark = pytest.mark.gpu


# (rows, k, n): ragged rows and outputs, depths of one block, of odd numbers of blocks and
# of more than a dword of scales.
CASES = [(16387, 256, 2056), (33000, 130, 1000), (20000, 700, 1288), (8200, 640, 1032), (5000, 1100, 2056), (4000, 384, 520),
         (2000, 1664, 1000), (130, 300, 40), (70, 4000, 200)]


@pytest.mark.parametrize("rows,k,n", CASES)
def test_tiles(ctx, rows, k, n):
    import ien

    rng = np.random.default_rng(rows + k + n)
    data, scales = whole_rows(rng, rows, k)
    check_whole(ctx, rng, E.values(data, scales, k), data, scales, k, whole_weights(rng, 1, k, n), 1, rows,
                lambda q, m, y, add: ien.multiply8(ctx, q, m, y, add=add))


@pytest.mark.parametrize("rows,k,n", CASES)
def test_tiles_without_a_residual(ctx, rows, k, n):
    import ien
    import torch

    rng = np.random.default_rng(rows + k + n)
    data, scales = whole_rows(rng, rows, k)
    w = whole_weights(rng, 1, k, n)
    b = rng.integers(-9, 10, n).astype(np.float32)
    want = torch.from_numpy((E.values(data, scales, k) @ E.weights(w, 1) + b).astype(np.float32)).cuda()
    q, m = rows8_of(data, scales, k, 16), ien.Matrix8(ctx, w, b)
    for dtype, exact in ((torch.float16, False), (torch.float16, True), (torch.float32, False)):
        for extra in (0, 3):
            y = torch.full((rows, n + extra), 5.0, dtype=dtype, device="cuda")
            ien.multiply8(ctx, q, m, y[:, :n], exact=exact)
            assert torch.equal(y[:, :n], want.to(dtype)) and bool((y[:, n:] == 5.0).all())


@pytest.mark.parametrize("images,h,w,step,c,n", [(1, 257, 127, 1, 256, 520), (3, 66, 130, 1, 200, 328),
                                                 (1, 300, 200, 2, 136, 264), (40, 9, 11, 1, 128, 600)])
def test_conv_tiles(ctx, images, h, w, step, c, n):
    import ien

    rng = np.random.default_rng(h + w + c)
    data, scales = whole_rows(rng, images * h * w, c)
    x = E.patches(E.values(data, scales, c), images, h, w, step)
    check_whole(ctx, rng, x, data, scales, c, whole_weights(rng, 9, c, n), 9, x.shape[0],
                lambda q, m, y, add: ien.conv8(ctx, q, images, h, w, m, y, step=step, add=add))


@pytest.mark.parametrize("rows,k,n", [(3, 200, 24), (300, 1280, 320), (4096, 384, 136), (16384, 384, 2048)])
def test_exact_whole_numbers(ctx, rows, k, n):
    import ien

    rng = np.random.default_rng(k)
    data, scales = whole_rows(rng, rows, k)
    check_whole(ctx, rng, E.values(data, scales, k), data, scales, k, whole_weights(rng, 1, k, n), 1, rows,
                lambda q, m, y, add: ien.multiply8(ctx, q, m, y, add=add, exact=True))


@pytest.mark.parametrize("taps,rows", [(1, 5), (1, 700), (9, 64)])
def test_exact_keeps_small_products_beside_large_ones(ctx, taps, rows):
    """2^16 + 1 - 2^16 in every sum, neighbours in the first half of a block:
    exactly 1, in f16 as in f32."""
    import ien
    import torch

    k, n = 128, 72
    x = np.zeros((rows, k), np.float32)
    x[:, :3] = 256, 1, 256
    w = np.zeros((taps * k, n), np.float32)
    t = taps // 2 * k  # the tap at the pixel itself
    w[t], w[t + 1], w[t + 2] = 256, 1, -256
    data, scales = E.quantize(x)
    q, m = rows8_of(data, scales, k), ien.Matrix8(ctx, w, taps=taps)
    for dtype in (torch.float16, torch.float32):
        y = torch.full((rows, n), 9.0, dtype=dtype, device="cuda")
        if taps == 1:
            ien.multiply8(ctx, q, m, y, exact=True)
        else:
            ien.conv8(ctx, q, 1, 8, rows // 8, m, y, exact=True)
        assert bool((y == 1).all())


def test_rows_far_apart(ctx):
    """Rows whose bytes lie past 2^31 from the first: 3000 of them a MiB less a
    step apart."""
    import ien
    import torch

    rng = np.random.default_rng(7)
    rows, k, n, stride = 3000, 300, 40, (1 << 20) - 128
    data, scales = whole_rows(rng, rows, k)
    flat = torch.empty(rows * stride, dtype=torch.uint8, device="cuda")
    at = flat.as_strided((rows, data.shape[1]), (stride, 1))
    at.copy_(torch.from_numpy(data))
    near = rows8_of(data, scales, k)
    w = whole_weights(rng, 1, k, n)
    m = ien.Matrix8(ctx, w)
    y, want = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    ien.multiply8(ctx, ien.Rows8(rows, k, data=at, scales=near.scales), m, y)
    ien.multiply8(ctx, near, m, want)
    assert torch.equal(y, want)
    del flat, at
    torch.cuda.empty_cache()
