"""The ends of the scales: what the formats between them hold is exact, what they do
not hold becomes what the header says.  Every e4m3 value alone in its row, by
weights of one power of two, so nothing else rounds."""

import numpy as np
import pytest

import eight_bits as E
from test_gpu_eight_bits import cuda, rows8_of

pytestmark = pytest.mark.gpu

BYTES = np.array([b for b in range(256) if b & 127 != 127], np.uint8)


def rows_of(scale):
    data = np.zeros((len(BYTES), 128), np.uint8)
    data[:, 0] = BYTES
    scales = np.full((len(BYTES), 1), scale, np.uint8)
    return data, scales, E.values(data, scales, 128)[:, 0]


@pytest.mark.parametrize("scale", [0, 1, 2, 3, 4, 9, 60, 127, 200, 245, 246, 247, 248, 253, 254])
def test_exact_products(ctx, scale):
    import ien
    import torch

    data, scales, v = rows_of(scale)
    w = np.zeros((128, 8), np.float32)
    w[0] = 2.0 ** (100 if scale < 127 else -100)
    y = torch.empty(len(BYTES), 8, device="cuda")
    ien.multiply8(ctx, rows8_of(data, scales, 128), ien.Matrix8(ctx, w), y)
    if 3 <= scale <= 246:
        taken = v
    else:
        taken = np.rint(v * 2.0**133) * 2.0**-133  # (ties to even)
        taken = np.where(np.abs(v) >= 2.0**128, np.copysign(np.inf, v), taken)
    assert np.array_equal(y.double().cpu().numpy(), np.repeat((taken * float(w[0, 0]))[:, None], 8, 1))


@pytest.mark.parametrize("scale", [1, 2, 3, 127, 246, 247, 253])
def test_fast_products(ctx, scale):
    """The 8-bit instructions apply the scales themselves: exact under all of them."""
    import ien
    import torch

    data, scales, v = rows_of(scale)
    w = np.zeros((128, 8), np.float32)
    w[0] = 2.0 ** (127 - scale)
    y = torch.empty(len(BYTES), 8, dtype=torch.float16, device="cuda")
    ien.multiply8(ctx, rows8_of(data, scales, 128), ien.Matrix8(ctx, w), y, exact=False)
    assert np.array_equal(y.double().cpu().numpy(), np.repeat((v * float(w[0, 0]))[:, None], 8, 1))


@pytest.mark.parametrize("scale", [0, 1, 3, 127, 246, 247, 254])
def test_read_back(ctx, scale):
    import ien
    import torch

    data, scales, v = rows_of(scale)
    y = torch.empty(len(BYTES), 128, device="cuda")
    ien.dequantize8(ctx, rows8_of(data, scales, 128), y)
    want = np.where(np.abs(v) >= 2.0**128, np.copysign(np.inf, v), v)
    assert np.array_equal(y[:, 0].double().cpu().numpy(), want)


def test_the_largest_f32(ctx):
    """Is rounded to 2^128, under scale 247, and comes back as infinity; a step of e4m3
    below it comes back as it is."""
    import ien
    import torch

    x = np.zeros((2, 8), np.float32)
    x[0, 0], x[1, 0] = np.finfo(np.float32).max, 240 * 2.0**120
    q, y = ien.Rows8(2, 8), torch.empty(2, 8, device="cuda")
    ien.quantize8(ctx, cuda(x), q)
    ien.dequantize8(ctx, q, y)
    assert q.scales[:, 0].tolist() == [247, 247]
    assert y[0, 0].item() == float("inf") and y[1, 0].item() == x[1, 0]
