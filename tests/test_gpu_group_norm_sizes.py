"""Group norm at the sizes where its launches change: many maps, many groups,
the last map that takes one launch, runs of channels that share no eight."""

import numpy as np
import pytest

import eight_bits as E
from test_gpu_eight_bits import cuda
from test_gpu_group_norm import check, features

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("images,pixels,c,groups,extra", [
    (1, 512, 128, 32, 0), (1, 513, 128, 32, 0), (2, 511, 256, 32, 0), (1, 103, 640, 32, 0), (1, 97, 640, 32, 0),
    (300, 700, 16, 2, 0), (700, 3, 36, 6, 0), (1, 40, 8192, 8192, 0), (1, 300, 8192, 1, 0), (1, 2000, 2000, 1000, 0),
    (2, 5000, 24, 24, 1), (1, 3000, 96, 96, 13), (1, 100000, 1, 1, 0), (1, 9000, 7, 1, 2), (1, 4000, 4090, 10, 0),
    (1, 1100, 6, 3, 0), (1, 50000, 12, 6, 0), (3, 2100, 130, 13, 6)])
@pytest.mark.parametrize("types", [(np.float16, np.float16), (np.float32, np.float32)])
def test_sizes(ctx, images, pixels, c, groups, extra, types):
    rng = np.random.default_rng(pixels * 3 + c)
    x = features(rng, images * pixels, c, types[0])
    gamma, beta = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32), rng.standard_normal(c).astype(np.float32)
    check(ctx, x, images, groups, gamma, beta, "silu", types[1], extra)


@pytest.mark.parametrize("images,pixels,c,groups", [(1, 16, 640, 32), (2, 100, 256, 32), (1, 64, 1280, 32), (5, 7, 96, 4),
                                                    (1, 700, 4090, 10), (1, 2000, 130, 13)])
def test_8_bits_of_the_result(ctx, images, pixels, c, groups):
    """Bit for bit the 8-bit form of the f32 result, whichever launches run."""
    import ien
    import torch

    rng = np.random.default_rng(c + pixels)
    x = cuda(features(rng, images * pixels, c, np.float16))
    y = torch.empty(images * pixels, c, device="cuda")
    want, got = ien.Rows8(images * pixels, c), ien.Rows8(images * pixels, c)
    got.data.fill_(99)
    ien.group_norm(ctx, x, images, groups, None, None, y, act=ien.ACT_SILU)
    ien.quantize8(ctx, y, want)
    ien.group_norm(ctx, x, images, groups, None, None, got, act=ien.ACT_SILU)
    blocks = -(-c // 128)
    assert torch.equal(got.scales[:, :blocks], want.scales[:, :blocks]) and torch.equal(got.data, want.data)


@pytest.mark.parametrize("pixels", [30, 3000])
def test_far_first_values(ctx, pixels):
    """A first pixel thousands of deviations from the others: the parts' and
    batches' sums start from it."""
    rng = np.random.default_rng(5)
    x = (3 + 0.1 * rng.standard_normal((pixels, 64))).astype(np.float32)
    x[0] = 5000
    x[pixels // 2, ::7] = -7000
    check(ctx, x, 1, 8, None, None, "none", np.float32)
