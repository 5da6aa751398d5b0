"""Thousands of groups: their statistics take more than 64 KB of LDS beside the
lanes' (one launch and two)."""

import numpy as np
import pytest

from test_gpu_group_norm import check, features

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(np.float16, np.float16), (np.float32, np.float32)])
@pytest.mark.parametrize("c,groups", [(8191, 8191), (8190, 2730), (8192, 8192), (7000, 7000), (5001, 1667)])
@pytest.mark.parametrize("images,pixels", [(1, 5), (2, 8), (1, 40), (1, 1000)])
def test_many_groups(ctx, images, pixels, c, groups, types):
    rng = np.random.default_rng(pixels + c)
    x = features(rng, images * pixels, c, types[0])
    gamma, beta = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32), rng.standard_normal(c).astype(np.float32)
    check(ctx, x, images, groups, gamma, beta, "silu", types[1], 3)


@pytest.mark.parametrize("pixels", [5, 40])
def test_many_groups_into_8_bits(ctx, pixels):
    """Bit for bit the 8-bit form of the f32 result."""
    import ien
    import torch

    c = 8191
    x = torch.randn(pixels, c, device="cuda").half()
    y = torch.empty(pixels, c, device="cuda")
    want, got = ien.Rows8(pixels, c), ien.Rows8(pixels, c)
    ien.group_norm(ctx, x, 1, c, None, None, y, act=ien.ACT_SILU)
    ien.quantize8(ctx, y, want)
    ien.group_norm(ctx, x, 1, c, None, None, got, act=ien.ACT_SILU)
    assert torch.equal(got.data, want.data) and torch.equal(got.scales[:, :64], want.scales[:, :64])
