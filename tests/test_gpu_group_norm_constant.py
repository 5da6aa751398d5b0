"""Groups of equal values, whatever their sizes: every deviation is exactly 0 (all
sums are of differences from one of the values), so the result is 0 where f32 does
not hold the sum of the values.  A mean that is off by one step of f32 would give
0.02 at 1000."""

import pytest

pytestmark = pytest.mark.gpu


# Lanes with one to eight pixels and more, one launch and two.
@pytest.mark.parametrize("pixels", [1, 3, 5, 7, 64, 150, 190, 200, 300, 350, 400, 450, 512, 700, 3000, 20000])
@pytest.mark.parametrize("per", [1, 3, 5, 6, 7, 10, 12, 20, 40, 72])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_constant_groups(ctx, per, pixels, dtype):
    import ien
    import torch

    values = torch.tensor([1000.1, -777.7, 1234.567, 1e-3], device="cuda").to(getattr(torch, dtype))
    x = values.repeat_interleave(per).repeat(2 * pixels, 1)
    y = torch.full((2 * pixels, 4 * per), 9.0, device="cuda")
    ien.group_norm(ctx, x, 2, 4, None, None, y)
    assert bool((y == 0).all()), float(y.abs().max())
