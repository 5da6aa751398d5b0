"""Maps whose rows or images take more lanes than one launch has."""

import pytest

pytestmark = pytest.mark.gpu


def test_quantize8_in_turns(ctx):
    """More blocks than the lanes of a launch: rows at both ends and where turns meet."""
    import ien
    import torch

    rows = (1 << 24) + 5000
    x = torch.randn(rows, 3, device="cuda")
    q = ien.Rows8(rows, 3)
    ien.quantize8(ctx, x, q)
    y = torch.empty_like(x)
    ien.dequantize8(ctx, q, y)
    for begin in (0, (1 << 24) - 70, rows - 300):
        part = x[begin:begin + 300].contiguous()
        p, z = ien.Rows8(300, 3), torch.empty_like(part)
        ien.quantize8(ctx, part, p)
        ien.dequantize8(ctx, p, z)
        assert torch.equal(q.data[begin:begin + 300], p.data) and torch.equal(q.scales[begin:begin + 300, 0], p.scales[:, 0])
        assert torch.equal(y[begin:begin + 300], z)
    # Every value within half a step of e4m3 (2^-4 of itself, or 2^-10 of the scale).
    tol = torch.maximum(x.abs() * 2.0**-4, 2.0**-10 * torch.exp2(q.scales[:, :1].float() - 127))
    assert bool(((y - x).abs() <= tol).all())
    del x, q, y, tol
    torch.cuda.empty_cache()
