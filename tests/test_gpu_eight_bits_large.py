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


@pytest.mark.parametrize("images,pixels,c,groups", [(65600, 1, 8192, 1024), (70000, 2, 512, 64)])
@pytest.mark.parametrize("into", ["float16", "8 bits"])
def test_group_norm_of_many_maps(ctx, images, pixels, c, groups, into):
    """More workgroups than a launch has: maps at both ends and where turns meet have the
    bits that they have alone."""
    import ien
    import torch

    x = torch.randn(images * pixels, c, device="cuda").half()

    def run(x, images):
        if into == "8 bits":
            y = ien.Rows8(images * pixels, c)
            ien.group_norm(ctx, x, images, groups, None, None, y, act=ien.ACT_SILU)
            return y.data, y.scales[:, :c // 128]
        y = torch.empty_like(x)
        ien.group_norm(ctx, x, images, groups, None, None, y, act=ien.ACT_SILU)
        return (y,)

    whole = run(x, images)
    for begin in (0, 32768 - 20, 65536 - 40, images - 50):
        rows = slice(begin * pixels, (begin + 50) * pixels)
        for w, p in zip(whole, run(x[rows].contiguous(), 50)):
            assert torch.equal(w[rows], p)
    del x, whole
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,add", [("float16", True), ("float32", False)])
def test_multiply8_in_parts(ctx, dtype, add):
    """More tiles than a launch has (17 GB of rows): rows at both ends and where the
    parts meet have the bits that they have alone."""
    import ien
    import numpy as np
    import torch

    rows, k, n, dtype = (1 << 27) + 300, 24, 8, getattr(torch, dtype)
    data = torch.randint(0, 120, (4096, 128), dtype=torch.uint8, device="cuda")
    data[:, k:] = 0
    data = data.repeat(rows // 4096 + 1, 1)[:rows]
    q = ien.Rows8(rows, k, data=data)
    q.scales.fill_(124)
    rng = np.random.default_rng(1)
    m = ien.Matrix8(ctx, rng.standard_normal((k, n)).astype(np.float32), rng.standard_normal(n).astype(np.float32))
    y = torch.full((rows, n), float("nan"), dtype=dtype, device="cuda")
    old = torch.randn(rows, n, device="cuda").to(dtype) if add else None
    ien.multiply8(ctx, q, m, y, add=old)
    for begin in (0, (1 << 27) - 200, rows - 250):
        part = slice(begin, begin + 250)
        p = ien.Rows8(250, k, data=data[part].contiguous())
        p.scales.fill_(124)
        z = torch.empty(250, n, dtype=dtype, device="cuda")
        ien.multiply8(ctx, p, m, z, add=old[part].contiguous() if add else None)
        assert torch.equal(y[part], z)
    assert not bool(y.isnan().any())
    del data, q, y, old
    torch.cuda.empty_cache()
