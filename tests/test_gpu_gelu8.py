"""GELU of the 8-bit products and of the norm, over the whole line, in f32 and f16.

v Phi(v) = max(v, 0) - |v| Phi(-|v|).  The tail |v| Phi(-|v|) is allowed, in steps
of 2^-24 of itself, 6 for the reciprocal (a step of 2^-23 through a slope of 2.7),
3 for the polynomial, 3 for the exponential and the products, and v^2 for the
exponential's argument (two roundings of v^2 / 2); and the result its rounding,
half a step of its type.  Exponentials under 2^-126 are 0."""

import numpy as np
import pytest

from test_gpu_eight_bits import cuda

pytestmark = pytest.mark.gpu


def values(count):
    spread = np.concatenate([np.linspace(-14, 14, count // 2), np.geomspace(1e-8, 30, count // 4), -np.geomspace(1e-8, 30, count // 4)])
    ends = [0.0, -0.0, 100, -100, 1000, -1000, 60000, -60000, 3e38, -3e38, np.inf, -np.inf, np.nan]
    return np.concatenate([spread, ends]).astype(np.float32)


def check(v, got, dtype):
    from scipy.special import ndtr

    x, got = v.astype(np.float64), got.astype(np.float64)
    fine = np.isfinite(x) & (np.abs(x) < (65504 if dtype == "float16" else 4e38))
    a = np.abs(np.where(fine, x, 0.0))
    tail = a * ndtr(-a)
    want = np.where(np.where(fine, x, 0.0) > 0, a, 0.0) - tail
    half = 2.0**-11 if dtype == "float16" else 2.0**-24
    tol = (12 + a * a) * 2.0**-24 * tail + half * np.abs(want) + (2.0**-25 if dtype == "float16" else 2.0**-120)
    off = np.abs(got - want)[fine]
    assert (off <= tol[fine]).all(), (float((off / tol[fine]).max()), x[fine][np.argmax(off / tol[fine])])
    assert (got[x < -15] == 0).all() and (got[x == np.inf] == np.inf).all()
    assert np.array_equal(np.isnan(got), np.isnan(x))


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_products(ctx, dtype, exact):
    """Rows of zeros: the result is the bias's."""
    import ien
    import torch

    v = values(40000)
    m = ien.Matrix8(ctx, np.zeros((16, len(v)), np.float32), v)
    q = ien.Rows8(3, 16)
    ien.quantize8(ctx, torch.zeros(3, 16, device="cuda"), q)
    y = torch.empty(3, len(v), dtype=getattr(torch, dtype), device="cuda")
    ien.multiply8(ctx, q, m, y, act=ien.ACT_GELU, exact=exact)
    assert all(torch.equal(r.view(torch.uint8), y[0].view(torch.uint8)) for r in y)
    check(v, y[1].cpu().numpy(), dtype)


@pytest.mark.parametrize("pixels", [4, 3000])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_norm(ctx, dtype, pixels):
    """Maps without deviations: the result is beta's."""
    import ien
    import torch

    v = values(8000)
    y = torch.empty(pixels, len(v), dtype=getattr(torch, dtype), device="cuda")
    ien.group_norm(ctx, torch.full((pixels, len(v)), 2.5, device="cuda"), 1, 1, None, cuda(v), y, act=ien.ACT_GELU)
    assert torch.equal(y[0].view(torch.uint8), y[-1].view(torch.uint8))
    check(v, y[pixels // 2].cpu().numpy(), dtype)
