"""ien_rms_norm against its definition in 64 bits.

The sum is one f32 addition, which numpy rounds alike: compared for equality.  The
norm of the f32 sum takes a factor rounded to f32 and two products, 2^-24 each (the
mean of squares is f64's): 2^-22 of the value covers the three, with half a step of
the output (2^-24 of the value in f32, 2^-11 in f16 or 2^-25 among its subnormals).  The
result in 8 bits is the quantised f32 result, bit for bit."""

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import cuda, strided

pytestmark = pytest.mark.gpu


def close(got, want, dtype):
    half = 2.0**-11 if dtype == np.float16 else 2.0**-24
    tol = (2.0**-22 + half) * np.abs(want) + (2.0**-25 if dtype == np.float16 else 2.0**-149)
    assert (np.abs(got.astype(np.float64) - want) <= tol).all(), np.max(np.abs(got - want) / tol)


def rows(rng, r, c, dtype):
    return (rng.standard_normal((r, c)) * 2.0 ** rng.integers(-3, 4, (r, c)) + 0.25).astype(dtype)


SIZES = [(1, 1), (3, 7), (17, 8), (5, 128), (33, 129), (2, 387), (9, 512), (70, 520), (1, 768), (6, 1024), (5, 1031), (3, 2048),
         (2, 2050), (3, 4096), (1, 4097), (2, 8192), (1100, 64), (4099, 24)]


@pytest.mark.parametrize("r,c", SIZES)
@pytest.mark.parametrize("into,added,outof", [
    (np.float16, None, np.float16), (np.float16, np.float16, np.float16), (np.float16, np.float32, np.float32),
    (np.float32, np.float16, np.float16), (np.float32, np.float32, np.float32), (np.float32, None, np.float16)])
def test_rms_norm(ctx, r, c, into, added, outof):
    import ien
    import torch

    rng = np.random.default_rng(c + r)
    x, gamma = rows(rng, r, c, into), (1 + 0.2 * rng.standard_normal(c)).astype(np.float32)
    a = None if added is None else rows(rng, r, c, added)
    s = x.astype(np.float32) + (0 if a is None else a.astype(np.float32))
    for extra, g in ((0, gamma), (5, None)):
        want = X.rms_norm(s, g, 1e-6)
        total, y = strided(np.zeros_like(x), extra, 7.0), strided(np.zeros((r, c), outof), extra, 7.0)
        q = ien.Rows8(r, c)
        q.data.fill_(99)
        q.scales.fill_(99)
        ien.rms_norm(ctx, strided(x, extra), None if g is None else cuda(g), y, q, add=None if a is None else strided(a, extra),
                     total=total)
        assert np.array_equal(total.cpu().numpy(), s.astype(into))
        close(y.cpu().numpy(), want, outof)
        y32 = torch.empty(r, c, dtype=torch.float32, device="cuda")
        ien.rms_norm(ctx, strided(x, extra), None if g is None else cuda(g), y32, add=None if a is None else strided(a, extra))
        data, scales = E.quantize(y32.cpu().numpy())
        assert np.array_equal(q.data.cpu().numpy(), data)
        assert np.array_equal(q.scales[:, :scales.shape[1]].cpu().numpy(), scales)
        if extra:  # what lies between the rows stays
            for t in (total, y):
                wide = torch.as_strided(t, (r, c + extra), (c + extra, 1))
                assert bool((wide[:, c:] == 7.0).all())


@pytest.mark.parametrize("r,c", [(40, 96), (7, 1024), (3, 5000)])
def test_in_place(ctx, r, c):
    """The sum in place of either addend, and the norm in place of the input."""
    import ien

    rng = np.random.default_rng(c)
    x, a = rows(rng, r, c, np.float16), rows(rng, r, c, np.float16)
    s = x.astype(np.float32) + a.astype(np.float32)
    want = X.rms_norm(s, None, 1e-6)
    for over in ("x", "add"):
        xt, at, y = cuda(x), cuda(a), cuda(np.zeros_like(x))
        ien.rms_norm(ctx, xt, None, y, add=at, total=xt if over == "x" else at)
        assert np.array_equal((xt if over == "x" else at).cpu().numpy(), s.astype(np.float16))
        close(y.cpu().numpy(), want, np.float16)
    xt = cuda(x)
    ien.rms_norm(ctx, xt, None, xt, add=cuda(a))
    close(xt.cpu().numpy(), want, np.float16)


def test_rows_that_have_no_ordinary_norm(ctx):
    """Zeros (also without an epsilon), squares past f32, infinities and NaN: those
    rows alone are touched."""
    import ien
    import torch

    x = np.ones((6, 200), np.float32)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 5] = np.inf
    x[4, 7] = np.nan
    y, q = torch.empty(6, 200, device="cuda"), ien.Rows8(6, 200)
    ien.rms_norm(ctx, cuda(x), None, y, q, eps=0.0)
    got = y.cpu().numpy()
    assert np.isnan(got[0]).all() and np.isnan(got[4]).all()  # 0 / 0 as written
    assert np.abs(got[[1, 2, 5]] - 1).max() <= 2.0**-22
    assert np.isnan(got[3, 5]) and (np.delete(got[3], 5) == 0).all()
    ien.rms_norm(ctx, cuda(x), None, y, q, eps=1e-6)
    got = y.cpu().numpy()
    assert (got[0] == 0).all() and (q.data[0].cpu().numpy() == 0).all()
    assert (np.abs(got[2] - 1e-27) <= 1e-33).all()


def test_nothing_is_asked_for(ctx):
    """No rows, and a sum alone."""
    import ien
    import torch

    ien.rms_norm(ctx, torch.empty(0, 16, dtype=torch.float16, device="cuda"), None)
    x = cuda(np.ones((2, 16), np.float16))
    ien.rms_norm(ctx, x, None, add=x, total=x)
    assert bool((x == 2).all())
