"""ien_rms_norm of rows whose root has no normal reciprocal in f32: subnormal rows without
an epsilon, and rows near f32's end.  The tolerance is test_gpu_rms_norm's: moving a row
by a power of two rounds nothing."""

import numpy as np
import pytest

import eight_bits as E
import expert_forms as X
from test_gpu_eight_bits import cuda, strided
from test_gpu_rms_norm import SIZES, close

pytestmark = pytest.mark.gpu

SCALES = [2.0**-149, 2.0**-140, 1e-40, 2.0**-127, 2.0**-126, 2.0**-125, 1.0, 2.0**125, 2.0**126, 1.1e38, 1.9e38]


@pytest.mark.parametrize("r,c", SIZES)
@pytest.mark.parametrize("into,added", [(np.float32, None), (np.float32, np.float16), (np.float32, np.float32), (np.float16, np.float32)])
@pytest.mark.parametrize("outof", [np.float16, np.float32])
def test_far_rows(ctx, r, c, into, added, outof):
    import ien
    import torch

    rng = np.random.default_rng(c + r)
    rows = len(SCALES) * min(r, 9)
    s = rng.integers(-7, 8, (rows, c)).astype(np.float64) / 4
    s[:, 0] = 1.75
    with np.errstate(under="ignore"):
        s = (s * np.tile(SCALES, rows // len(SCALES))[:, None]).astype(np.float32)
    assert np.isfinite(s).all() and (np.abs(s).max(1) > 0).all()
    x, a = s, None
    if added == np.float32:
        x, a = np.zeros((rows, c), into), s
    elif added == np.float16:
        a = np.zeros((rows, c), np.float16)
    gamma = (1 + 0.2 * rng.standard_normal(c)).astype(np.float32)
    total, y, q = strided(np.zeros((rows, c), into), 3, 7.0), strided(np.zeros((rows, c), outof), 3, 7.0), ien.Rows8(rows, c)
    ien.rms_norm(ctx, cuda(x), cuda(gamma), y, q, add=None if a is None else cuda(a), total=total, eps=0.0)
    with np.errstate(over="ignore"):
        assert np.array_equal(total.cpu().numpy(), s.astype(into))
    close(y.cpu().numpy(), X.rms_norm(s, gamma, 0.0), outof)
    y32 = torch.empty(rows, c, dtype=torch.float32, device="cuda")
    ien.rms_norm(ctx, cuda(x), cuda(gamma), y32, add=None if a is None else cuda(a), eps=0.0)
    data, scales = E.quantize(y32.cpu().numpy())
    assert np.array_equal(q.data.cpu().numpy(), data) and np.array_equal(q.scales[:, :scales.shape[1]].cpu().numpy(), scales)


def test_rows_without_a_root(ctx):
    """Zeros without an epsilon, and infinities, beside far rows of the same wave: as before."""
    import ien
    import torch

    x = np.full((5, 24), 1e-40, np.float32)
    x[1] = 0
    x[2, 3] = np.inf
    x[3, 4] = np.nan
    x[4] = 3e38
    y = torch.empty(5, 24, device="cuda")
    ien.rms_norm(ctx, cuda(x), None, y, eps=0.0)
    got = y.cpu().numpy()
    assert np.abs(got[[0, 4]] - 1).max() <= 2.0**-22 and np.isnan(got[[1, 3]]).all()
    assert np.isnan(got[2, 3]) and (np.delete(got[2], 3) == 0).all()
