"""What the bindings of the 8-bit entry points refuse before the library is asked:
tensors too narrow for the rows they hold, and tensors that are not on the
context's GPU."""

import pytest
import torch

import ien


def byte_rows(rows, width, of=None):
    return torch.zeros(rows, of or width, dtype=torch.uint8)[:, :width]


@pytest.mark.parametrize("rows,k,width,scale_width", [
    (6, 640, 128, 8), (6, 640, 639, 8), (6, 640, 640, 4), (6, 40, 127, 4), (6, 40, 128, 3), (1, 129, 128, 4), (1, 513, 640, 7),
    (6, 1, 0, 4)])
@pytest.mark.parametrize("wide", [0, 4096])
def test_rows8_refuses_narrow_tensors(rows, k, width, scale_width, wide):
    """Also as a part of wide enough rows, which is no row of its own."""
    with pytest.raises(ValueError, match="bytes"):
        ien.Rows8(rows, k, data=byte_rows(rows, width, wide), scales=byte_rows(rows, scale_width, wide))


def test_rows8_takes_wide_enough_tensors():
    q = ien.Rows8(6, 640, data=byte_rows(6, 640, 1024), scales=byte_rows(6, 8))
    assert q._fields[1] == 1024 and q._fields[3] == 8
    assert ien.Rows8(0, 640, data=byte_rows(0, 640), scales=byte_rows(0, 8)).rows == 0
