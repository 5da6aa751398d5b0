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


class OnGpu:
    """What the bindings read of a tensor on GPU `index`; its address is never followed."""

    def __init__(self, rows, c, index=0, dtype=torch.float16, flat=False):
        self.shape, self._strides = ((c,), (1,)) if flat else ((rows, c), (c, 1))
        self.index, self.dtype, self.is_cuda, self.device = index, dtype, True, f"cuda:{index}"

    def stride(self):
        return self._strides

    def data_ptr(self):
        return 0x10000

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True


class Somewhere(ien.Rows8):
    """Rows on GPU `index` (-1: the host) without tensors there."""

    def __init__(self, rows, k, index):
        super().__init__(rows, k, device="cpu")
        self._device = index


CTX = type("Context", (), dict(h=None, device=0))()
OTHER = type("Context", (), dict(h=None, device=1))()


def calls(x, q, gamma=None, matrix_ctx=CTX):
    m = type("Matrix8", (), dict(h=None, c=40, n=40, taps=1, ctx=matrix_ctx))()
    return [lambda: ien.quantize8(CTX, x, q), lambda: ien.dequantize8(CTX, q, x),
            lambda: ien.multiply8(CTX, q, m, x), lambda: ien.conv8(CTX, q, 1, 2, 3, m, x),
            lambda: ien.group_norm(CTX, x, 1, 8, gamma, None, q), lambda: ien.group_norm(CTX, x, 1, 8, None, gamma, q)]


@pytest.mark.parametrize("index", [-1, 1])
def test_rows8_of_the_host_or_another_gpu(index):
    for call in calls(OnGpu(6, 40), Somewhere(6, 40, index)):
        with pytest.raises(ValueError, match="GPU 0"):
            call()


def test_tensors_of_another_gpu():
    here, there = OnGpu(6, 40), OnGpu(6, 40, 1)
    for call in calls(there, Somewhere(6, 40, 0)):
        with pytest.raises(ValueError, match="GPU 0"):
            call()
    for call in calls(here, Somewhere(6, 40, 0), OnGpu(1, 40, 1, torch.float32, flat=True))[4:]:
        with pytest.raises(ValueError, match="GPU 0"):
            call()
    for call in calls(here, Somewhere(6, 40, 0), matrix_ctx=OTHER)[2:4]:
        with pytest.raises(ValueError, match="GPU 0"):
            call()
    m = type("Matrix8", (), dict(h=None, c=40, n=40, taps=1, ctx=CTX))()
    for call in (lambda: ien.multiply8(CTX, Somewhere(6, 40, 0), m, here, add=there),
                 lambda: ien.group_norm(CTX, here, 1, 8, None, None, there)):
        with pytest.raises(ValueError, match="GPU 0"):
            call()


def test_tensors_of_the_contexts_gpu_reach_the_library():
    """(Which refuses: these contexts hold none of its own.)"""
    for call in calls(OnGpu(6, 40), Somewhere(6, 40, 0), OnGpu(1, 40, 0, torch.float32, flat=True)):
        with pytest.raises(ien.IenError):
            call()
