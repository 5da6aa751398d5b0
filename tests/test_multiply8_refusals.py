"""What ien_multiply8 refuses because its tiles address rows by 31-bit offsets,
and what the bindings refuse before the library is asked."""

import ctypes
import types

import pytest

import ien
from test_eight_bits import CTX, FakeMatrix8, P, refused, rows8


def call(c, stride, scale_stride=None, width=5, height=7, npad=128, kind=ien.INPUT_IMAGE, rows=1):
    blocks = -(-c // 128)
    m = FakeMatrix8(None, 9 if kind == ien.INPUT_IMAGE else 1, c, 24, blocks, npad, P, P, P)
    inp = ien.Input8(kind, rows8(stride=stride, scale_stride=scale_stride or 4 * -(-blocks // 4)), 1, height, width, 1)
    out = ien.Output(P, 24, ien.NHWC, ien.OUT_F16)
    return ien.load().ien_multiply8(CTX, ctypes.byref(inp), 0, rows, ctypes.byref(m), ctypes.byref(out), ien.ACT_NONE, None, 0)


@pytest.mark.parametrize("kind", [ien.INPUT_ROWS, ien.INPUT_IMAGE])
def test_rows_too_far_apart(kind):
    refused(call(200, 1 << 20, kind=kind))
    refused(call(200, 256, scale_stride=1 << 20, kind=kind))


def test_lines_too_long():
    refused(call(200, 256, width=(1 << 19) - 256))
    refused(call(4096, 1 << 19, width=1))


def test_too_many_weights():
    refused(call(200, 256, npad=1 << 24))


def test_too_many_panels():
    h = ctypes.c_void_p()
    refused(ien.load().ien_matrix8_new(CTX, P, ien.W_F32, 9, 1 << 20, 8, None, ctypes.byref(h)))


def test_bindings_refuse_a_map_that_is_none():
    ctx, q = types.SimpleNamespace(h=None), ien.Rows8(6, 40, device="cpu")
    m = types.SimpleNamespace(h=None, c=40, n=8)
    for shape, step, row0 in (((1, 2, 4), 1, 0), ((-1, -2, 3), 1, 0), ((1, 2, 3), 3, 0), ((1, 2, 3), 0, 0), ((1, 2, 3), 1, -1)):
        with pytest.raises(ValueError):
            ien.conv8(ctx, q, *shape, m, q.data, step=step, row0=row0)
    with pytest.raises(ValueError):
        ien.multiply8(ctx, q, m, q.data, row0=1)


def test_bindings_refuse_tensors_of_the_host():
    import torch

    ctx, q = types.SimpleNamespace(h=None), ien.Rows8(6, 40, device="cpu")
    x = torch.zeros(6, 40)
    for f in (lambda: ien.quantize8(ctx, x, q), lambda: ien.dequantize8(ctx, q, x),
              lambda: ien.group_norm(ctx, x, 1, 8, None, None, q)):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_rows8_keeps_its_tensors():
    q = ien.Rows8(6, 40, device="cpu")
    with pytest.raises(AttributeError):
        q.data = q.scales
