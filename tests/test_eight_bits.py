"""Rows in 8 bits, their products and group norm without a GPU: sizes, what
the entry points refuse (before they touch the device), and the definitions
that the GPU tests compare with."""

import ctypes

import numpy as np
import pytest

import eight_bits as E
import ien


class FakeMatrix8(ctypes.Structure):
    """The fields of ien_matrix8 that a refusal reads."""
    _fields_ = [("ctx", ctypes.c_void_p), ("taps", ctypes.c_size_t), ("c", ctypes.c_size_t), ("n", ctypes.c_size_t),
                ("cb", ctypes.c_int), ("npad", ctypes.c_long), ("w", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("bias", ctypes.c_void_p)]


CTX = ctypes.create_string_buffer(4096)  # never read by a call that is refused
P = 0x10000  # an aligned address, never read either


def matrix(taps=1, c=200, n=24):
    m = FakeMatrix8(None, taps, c, n, -(-c // 128), 128, P, P, P)
    return ctypes.byref(m)


def rows8(data=P, stride=256, scales=P, scale_stride=4):
    return ien.Rows8Struct(data, stride, scales, scale_stride)


def refused(status):
    assert status == ien.ERR_INPUT
    assert ien.load().ien_last_error().startswith(b"input: ")


def test_strides():
    L = ien.load()
    assert [L.ien_rows8_stride(k) for k in (1, 128, 129, 640)] == [128, 128, 256, 640]
    assert [L.ien_rows8_scale_stride(k) for k in (1, 512, 513, 4096)] == [4, 4, 8, 32]


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(x=None), dict(type=2), dict(stride=199), dict(k=1 << 30), dict(out=None),
    dict(out=rows8(data=None)), dict(out=rows8(scales=None)), dict(out=rows8(data=P + 8)),
    dict(out=rows8(scales=P + 2)), dict(out=rows8(stride=240)), dict(out=rows8(stride=264)),
    dict(out=rows8(scale_stride=2)), dict(out=rows8(scale_stride=0))])
def test_quantize8_refusals(bad):
    a = dict(ctx=CTX, x=P, type=ien.OUT_F16, rows=3, k=200, stride=200, out=rows8()) | bad
    out = None if a["out"] is None else ctypes.byref(a["out"])
    L = ien.load()
    refused(L.ien_quantize8(a["ctx"], a["x"], a["type"], a["rows"], a["k"], a["stride"], out))
    refused(L.ien_dequantize8(a["ctx"], out, a["rows"], a["k"], a["x"], a["type"], a["stride"]))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(w=None), dict(type=7), dict(taps=0), dict(taps=4), dict(c=0), dict(n=0), dict(c=1 << 22),
    dict(n=1 << 22), dict(out=False)])
def test_matrix8_refusals(bad):
    a = dict(ctx=CTX, w=P, type=ien.W_F32, taps=1, c=8, n=8, out=True) | bad
    h = ctypes.c_void_p()
    refused(ien.load().ien_matrix8_new(a["ctx"], a["w"], a["type"], a["taps"], a["c"], a["n"], None,
                                       ctypes.byref(h) if a["out"] else None))
    ien.load().ien_matrix8_free(None)


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(m=None), dict(act=ien.ACT_PRELU), dict(act=6), dict(act=-1), dict(type=2),
    dict(layout=ien.NCHW), dict(y=None), dict(stride=23), dict(add=P, add_stride=23), dict(kind=2), dict(step=0),
    dict(step=3), dict(rows=36), dict(row0=36), dict(row0=30, rows=6), dict(step=2, rows=13),
    dict(kind=ien.INPUT_ROWS), dict(map=rows8(data=P + 4)), dict(map=rows8(stride=128)),
    dict(map=rows8(scale_stride=6)), dict(width=1 << 20), dict(images=1 << 20)])
def test_multiply8_refusals(bad):
    # 1 map of 7 x 5 pixels, 3 x 3 taps.
    a = dict(ctx=CTX, m=matrix(taps=9), kind=ien.INPUT_IMAGE, map=rows8(), images=1, height=7, width=5, step=1, row0=0,
             rows=35, y=P, stride=24, layout=ien.NHWC, type=ien.OUT_F16, act=ien.ACT_NONE, add=None, add_stride=0) | bad
    inp = ien.Input8(a["kind"], a["map"], a["images"], a["height"], a["width"], a["step"])
    out = ien.Output(a["y"], a["stride"], a["layout"], a["type"])
    refused(ien.load().ien_multiply8(a["ctx"], ctypes.byref(inp), a["row0"], a["rows"], a["m"], ctypes.byref(out),
                                     a["act"], a["add"], a["add_stride"]))


NORM = dict(ctx=CTX, x=P, type=ien.OUT_F16, images=2, pixels=5, c=200, stride=200, groups=8, eps=1e-5,
            act=ien.ACT_SILU, y=P + 4096, y_type=ien.OUT_F16, y_stride=200, out=rows8())


def norm(a):
    L = ien.load()
    first = (a["ctx"], a["x"], a["type"], a["images"], a["pixels"], a["c"], a["stride"], a["groups"], None, None,
             a["eps"], a["act"])
    return (lambda: L.ien_group_norm(*first, a["y"], a["y_type"], a["y_stride"]),
            lambda: L.ien_group_norm8(*first, None if a["out"] is None else ctypes.byref(a["out"])))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(x=None), dict(type=2), dict(c=0), dict(c=8200, groups=1), dict(groups=0), dict(groups=7),
    dict(stride=199), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(act=ien.ACT_PRELU),
    dict(act=9), dict(images=1 << 20), dict(pixels=1 << 40), dict(stride=1 << 31)])
def test_group_norm_refusals(bad):
    for call in norm(NORM | bad):
        refused(call())


def test_group_norm_refusals_of_the_result():
    for bad in (dict(y=None), dict(y_type=2), dict(y_stride=199), dict(y=P, y_type=ien.OUT_F32),
                dict(y=P, y_stride=208), dict(y_stride=1 << 31)):
        refused(norm(NORM | bad)[0]())
    for bad in (dict(out=None), dict(out=rows8(stride=128)), dict(out=rows8(data=P + 1))):
        refused(norm(NORM | bad)[1]())


def test_nothing_to_do():
    L = ien.load()
    q = rows8()
    assert L.ien_quantize8(CTX, None, ien.OUT_F16, 0, 8, 8, ctypes.byref(q)) == ien.OK
    assert L.ien_dequantize8(CTX, ctypes.byref(q), 0, 8, None, ien.OUT_F16, 8) == ien.OK
    assert all(call() == ien.OK for call in norm(NORM | dict(images=0)) + norm(NORM | dict(pixels=0)))
    inp, out = ien.Input8(ien.INPUT_ROWS, q, 1, 1, 1, 1), ien.Output(P, 24, ien.NHWC, ien.OUT_F16)
    assert L.ien_multiply8(CTX, ctypes.byref(inp), 0, 0, matrix(), ctypes.byref(out), ien.ACT_NONE, None, 0) == ien.OK


def test_f16_products_refuse_silu():
    inp, out = ien.Input(), ien.Output(P, 24, ien.NHWC, ien.OUT_F16)
    refused(ien.load().ien_multiply_ex(CTX, ctypes.byref(inp), 0, 1, P, ctypes.byref(out), ien.ACT_SILU, None, 0))


def test_bindings_refuse():
    import types

    import torch

    ctx = types.SimpleNamespace(h=None)
    x, q = torch.zeros(6, 40, dtype=torch.float16), ien.Rows8(6, 40, device="cpu")
    with pytest.raises(ValueError):
        ien.quantize8(ctx, x[:5], q)
    with pytest.raises(ValueError):
        ien.quantize8(ctx, x.double(), q)
    with pytest.raises(ValueError):
        ien.dequantize8(ctx, q, x.t())
    with pytest.raises(ValueError):
        ien.group_norm(ctx, x, 4, 8, None, None, q)
    with pytest.raises(ValueError):
        ien.group_norm(ctx, x, 1, 8, torch.ones(39), None, q)
    with pytest.raises(ValueError):
        ien.Rows8(6, 40, data=torch.zeros(5, 128, dtype=torch.uint8))


def test_definition_of_8_bits():
    """The oracle's own rounding: every e4m3 value stands for itself, ties go to
    even, and a block's scale is the smallest that holds it."""
    own = np.array([b for b in range(256) if b & 127 != 127], np.uint8)
    assert np.array_equal(E.to_bytes(E.E4M3[own]), own)
    assert np.array_equal(E.to_bytes(np.array([17.0, 19.0, 432.0, 2.0**-10, 3 * 2.0**-10])),
                          E.to_bytes(np.array([16.0, 20.0, 448.0, 0.0, 2.0**-8])))
    x = np.zeros((5, 130), np.float32)
    x[:, 3] = [448, 449, 0, 2.0**-140, 3.0e38]
    _, s = E.quantize(x)
    assert s.tolist() == [[127, 127], [128, 127], [127, 127], [0, 127], [247, 127]]
