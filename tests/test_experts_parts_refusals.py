"""What the experts' second product with a branch, or with products of another type
than its result's, refuses: without a GPU."""

import ctypes

import pytest
import torch

import ien
from test_eight_bits import CTX, P, refused, rows8
from test_experts_refusals import F16, F32, BOUND, OnGpu, Somewhere, experts, routes

L = ien.load()


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(w=experts(gated=1)), dict(parts=None), dict(parts=P + 8), dict(parts_type=2), dict(type=F32, parts_type=F16), dict(type=2),
    dict(type=2, parts_type=2), dict(branch_stride=23), dict(branch_type=3), dict(add_stride=23), dict(stride=8), dict(h=rows8(data=None)),
    dict(r=routes(top=5)), dict(layout=ien.NCHW), dict(y=None)])
def test_out8_ex(bad):
    a = dict(ctx=CTX, h=rows8(), r=routes(), w=experts(), parts=P, parts_type=F32, add=P, add_stride=24, branch=P, branch_type=F16,
             branch_stride=24, y=P, stride=24, layout=ien.NHWC, type=F16) | bad
    out = ien.Output(a["y"], a["stride"], a["layout"], a["type"])
    refused(L.ien_experts_out8_ex(a["ctx"], ctypes.byref(a["h"]), a["r"], a["w"], 0, a["parts"], a["parts_type"], a["add"], a["add_stride"],
                                  a["branch"], a["branch_type"], a["branch_stride"], ctypes.byref(out)))
    refused(L.ien_experts_out8_ex(CTX, ctypes.byref(rows8()), routes(), experts(), 0, P, F32, None, 0, None, F16, 0, None))


def test_bindings():
    m = type("Experts8", (), dict(h=None, experts=4, c=40, n=24, ctx=BOUND))()
    here = ien.Routes(6, 4, 2, device="cpu")
    here._device = 0
    h, y, y32 = Somewhere(12, 40, 0), OnGpu(6, 24), OnGpu(6, 24, 0, torch.float32)

    class Parts(OnGpu):
        def is_contiguous(self):
            return True

        def numel(self):
            return self.shape[0] * self.shape[1]

    parts = lambda n=24, dtype=torch.float32, device=0: Parts(12, n, device, dtype)  # noqa: E731
    for call in (lambda: ien.experts_out8(BOUND, h, here, m, parts(23), y), lambda: ien.experts_out8(BOUND, h, here, m, parts(device=1), y),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(dtype=torch.float16), y32),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(dtype=torch.bfloat16), y),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(), y, add=y32),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(), y, branch=OnGpu(6, 23)),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(), y, branch=OnGpu(5, 24)),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(), y, branch=OnGpu(6, 24, 1)),
                 lambda: ien.experts_out8(BOUND, h, here, m, parts(), y, branch=OnGpu(6, 24, 0, torch.bfloat16))):
        with pytest.raises(ValueError):
            call()
