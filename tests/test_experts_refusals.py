"""What the norm, the router and the experts' products refuse before they touch the
device, the sizes of plans, and the choice of tiles: without a GPU."""

import ctypes

import pytest
import torch

import ien
from internal import _function
from test_eight_bits import CTX, P, refused, rows8
from test_rows8_bindings import CTX as BOUND, OnGpu, Somewhere

L = ien.load()
F16, F32 = ien.OUT_F16, ien.OUT_F32


class FakeExperts(ctypes.Structure):
    """The fields of ien_experts8 that a refusal reads."""
    _fields_ = [("ctx", ctypes.c_void_p), ("experts", ctypes.c_size_t), ("c", ctypes.c_size_t), ("n", ctypes.c_size_t),
                ("gated", ctypes.c_int), ("cb", ctypes.c_int), ("npad", ctypes.c_long), ("w", ctypes.c_void_p),
                ("scales", ctypes.c_void_p), ("bias", ctypes.c_void_p)]


def experts(gated=0, c=200, n=24, npad=128, w=P, many=4):
    return ctypes.byref(FakeExperts(None, many, c, n, gated, -(-c // 128), npad, w, P, P))


def routes(tokens=6, many=4, top=2, index=P, weight=P, plan=P):
    return ctypes.byref(ien.RoutesStruct(tokens, many, top, index, weight, plan))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(x=None), dict(type=2), dict(add_type=3), dict(y_type=-1), dict(c=8193, stride=9000), dict(stride=199),
    dict(add_stride=199), dict(sum_stride=100), dict(y_stride=0), dict(eps=-1.0), dict(eps=float("nan")), dict(rows=1 << 40),
    dict(out=rows8(data=None)), dict(out=rows8(data=P + 8)), dict(out=rows8(stride=240)), dict(out=rows8(scale_stride=2))])
def test_rms_norm(bad):
    a = dict(ctx=CTX, x=P, type=F16, rows=3, c=200, stride=200, add=P, add_type=F32, add_stride=200, sum=P, sum_stride=200,
             gamma=P, eps=1e-6, y=P, y_type=F16, y_stride=200, out=rows8()) | bad
    refused(L.ien_rms_norm(a["ctx"], a["x"], a["type"], a["rows"], a["c"], a["stride"], a["add"], a["add_type"], a["add_stride"],
                           a["sum"], a["sum_stride"], a["gamma"], a["eps"], a["y"], a["y_type"], a["y_stride"],
                           ctypes.byref(a["out"])))


BAD_ROUTES = [dict(top=0), dict(top=5), dict(top=17, many=64), dict(many=0), dict(many=1025), dict(tokens=(1 << 27) + 1), dict(index=None),
              dict(weight=None), dict(plan=None), dict(plan=P + 8), dict(index=P + 2), dict(weight=P + 1)]


@pytest.mark.parametrize("bad", BAD_ROUTES)
def test_routes(bad):
    r = routes(**bad)
    how = ien.Router(0, None, 1, 1, 1, 1, 1.0)
    refused(L.ien_routes_plan(CTX, r))
    refused(L.ien_route(CTX, P, F32, 64, ctypes.byref(how), r))
    refused(L.ien_experts_in8(CTX, ctypes.byref(rows8()), r, experts(many=bad.get("many", 4)), 0, 0, ctypes.byref(rows8(stride=128))))
    out = ien.Output(P, 24, ien.NHWC, F16)
    refused(L.ien_experts_out8(CTX, ctypes.byref(rows8()), r, experts(many=bad.get("many", 4)), 0, P, None, 0, ctypes.byref(out)))


def test_no_routes():
    refused(L.ien_routes_plan(CTX, None))
    refused(L.ien_routes_plan(None, routes()))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(logits=None), dict(type=5), dict(stride=3), dict(score=2), dict(groups=0), dict(groups=3), dict(kept=0),
    dict(kept=3, groups=2), dict(group_top=0), dict(group_top=3)])
def test_route(bad):
    a = dict(ctx=CTX, logits=P, type=F32, stride=4, score=0, groups=1, kept=1, group_top=1) | bad
    how = ien.Router(a["score"], None, a["groups"], a["kept"], a["group_top"], 1, 1.0)
    refused(L.ien_route(a["ctx"], a["logits"], a["type"], a["stride"], ctypes.byref(how), routes()))
    refused(L.ien_route(CTX, P, F32, 4, None, routes()))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(w=None), dict(type=2), dict(many=0), dict(many=1025), dict(c=0), dict(n=0), dict(c=1 << 22), dict(n=1 << 22),
    dict(n=25, gated=1), dict(many=1024, c=8192), dict(c=1 << 21, n=1 << 15), dict(out=False)])
def test_weights(bad):
    a = dict(ctx=CTX, w=P, type=ien.W_F32, many=4, c=200, n=24, gated=0, out=True) | bad
    h = ctypes.c_void_p()
    refused(L.ien_experts8_new(a["ctx"], a["w"], a["type"], a["many"], a["c"], a["n"], a["gated"], P,
                               ctypes.byref(h) if a["out"] else None))
    L.ien_experts8_free(None)


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(w=None), dict(w=experts(w=None)), dict(w=experts(many=5)), dict(act=3), dict(act=9), dict(x=rows8(data=None)),
    dict(x=rows8(stride=128)), dict(x=rows8(stride=1 << 20)), dict(x=rows8(scale_stride=1 << 20)), dict(out=rows8(data=P + 4)),
    dict(out=rows8(stride=1 << 20)), dict(out=rows8(stride=64)), dict(r=routes(tokens=1 << 23))])
def test_in8(bad):
    a = dict(ctx=CTX, x=rows8(), r=routes(), w=experts(), act=0, out=rows8(stride=128)) | bad
    refused(L.ien_experts_in8(a["ctx"], ctypes.byref(a["x"]), a["r"], a["w"], a["act"], 0, ctypes.byref(a["out"])))


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(w=None), dict(w=experts(w=None)), dict(w=experts(many=5)), dict(w=experts(gated=1)), dict(h=rows8(data=None)),
    dict(h=rows8(stride=128)), dict(h=rows8(stride=1 << 20)), dict(parts=None), dict(parts=P + 8), dict(stride=23), dict(add_stride=8),
    dict(type=2), dict(layout=ien.NCHW), dict(y=None)])
def test_out8(bad):
    a = dict(ctx=CTX, h=rows8(), r=routes(), w=experts(), parts=P, add=P, add_stride=24, y=P, stride=24, layout=ien.NHWC, type=F16) | bad
    out = ien.Output(a["y"], a["stride"], a["layout"], a["type"])
    refused(L.ien_experts_out8(a["ctx"], ctypes.byref(a["h"]), a["r"], a["w"], 0, a["parts"], a["add"], a["add_stride"], ctypes.byref(out)))
    refused(L.ien_experts_out8(CTX, ctypes.byref(rows8()), routes(), experts(), 0, P, None, 0, None))


def test_more_tiles_than_a_launch_has():
    """In place of a launch of 2^32 lanes or more: 2^27 pairs by 2^20 columns."""
    wide = experts(n=1 << 20, npad=1 << 20)
    many = routes(tokens=1 << 23, top=4)
    refused(L.ien_experts_in8(CTX, ctypes.byref(rows8(stride=256)), routes(tokens=8 << 19, top=4), wide, 0, 0,
                              ctypes.byref(rows8(stride=(1 << 20) - 128, scale_stride=4 * (1 << 13)))))
    out = ien.Output(P, 1 << 20, ien.NHWC, F16)
    refused(L.ien_experts_out8(CTX, ctypes.byref(rows8()), many, wide, 0, P, None, 0, ctypes.byref(out)))


def test_parts():
    assert L.ien_experts_parts(routes(tokens=6, top=2), experts(n=24)) == 6 * 2 * 24
    assert L.ien_experts_parts(routes(tokens=5, top=3), experts(n=25)) == 5 * 3 * 32
    assert L.ien_experts_parts(None, experts()) == 0 and L.ien_experts_parts(routes(), None) == 0


@pytest.mark.parametrize("experts_", [1, 2, 63, 64, 1000, 1024])
@pytest.mark.parametrize("tokens", [0, 1, 64, 65, 16384, 16385, 100001, 1 << 24])
def test_plans_fit_their_ints(tokens, experts_):
    """Room for offsets, order, places, tiles of four sizes and the chunks' counts; none for what is refused."""
    for top in (1, min(experts_, 16)):
        pairs = tokens * top
        tiles = sum(4 * (pairs // s + min(pairs, experts_)) for s in (16, 64, 128, 256))
        least = experts_ + 1 + 2 * pairs + 4 + tiles + max(1, min(256, -(-tokens // 64)) // 2) * (experts_ + 1)
        got = L.ien_routes_ints(tokens, experts_, top)
        assert least <= got <= least + 256 * (experts_ + 4) + 64
        assert L.ien_routes_order(experts_) >= experts_ + 1 and L.ien_routes_order(experts_) % 4 == 0
    assert L.ien_routes_ints(tokens, 0, 1) == L.ien_routes_ints(tokens, 1025, 1) == L.ien_routes_ints(tokens, 64, 17) == 0
    assert L.ien_routes_ints((1 << 28) + 1, 64, 1) == 0


in_choice = _function("_ZN3ien17experts_in_choiceEilllii", ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int,
                      ctypes.c_int)
out_choice = _function("_ZN3ien18experts_out_choiceElli", ctypes.c_long, ctypes.c_long, ctypes.c_int)


def test_choices_for_every_size():
    """Some tile for any pairs, experts, columns and depth; larger ones for more rows."""
    seen = set()
    for many in (1, 8, 64, 1024):
        for pairs in (1, 2, 7, 8, 9, 100, 1000, 10**4, 10**5, 10**6, 1 << 28):
            for npad in (128, 256, 1536, 8192, 1 << 20):
                for chunks in (1, 3, 8, 64):
                    for gated in (0, 1):
                        c = in_choice(256, pairs, many, npad, chunks, gated)
                        assert 0 <= c <= (3 if gated else 2)
                        seen.add((gated, c))
                    assert 0 <= out_choice(pairs, many, chunks) <= 3
    assert seen == {(1, k) for k in range(4)} | {(0, k) for k in range(3)}
    assert in_choice(256, 8, 64, 4096, 8, 1) == 0 and in_choice(256, 65536, 32, 4096, 8, 1) == 3
    assert in_choice(256, 8, 64, 4096, 8, 0) == 0 and in_choice(256, 65536, 32, 4096, 8, 0) == 2
    assert out_choice(8, 64, 16) == 3 and out_choice(8, 64, 8) == 0 and out_choice(65536, 32, 16) == 2


def test_bindings_refuse():
    h, h32 = OnGpu(6, 40), OnGpu(6, 40, 0, torch.float32)
    q = Somewhere(6, 40, 0)
    for call in (lambda: ien.rms_norm(BOUND, h, None, add=OnGpu(5, 40)), lambda: ien.rms_norm(BOUND, h, None, add=OnGpu(6, 41)),
                 lambda: ien.rms_norm(BOUND, h, None, total=h32), lambda: ien.rms_norm(BOUND, h, None, OnGpu(6, 8)),
                 lambda: ien.rms_norm(BOUND, h, None, None, Somewhere(6, 41, 0)),
                 lambda: ien.rms_norm(BOUND, h, OnGpu(1, 39, 0, torch.float32, flat=True))):
        with pytest.raises(ValueError):
            call()
    for there in (OnGpu(6, 40, 1),):
        for call in (lambda: ien.rms_norm(BOUND, there, None), lambda: ien.rms_norm(BOUND, h, None, add=there),
                     lambda: ien.rms_norm(BOUND, h, None, total=there), lambda: ien.rms_norm(BOUND, h, None, there),
                     lambda: ien.rms_norm(BOUND, h, None, None, Somewhere(6, 40, 1)),
                     lambda: ien.rms_norm(BOUND, h, OnGpu(1, 40, 1, torch.float32, flat=True))):
            with pytest.raises(ValueError, match="GPU 0"):
                call()
    host = ien.Routes(6, 4, 2, device="cpu")
    for bad in (dict(index=torch.zeros(6, 3, dtype=torch.int32)), dict(index=torch.zeros(6, 2)), dict(weight=torch.zeros(6, 2, dtype=torch.float16)),
                dict(index=torch.zeros(2, 6, dtype=torch.int32).t())):
        with pytest.raises(ValueError):
            ien.Routes(6, 4, 2, device="cpu", **bad)
    for size in ((6, 4, 5), (6, 0, 1), (6, 2000, 1)):
        with pytest.raises(ValueError):
            ien.Routes(*size, device="cpu")
    assert host.offsets.tolist() == [0] * 5 and host.order.tolist() == [0] * 12
    with pytest.raises(ValueError, match="GPU 0"):
        ien.plan_routes(BOUND, host)
    with pytest.raises(ValueError, match="GPU 0"):
        ien.route(BOUND, OnGpu(6, 4), host)
    with pytest.raises(ValueError):
        ien.route(BOUND, OnGpu(6, 5), host)
    for bad in (dict(groups=0), dict(groups=-2), dict(kept=-1, groups=2), dict(group_top=-1)):
        with pytest.raises(ValueError):
            here = ien.Routes(6, 4, 2, device="cpu")
            here._device = 0
            ien.route(BOUND, OnGpu(6, 4), here, **bad)

    m = type("Experts8", (), dict(h=None, experts=4, c=40, n=24, ctx=BOUND))()
    here = ien.Routes(6, 4, 2, device="cpu")
    here._device = 0
    other = type("Experts8", (), dict(h=None, experts=4, c=40, n=24, ctx=type("C", (), dict(h=None, device=1))()))()
    for call in (lambda: ien.experts_in8(BOUND, Somewhere(5, 40, 0), here, m, Somewhere(12, 24, 0)),
                 lambda: ien.experts_in8(BOUND, q, here, m, Somewhere(6, 24, 0)), lambda: ien.experts_in8(BOUND, q, here, m, Somewhere(12, 25, 0)),
                 lambda: ien.experts_in8(BOUND, q, ien.Routes(6, 5, 2, device="cpu"), m, Somewhere(12, 24, 0)),
                 lambda: ien.experts_in8(BOUND, q, host, m, Somewhere(12, 24, 0)), lambda: ien.experts_in8(BOUND, q, here, other, Somewhere(12, 24, 0)),
                 lambda: ien.experts_in8(BOUND, q, here, m, Somewhere(12, 24, 1)),
                 lambda: ien.experts_out8(BOUND, q, here, m, None, OnGpu(6, 24)),
                 lambda: ien.experts_out8(BOUND, Somewhere(12, 40, 0), here, m, None, OnGpu(5, 24)),
                 lambda: ien.experts_out8(BOUND, Somewhere(12, 40, 0), here, m, torch.zeros(500, dtype=torch.float16), OnGpu(6, 24))):
        with pytest.raises(ValueError):
            call()
