"""Routing with biases far larger than a score: experts switched off by the type's
lowest value or some large negative one, and such that are preferred.  As in
test_gpu_route, experts, offsets and order are compared for equality."""

import numpy as np
import pytest

from test_gpu_eight_bits import cuda
from test_gpu_route import check
from test_gpu_route_lowest_biases import GROUPS, LOWEST

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,groups,kept,top", GROUPS + [(16, 1, 1, 4), (256, 1, 1, 8), (40, 1, 1, 16), (300, 1, 1, 8)])
@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("far", [-1e9, -1e4, 1e4, 3e7])
@pytest.mark.parametrize("share", [0.05, 0.9])
def test_far_biases(ctx, softmax, experts, groups, kept, top, far, share):
    """Some or most experts' choices end above the scores' last bits: their order is that of the sums in f64."""
    rng = np.random.default_rng(experts + top)
    logits = rng.standard_normal((80, experts)).astype(np.float32)
    logits[50:] = np.round(logits[50:])  # (equal ones)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    bias[rng.random(experts) < share] += far
    for group_top in (1, 2):
        check(ctx, logits, top, softmax, bias=bias, groups=groups, kept=kept, group_top=group_top)


@pytest.mark.parametrize("softmax", [True, False])
def test_choices_that_f32_cannot_tell_apart_beside_far_ones(ctx, softmax):
    """Neighbouring sums in f32, of the wanted size, of a far one, and in groups of both."""
    rng = np.random.default_rng(2)
    base = np.float32(0.125 if softmax else 3.0)
    steps = np.stack([rng.permutation(64) for _ in range(100)])
    logits = (base + steps * np.spacing(base)).astype(np.float32)
    for bias in (1.0, 4096.0, -2.0**24):
        b = np.full(64, bias, np.float32)
        b[::7] = -1e9
        check(ctx, logits, 8, softmax, bias=b)
        check(ctx, logits, 8, softmax, bias=b, groups=8, kept=2, group_top=2)
        check(ctx, logits, 4, softmax, bias=b, groups=16, kept=3, group_top=2)


@pytest.mark.parametrize("groups", [1, 8])
@pytest.mark.parametrize("far", [-1e9, -1e4, LOWEST])
def test_experts_switched_off_cost_nothing(ctx, groups, far):
    """A choice in f64 for every token, where none is needed, took five times as long."""
    import ien
    import torch

    rng = np.random.default_rng(8)
    logits, routes = cuda(rng.standard_normal((32768, 256)).astype(np.float32)), ien.Routes(32768, 256, 8)
    near = (0.1 * rng.standard_normal(256)).astype(np.float32)
    off = near.copy()
    off[::50] = far
    biases = cuda(near), cuda(off)
    best = [1e30, 1e30]
    for _ in range(10):
        for k, b in enumerate(biases):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(5):
                ien.route(ctx, logits, routes, score=ien.SCORE_SIGMOID, bias=b, groups=groups, kept=min(4, groups), group_top=2)
            end.record()
            end.synchronize()
            best[k] = min(best[k], start.elapsed_time(end))
    assert best[1] < 2 * best[0], best
