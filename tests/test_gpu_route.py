"""ien_route and ien_routes_plan against their definition, a token and a choice at
a time, in 64 bits.

Experts, offsets and order are compared for equality.  Weights: a score's argument
is rounded by 2^-24 of its size at most, its exponential, the sum over the experts
(positive terms, at most ten additions deep), the quotient, the sum over the chosen,
the second quotient and the scale by some steps each: (32 + 2 |argument|) 2^-24 of
the weight."""

import numpy as np
import pytest

import expert_forms as X
from test_gpu_eight_bits import cuda, strided

pytestmark = pytest.mark.gpu


def check(ctx, logits, top, softmax=True, extra=0, **how):
    import ien
    import torch

    tokens, experts = logits.shape
    routes = ien.Routes(tokens, experts, top)
    routes.index.fill_(77)
    bias = how.get("bias")
    ien.route(ctx, strided(logits, extra), routes, score=ien.SCORE_SOFTMAX if softmax else ien.SCORE_SIGMOID,
              **{**how, "bias": None if bias is None else cuda(bias)})
    index, weight = X.route(logits, top, softmax, **how)
    got = routes.index.cpu().numpy()
    assert np.array_equal(got, index), np.argwhere(got != index)[:5]
    v = logits[np.isfinite(logits)].astype(np.float64)
    reach = (v.max() - v.min() if softmax else np.abs(v).max()) if v.size else 0.0
    w = routes.weight.cpu().numpy().astype(np.float64)
    assert (np.abs(w - weight) <= (32 + 2 * reach) * 2.0**-24 * np.abs(weight) + 1e-37).all()
    offsets, order = X.plan(index, experts)
    assert np.array_equal(routes.offsets.cpu().numpy(), offsets) and np.array_equal(routes.order.cpu().numpy(), order)
    torch.cuda.synchronize()
    return routes


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("tokens,experts,top", [
    (1, 1, 1), (1, 64, 8), (5, 3, 3), (17, 16, 16), (16, 17, 2), (300, 60, 4), (65, 64, 1), (700, 128, 6), (33, 129, 5),
    (400, 256, 8), (31, 257, 8), (40, 1000, 16), (9, 1024, 3), (2500, 8, 2)])
@pytest.mark.parametrize("softmax", [True, False])
def test_route(ctx, dtype, tokens, experts, top, softmax):
    rng = np.random.default_rng(tokens + experts)
    logits = (2 * rng.standard_normal((tokens, experts))).astype(dtype)  # (in f16 many are equal)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    check(ctx, logits, top, softmax)
    check(ctx, logits, top, softmax, extra=3, bias=bias, renormalise=False, scale=2.5)


@pytest.mark.parametrize("experts,groups,kept,top", [(8, 4, 2, 2), (64, 8, 3, 6), (60, 12, 5, 4), (256, 8, 4, 8), (256, 256, 16, 16),
                                                     (96, 3, 3, 8), (512, 16, 1, 16), (1024, 64, 4, 9), (130, 65, 9, 16)])
@pytest.mark.parametrize("softmax,biased,group_top", [(True, False, 1), (False, True, 2), (True, True, 2)])
def test_groups(ctx, experts, groups, kept, top, softmax, biased, group_top):
    rng = np.random.default_rng(experts + groups)
    logits = rng.standard_normal((150, experts)).astype(np.float32)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    check(ctx, logits, top, softmax, bias=bias, groups=groups, kept=kept, group_top=group_top, scale=0.5)


@pytest.mark.parametrize("softmax", [True, False])
def test_equal_choices_go_to_the_lowest_index(ctx, softmax):
    rng = np.random.default_rng(1)
    logits = rng.integers(0, 3, (500, 40)).astype(np.float32)
    check(ctx, logits, 7, softmax)
    check(ctx, logits, 7, softmax, groups=8, kept=3, group_top=2)
    check(ctx, np.zeros((20, 300), np.float32), 16, softmax)


@pytest.mark.parametrize("softmax", [True, False])
def test_choices_that_f32_cannot_tell_apart(ctx, softmax):
    """Neighbouring logits of a large common part, whose scores are equal in f32: the
    larger logit is first, wherever it stands; with a bias, the larger sum."""
    rng = np.random.default_rng(2)
    base = np.float32(0.125 if softmax else 3.0)
    steps = np.stack([rng.permutation(64) for _ in range(200)])
    logits = (base + steps * np.spacing(base)).astype(np.float32)
    check(ctx, logits, 8, softmax)
    check(ctx, logits, 8, softmax, bias=np.full(64, 1.0, np.float32))
    check(ctx, logits, 8, softmax, bias=np.full(64, 1.0, np.float32), groups=8, kept=2, group_top=2)


@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("groups", [1, 5])
def test_experts_that_are_off(ctx, softmax, groups):
    """-infinity and NaN, in logits and biases: fewer than top experts, or none."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((90, 40)).astype(np.float32)
    logits[rng.random((90, 40)) < 0.5] = -np.inf
    logits[rng.random((90, 40)) < 0.1] = np.nan
    logits[4] = -np.inf
    logits[5] = np.nan
    logits[6, 1:] = -np.inf
    logits[7] = np.finfo(np.float32).min  # the type's lowest value is a logit like others
    bias = rng.standard_normal(40).astype(np.float32)
    bias[[2, 9]] = -np.inf
    bias[11] = np.nan
    with np.errstate(over="ignore"):
        for b in (None, bias):
            r = check(ctx, logits, 6, softmax, bias=b, groups=groups, kept=2 if groups > 1 else 1, group_top=2)
            assert (r.index[4:6] == -1).all() and (r.weight[4:6] == 0).all()


def test_infinite_logits_share_the_softmax(ctx):
    logits = np.zeros((2, 20), np.float32)
    logits[0, [3, 17]] = np.inf
    logits[1, 5] = np.inf
    r = check(ctx, logits, 3)
    assert r.index[0].tolist() == [3, 17, 0] and r.weight[0].tolist() == [0.5, 0.5, 0.0] and r.weight[1].tolist() == [1.0, 0.0, 0.0]


@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 1024, 16), (2048, 1, 1), (2049, 4, 1), (1000, 1024, 16),
                                                (70001, 5, 3), (300000, 300, 8)])
def test_plans_of_any_index(ctx, tokens, experts, top):
    """Values that are no expert go last; equal experts by pair; the same every time."""
    import ien
    import torch

    rng = np.random.default_rng(tokens)
    index = np.minimum(rng.integers(-3, experts + 3, (tokens, top)), rng.integers(-1, 2**31 - 1, (tokens, top))).astype(np.int32)
    index[rng.random((tokens, top)) < 0.01] = np.iinfo(np.int32).min
    routes = ien.Routes(tokens, experts, top, index=cuda(index))
    for _ in range(3):
        ien.plan_routes(ctx, routes)
        offsets, order = X.plan(index, experts)
        assert np.array_equal(routes.offsets.cpu().numpy(), offsets)
        assert np.array_equal(routes.order.cpu().numpy(), order)
    torch.cuda.synchronize()


def test_no_tokens(ctx):
    import ien
    import torch

    ien.route(ctx, torch.empty(0, 8, device="cuda"), ien.Routes(0, 8, 2))
    ien.plan_routes(ctx, ien.Routes(0, 8, 2))


@pytest.mark.parametrize("per,many", [(16, 2), (16, 4), (16, 8), (16, 13), (16, 16), (32, 2), (32, 3), (32, 8), (64, 2), (64, 3),
                                      (64, 4), (128, 2), (64, 7), (64, 16), (128, 5), (256, 3), (512, 2), (48, 5)])
@pytest.mark.parametrize("softmax,biased,group_top", [(True, False, 1), (False, True, 2), (False, False, 2)])
def test_groups_of_whole_lanes(ctx, per, many, softmax, biased, group_top):
    """Groups of some experts of every lane, with equal ones, and with experts and whole groups that are off."""
    rng = np.random.default_rng(per + many)
    experts = per * many
    logits = rng.standard_normal((90, experts)).astype(np.float32)
    logits[:30] = rng.integers(0, 3, (30, experts))
    logits[30:60][rng.random((30, experts)) < 0.7] = -np.inf
    for t in range(40, 60):
        logits[t].reshape(many, per)[rng.integers(0, many)] = np.nan
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    if biased:
        bias[rng.integers(0, experts, 5)] = -np.inf
    for kept in {1, (many + 1) // 2, many - 1}:
        check(ctx, logits, min(8, per * kept), softmax, bias=bias, groups=many, kept=kept, group_top=group_top)


@pytest.mark.parametrize("tokens", [1, 64, 65])
@pytest.mark.parametrize("experts,groups", [(16, 8), (60, 30), (128, 128), (256, 256), (250, 125), (1024, 1024), (1000, 40), (999, 3)])
def test_many_groups_in_one_launch_and_in_two(ctx, tokens, experts, groups):
    """The most that a workgroup keeps: a rank a group and, of one chunk, its pairs."""
    rng = np.random.default_rng(tokens + groups)
    logits = rng.standard_normal((tokens, experts)).astype(np.float32)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    per = experts // groups
    for kept in {1, groups // 2, groups - 1}:
        check(ctx, logits, min(16, per * kept), False, bias=bias, groups=groups, kept=kept, group_top=2)
        check(ctx, np.round(logits), min(16, per * kept), True, groups=groups, kept=kept)
