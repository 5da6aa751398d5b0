"""Groups of experts by the sum of two choices that f32 does not hold: biases of the
type's lowest value (a usual way to switch an expert off) or its largest.  As in
test_gpu_route, experts, offsets and order are compared for equality."""

import numpy as np
import pytest

from test_gpu_route import check

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min

# experts, groups, kept, top: groups of whole rounds of the lanes, of parts of one, more than the lanes; 64 lanes a token.
GROUPS = [(64, 4, 1, 3), (64, 4, 3, 8), (256, 8, 4, 8), (60, 12, 5, 4), (128, 64, 9, 8), (512, 4, 2, 8), (1000, 40, 7, 16)]


@pytest.mark.parametrize("experts,groups,kept,top", GROUPS)
@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("far", [LOWEST, -LOWEST])
def test_two_biases_whose_sum_is_past_f32(ctx, softmax, experts, groups, kept, top, far):
    """A group of nothing but experts with the lowest (or the largest) bias is one that has experts: before those that have
    none, in the order of its sum."""
    rng = np.random.default_rng(experts + top)
    per = experts // groups
    logits = rng.standard_normal((80, experts)).astype(np.float32)
    logits[:40, :per] = -np.inf  # (nothing in group 0)
    logits[20:30, per:2 * per] = np.nan
    bias = np.full(experts, far, np.float32)
    check(ctx, logits, top, softmax, bias=bias, groups=groups, kept=kept, group_top=2)
    uneven = (far * (1 - rng.integers(0, 5, experts) / 16)).astype(np.float32)
    check(ctx, logits, top, softmax, bias=uneven, groups=groups, kept=kept, group_top=2)
    bias[-per:] = 0.1 * rng.standard_normal(per)  # one ordinary group, the last
    check(ctx, logits, top, softmax, bias=bias, groups=groups, kept=kept, group_top=2)
    bias[rng.random(experts) < 0.5] = 0.25
    for group_top in (1, 2):
        check(ctx, logits, top, softmax, bias=bias, groups=groups, kept=kept, group_top=group_top)
