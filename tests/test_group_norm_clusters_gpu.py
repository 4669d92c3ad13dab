"""he_plan_group_norm in clusters of several CTAs whose rows are no whole vectors, against 64 bits; tolerances as in
test_group_norm_gpu.py."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_group_norm_gpu import _check_forward, _inputs, test_backward as _check_backward, test_forward as _check_all_activations

pytestmark = pytest.mark.gpu

# super-rows of 8 (f32: 4) rows that end inside a picture, and that do not; groups that share vectors
SIZES = [(5, 1961, 77, 7), (6, 1960, 77, 7), (4, 1501, 60, 6), (3, 4001, 35, 5), (40, 40001, 3, 1)]


def _clusters(ctx, direction, size, dt):
    text = hb.Plan.group_norm(ctx, direction, *size, dtype=dt).description
    return "one pass" in text and "clusters of 1 " not in text


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES)
def test_forward(ctx, size, dt):
    assert _clusters(ctx, "fwd", size, dt)
    _check_all_activations(ctx, size, dt)


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES + [(3, 437, 320, 32)])
def test_backward(ctx, size, dt):
    assert _clusters(ctx, "bwd", size, dt)
    _check_backward(ctx, size, dt)


@pytest.mark.parametrize("dt,offset", [(ir.F32, 1000.0), (ir.F32, -30.0), (ir.BF16, 30.0), (ir.F16, -100.0)])
@pytest.mark.parametrize("size", SIZES + [(64, 49, 512, 32), (2, 500, 24, 8), (3, 437, 320, 32)])
def test_mean_far_from_zero(ctx, size, dt, offset):
    """The second round over the tile, for groups of whole and of shared vectors, in clusters and in single CTAs."""
    n, p, c, groups = size
    x, gamma, beta, _ = _inputs(n, p, c, dt, seed=9, offset=offset)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt)
    assert "one pass" in plan.description
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "none", dt, y, mean, rstd)
