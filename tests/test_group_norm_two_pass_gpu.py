"""The forward pass of he_plan_group_norm in two passes: values that its shifted sums could trip over.  u = 2^-24."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_group_norm_gpu import _act, _check_forward, _inputs, _per_channel, u

pytestmark = pytest.mark.gpu


def _plan(ctx, n, p, c, groups, dt, act="none", eps=1e-5):
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation=act, eps=eps)
    assert "two passes" in plan.description, plan.description
    return plan


@pytest.mark.parametrize("dt,p", [(ir.F32, 20001), (ir.BF16, 40001)])
def test_a_threads_first_value_far_from_all_others(ctx, dt, p):
    """Some 230 values a thread, the first of one thread's columns 100, 300 or 10^4 deviations away.

    A thread's squares are taken about its first value M, then about the mean of its first n for n = 8, 64, 512: the 7 n values
    between two of these are about (M / n)^2 each, a sum of 7 M^2 / n that grows evenly and takes 7 n roundings of half of it
    on average: 25 u M^2 at most, and as much before the first; M^2 is itself part of the result: 75 u for the three stretches.  The
    ordinary values' sum of n squares is sqrt(n) / 3 u off (independent roundings), times the nine that may cancel 45 u.
    rstd is off by half of the 120 u, and a few roundings: 64 u."""
    import torch
    n, c, groups = 300, 24, 1
    g = torch.Generator(device="cuda").manual_seed(31)
    x = torch.randn(n, p, c, generator=g, device="cuda", dtype=torch.float32).to({ir.F32: torch.float32, ir.BF16: torch.bfloat16}[dt])
    for i in range(n):
        x[i, 0, i % c] = (100.0, 300.0, 1e4)[i % 3]
    plan = _plan(ctx, n, p, c, groups, dt)
    _, mean, rstd = plan.launch([x, torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")])
    worst = 0.0
    for i in range(n):
        v = x[i].double()
        m = v.mean()
        r = 1 / ((v - m).square().mean() + 1e-5).sqrt()
        worst = max(worst, abs(float(rstd[i, 0].double() / r) - 1))
        # p c / (p c) values of size 1 and the one of size M: 256 u of their mean size, as in the other tests of the mean
        assert abs(float(mean[i, 0].double() - m)) <= 256 * u * float(v.abs().mean())
    assert worst <= 64 * u, worst / u


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("size", [(1, 70001, 40, 8), (1, 120001, 77, 7), (300, 20001, 24, 3)])
def test_mean_far_from_zero(ctx, size, dt):
    n, p, c, groups = size
    x, gamma, beta, _ = _inputs(n, p, c, dt, seed=9, offset=1000.0 if dt == ir.F32 else 30.0)
    plan = _plan(ctx, n, p, c, groups, dt)
    y, mean, rstd = plan.launch([x, gamma, beta])
    k = slice(0, min(n, 8))
    _check_forward(plan, x[k], gamma, beta, groups, "none", dt, y[k], mean[k], rstd[k])


@pytest.mark.parametrize("size", [(1, 70001, 40, 8), (1, 120001, 77, 7)])
def test_a_constant_group(ctx, size):
    """Multiples of 1/4 add up exactly (below 2^22); the mean is that times a rounded 1 / count: 2 u.  The spread comes out as at
    most the square of that, nothing beside eps, and (x - mean) rstd gamma as 2 u 3.25 rstd gamma beside beta."""
    import torch
    n, p, c, groups = size
    x, gamma, beta, _ = _inputs(n, p, c, ir.F32, seed=10)
    per = c // groups
    x[0, :, per:2 * per] = 3.25
    plan = _plan(ctx, n, p, c, groups, ir.F32, "silu")
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "silu", ir.F32, y, mean, rstd)
    assert abs(float(mean[0, 1]) - 3.25) <= 2 * u * 3.25
    assert abs(float(rstd[0, 1].double()) * 1e-5 ** 0.5 - 1) <= 8 * u
    want = _act(beta[per:2 * per].double(), "silu")
    tol = 1.1 * 2 * u * 3.25 * 1e-5 ** -0.5 * gamma[per:2 * per].double().abs() + 64 * u * (1 + want.abs())
    assert bool(((y[0, :, per:2 * per].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("size", [(2, 120001, 40, 8), (2, 120001, 77, 7), (2, 700001, 3, 1)])
def test_a_nan_stays_in_its_group(ctx, size, dt):
    import torch
    n, p, c, groups = size
    for bad, where in ((float("nan"), 0), (float("inf"), p - 1), (-float("inf"), p // 2)):
        x, gamma, beta, dy = _inputs(n, p, c, dt, seed=11)
        x[1, where, 0] = bad
        y, mean, rstd = _plan(ctx, n, p, c, groups, dt, "relu").launch([x, gamma, beta])
        hit = torch.zeros(n, p, c, dtype=torch.bool, device="cuda")
        hit[1, :, :c // groups] = True
        assert bool(torch.isnan(y[hit]).all()) and not bool(torch.isnan(y[~hit]).any())
        assert int(torch.isnan(mean).sum() + torch.isinf(mean).sum()) == 1 and int(torch.isnan(rstd).sum()) == 1
        bwd = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt, activation="silu")
        assert "two passes" in bwd.description
        dx, dgamma, dbeta = bwd.launch([dy, x, gamma, beta, mean, rstd])
        assert bool(torch.isnan(dx[hit]).all()) and not bool(torch.isnan(dx[~hit]).any())
        assert not bool(torch.isnan(dgamma[c // groups:]).any()) and not bool(torch.isnan(dbeta[c // groups:]).any())


def test_eps_zero(ctx):
    """A spread of its own: no eps is needed, and a variance that comes out below zero by rounding may not become a NaN."""
    import torch
    n, p, c, groups = 1, 70001, 40, 8
    x, gamma, beta, _ = _inputs(n, p, c, ir.F32, seed=12, offset=1000.0)
    y, mean, rstd = _plan(ctx, n, p, c, groups, ir.F32, eps=0.0).launch([x, gamma, beta])
    v = x.double().reshape(n, p, groups, -1)
    m = v.mean((1, 3))
    r = 1 / (v - m[:, None, :, None]).square().mean((1, 3)).sqrt()
    assert bool(((rstd.double() / r - 1).abs() <= 512 * u * (1 + (256 * u * 1000) ** 2 / u)).all())
    want = (x.double() - _per_channel(m, c)) * _per_channel(r, c) * gamma.double() + beta.double()
    assert not bool(torch.isnan(y).any())
    assert bool(((y.double() - want).abs() <= 512 * u * (1 + want.abs()) * (gamma.double().abs() * 2010 * _per_channel(r, c) + beta.double().abs())).all())
