"""he_plan_group_norm on whole numbers, whose sums f32 holds exactly: one row lost, doubled or taken from a neighbour shows.

Backward (no activation): x, dy, mean are small whole numbers, rstd and gamma powers of two; every product is a multiple of 1/2 and
every partial sum stays below 2^22 in those steps (signs are random: sqrt(2e6) * 60 at most, with a wide margin), so dgamma and
dbeta come out exactly whatever the order.  dx = rstd (gamma g - m1 - xh m2) has then the two means' roundings (of 1 / count and the
product) and three of its own: 8 u of its terms, and the output's.
Forward: the sum of x in 1 .. 8 is exact (below 2^24; the shifts of the two-pass kernels are means of 8, 64, 512 such numbers),
the mean is it times a rounded 1 / count: 2 u.  One value more or less in the 2.1 million of the largest group is 8 u.
Outputs start as NaN."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_group_norm_gpu import FLOOR, HALF_STEP, SIZES, _dtype, _per_channel, u

pytestmark = pytest.mark.gpu

# besides those: several slices or clusters with rows of the neighbouring pictures at both ends, and without
MORE = [(5, 1961, 77, 7), (6, 1960, 77, 7), (3, 437, 320, 32), (4, 701, 60, 6), (3, 2001, 3, 1), (40, 40001, 3, 1), (2, 250007, 5, 5), (9, 17, 1001, 7),
        (300, 20001, 12, 3), (128, 784, 128, 32)]


def _whole(shape, dt, gen, lo, hi, zero=True):
    import torch
    v = torch.empty(shape, device="cuda", dtype=torch.float32)
    v.random_(lo, hi + 1, generator=gen)
    if not zero:
        v[v == 0] = 1
    return v.to(_dtype(dt))


def _nan_outputs(plan):
    import torch
    return [torch.full(s, float("nan"), dtype=_dtype(d), device="cuda") for s, d in zip(plan.out_shapes, plan.out_dtypes)]


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES + MORE)
def test_backward(ctx, size, dt):
    import torch
    n, p, c, groups = size
    gen = torch.Generator(device="cuda").manual_seed(p + c)
    x, dy = _whole((n, p, c), dt, gen, -4, 4), _whole((n, p, c), dt, gen, -3, 3, zero=False)
    mean = _whole((n, groups), ir.F32, gen, -1, 1)
    rstd, gamma = [2.0 ** _whole(s, ir.F32, gen, -1, 1) for s in ((n, groups), (c,))]
    beta = torch.zeros(c, device="cuda")
    plan = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt)
    dx, dgamma, dbeta = plan.launch([dy, x, gamma, beta, mean, rstd], _nan_outputs(plan))
    r = _per_channel(rstd.double(), c)
    xh, g = (x.double() - _per_channel(mean.double(), c)) * r, dy.double()
    assert torch.equal(dbeta.double(), g.sum((0, 1))), plan.description
    assert torch.equal(dgamma.double(), (g * xh).sum((0, 1))), plan.description
    mean_of = lambda v: _per_channel(v.reshape(n, p, groups, -1).mean((1, 3)), c)  # noqa: E731
    g = g * gamma.double()
    m1, m2 = mean_of(g), mean_of(g * xh)
    want = r * (g - m1 - xh * m2)
    tol = HALF_STEP[dt] * want.abs() + FLOOR[dt] + 8 * u * r * (g.abs() + m1.abs() + (xh * m2).abs())
    assert bool(((dx.double() - want).abs() <= tol).all()), plan.description


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES + MORE)
def test_forward(ctx, size, dt):
    import torch
    n, p, c, groups = size
    gen = torch.Generator(device="cuda").manual_seed(p + c)
    x = _whole((n, p, c), dt, gen, 1, 8)
    ones, zeros = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, eps=1e-3)
    y, mean, rstd = plan.launch([x, ones, zeros], _nan_outputs(plan))
    xg = x.double().reshape(n, p, groups, -1)
    wm = xg.mean((1, 3))
    wr = 1 / ((xg - wm[:, None, :, None]).square().mean((1, 3)) + 1e-3).sqrt()
    assert bool(((mean.double() - wm).abs() <= 2 * u * wm).all()), plan.description
    # sums of at most 64 + 64 + 70 rounded additions of positive terms, of which up to 16 times the result cancels in the slabs
    # (nine in the two-pass kernels): statistically sqrt(200) / 3 * 17 u, halved by the root; eps keeps a constant group's finite
    assert bool(((rstd.double() - wr).abs() <= 64 * u * wr).all()), plan.description
    # y from the statistics that came out
    want = (x.double() - _per_channel(mean.double(), c)) * _per_channel(rstd.double(), c)
    size_of = (x.double() + _per_channel(mean.double(), c)) * _per_channel(rstd.double(), c)
    assert bool(((y.double() - want).abs() <= HALF_STEP[dt] * want.abs() + FLOOR[dt] + 4 * u * size_of).all()), plan.description


def test_backward_offsets_past_32_bits(ctx):
    """More than 2^32 bytes and 2^31 elements a tensor."""
    import torch
    n, p, c, groups = 3, 11_500_003, 64, 8
    gen = torch.Generator(device="cuda").manual_seed(13)
    x, dy = [torch.empty(n, p, c, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for i in range(n):
        x[i].random_(-4, 5, generator=gen)
        dy[i].random_(-3, 4, generator=gen)
    mean = _whole((n, groups), ir.F32, gen, -1, 1)
    rstd, gamma = [2.0 ** _whole(s, ir.F32, gen, -1, 1) for s in ((n, groups), (c,))]
    plan = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups)
    dx, dgamma, dbeta = plan.launch([dy, x, gamma, torch.zeros(c, device="cuda"), mean, rstd])
    wb, wg, means = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda"), []
    for i in range(n):
        b, w = torch.zeros_like(wb), torch.zeros_like(wb)
        for k in range(0, p, 2_000_000):
            g = dy[i, k:k + 2_000_000].double()
            b += g.sum(0)
            w += (g * ((x[i, k:k + 2_000_000].double() - mean[i].double().repeat_interleave(8)) * rstd[i].double().repeat_interleave(8))).sum(0)
        wb += b
        wg += w
        means.append([(gamma.double() * v).view(groups, 8).sum(1) / (p * 8) for v in (b, w)])
    # partial sums of a channel stay below 60 sqrt(3.5e7) = 3.5e5 in steps of 1/2
    assert torch.equal(dbeta.double(), wb) and torch.equal(dgamma.double(), wg)
    for i in range(n):
        for rows in (slice(0, 1000), slice(p // 2, p // 2 + 1000), slice(p - 1000, p)):
            r, m1, m2 = [v.double().repeat_interleave(8) for v in (rstd[i], *means[i])]
            xh, g = (x[i, rows].double() - mean[i].double().repeat_interleave(8)) * r, dy[i, rows].double() * gamma.double()
            want = r * (g - m1 - xh * m2)
            tol = 2.0 ** -8 * want.abs() + 1e-38 + 8 * u * r * (g.abs() + m1.abs() + (xh * m2).abs())
            assert bool(((dx[i, rows].double() - want).abs() <= tol).all()), (i, rows)
