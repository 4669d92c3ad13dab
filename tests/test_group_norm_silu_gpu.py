"""SiLU behind he_plan_group_norm where its argument is far from zero: a channel switched off by its beta.  u = 2^-24, U the half
step of the type.

z = (x - mean) rstd gamma + beta is 128 u off, of its terms' sizes T added without signs (rstd's own sums are 64 u, the rest a
few roundings); y moves by that times the slope.  exp(-z) is as many u off as z is large, and a few roundings follow: y is
within U |y| + 32 u (1 + |z|) |y| + 128 u T |slope|.  Below 2^-126 a sigmoid may be flushed to zero: 1e-35."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_group_norm_gpu import HALF_STEP, _dtype, _per_channel, u

pytestmark = pytest.mark.gpu

BETAS = [-3e38, -1e20, -1e6, -1000.0, -150.0, -80.0, -60.0, -46.0, -44.0, -43.0, -30.0, -5.0, 0.0, 30.0, 44.0, 80.0, 150.0, 1e20]


def _data(n, p, groups, dt):
    import torch
    c = groups * len(BETAS)
    g = torch.Generator(device="cuda").manual_seed(41)
    x = torch.randn(n, p, c, generator=g, device="cuda").to(_dtype(dt))
    dy = torch.randn(n, p, c, generator=g, device="cuda").to(_dtype(dt))
    beta = torch.tensor(BETAS * groups, device="cuda")      # neighbours of every size share a pair
    gamma = torch.where(beta.abs() > 20, 0.25, 1.0)
    xd = x.double().view(n, p, groups, -1)
    mean = xd.mean((1, 3))
    rstd = 1 / ((xd - mean[:, None, :, None]).square().mean((1, 3)) + 1e-5).sqrt()
    return x, dy, gamma, beta, mean, rstd


def _slope(z):
    import torch
    s = torch.sigmoid(z)
    return torch.where(z.abs() > 800, (z > 0).double(), s * (1 + z * (1 - s)))


# slabs and two passes, whole rows and odd channels (18 channels a group: no 16-byte vectors of 16-bit types in 3 groups)
SIZES = [(3, 50, 4), (3, 51, 3), (2, 120001, 4), (2, 120001, 3)]


@pytest.mark.parametrize("dt", [ir.F32, ir.BF16, ir.F16])
@pytest.mark.parametrize("size", SIZES)
def test_forward(ctx, size, dt):
    import torch
    n, p, groups = size
    x, _, gamma, beta, mean, rstd = _data(n, p, groups, dt)
    c = beta.numel()
    y = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation="silu").launch([x, gamma, beta])[0]
    z = (x.double() - _per_channel(mean, c)) * _per_channel(rstd, c) * gamma.double() + beta.double()
    want = z * torch.sigmoid(z)
    terms = (x.double().abs() + _per_channel(mean.abs(), c)) * _per_channel(rstd, c) * gamma.double() + beta.double().abs()
    if dt == ir.F16:                                         # 1e20 is beyond the type
        keep = want.abs() < 6e4
        assert bool((y.double()[~keep] == float("inf")).all())
        y, want, z, terms = y[keep], want[keep], z[keep], terms[keep]
    tol = HALF_STEP[dt] * want.abs() + (2.0 ** -25 if dt == ir.F16 else 1e-35) + torch.where(
        z > 100, 160 * u * terms, 32 * u * (1 + z.abs()) * want.abs() + 128 * u * terms * _slope(z).abs())
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() / tol).max())
    assert bool((y[z < -150] == 0).all())


@pytest.mark.parametrize("dt", [ir.F32, ir.BF16, ir.F16])
@pytest.mark.parametrize("size", SIZES)
def test_backward(ctx, size, dt):
    """dbeta is the sum of dy act'(z), with |act'(z)| < (1 + |z|) exp(-|z|) below zero and within that of 1 above."""
    import torch
    n, p, groups = size
    x, dy, gamma, beta, mean, rstd = _data(n, p, groups, dt)
    c = beta.numel()
    ins = [dy, x, gamma, beta, mean.float(), rstd.float()]
    dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt, activation="silu").launch(ins)
    xh = (x.double() - _per_channel(mean.float().double(), c)) * _per_channel(rstd.float().double(), c)
    z = xh * gamma.double() + beta.double()
    g = dy.double() * _slope(z)
    # the slope's error, 128 u T with T up to 4 + |z| on average, and the sum's, 512 u of its terms as in the other tests
    size_of = dy.double().abs() * torch.where(z < 0, (1 + z.abs()) * torch.exp(-z.abs()), 1 + z.abs() * torch.exp(-z.abs()))
    tol = 512 * u * ((4 + z.abs().clamp(max=1000.0)) * size_of).sum((0, 1)) + 1e-30
    assert bool(((dbeta.double() - g.sum((0, 1))).abs() <= tol).all())
    tol = 512 * u * ((4 + z.abs().clamp(max=1000.0)) * size_of * (1 + xh.abs())).sum((0, 1)) + 1e-30
    assert bool(((dgamma.double() - (g * xh).sum((0, 1))).abs() <= tol).all())
    t = g * gamma.double()
    mean_of = lambda v: _per_channel(v.reshape(n, p, groups, -1).mean((1, 3)), c)  # noqa: E731
    want = _per_channel(rstd, c) * (t - mean_of(t) - xh * mean_of(t * xh))
    assert not bool(torch.isnan(dx).any())
    assert float((dx.double() - want).norm() / want.norm()) <= 0.5 * HALF_STEP[dt] + 64 * u
