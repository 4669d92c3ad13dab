"""he_plan_muon on f32 gradients at the ends of f32's range, and on zero gradients with the smallest eps."""
import ctypes

import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_muon_gpu import _check, _matrix, _reference, _tolerance

pytestmark = pytest.mark.gpu

SHAPES = [(64, 288), (130, 190), (190, 130), (512, 640)]


@pytest.mark.parametrize("momentum", [None, 0.5])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e-40, 1e-38, 1e-36, 1e-34, 1e40])
def test_gradients_at_the_ends_of_the_range(ctx, shape, size, momentum):
    """Times 1e-3: from multiples of a few denormal steps on (the inputs are what those steps make of them) to 1e37.  With momentum
    the direction, 0.75 of the gradient, is rounded to denormal steps of 1.4e-45 twice, 0.6e-45 each (root mean square); next to
    the gradient's size that is an error of every singular direction, and the weakest of them, which the steps bring up to 1 like
    the others, lie ten times below it here.  Five times that is allowed."""
    if momentum and size < 1e-38:
        pytest.skip("the direction itself has two digits there")
    import torch
    g = (_matrix(shape, 5).double() * size).float()
    ins = [g] + ([torch.zeros(shape, device="cuda")] if momentum else [])
    o = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=momentum, nesterov=True, eps=0.0).launch(ins)[0]
    want, _ = _reference(g, torch.zeros(shape, device="cuda"), momentum, True, 5, eps=0.0)
    tol = _tolerance(ir.BF16, 5, g, eps=0.0)
    if momentum:
        tol = tol + 50 * 0.85e-45 / float(g.double().square().mean().sqrt())
    _check(o, want, tol, f"{shape} {size}")
    ctx.poll()


@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1e-36, 1e-30])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_zero_gradient_is_zero_for_any_eps(ctx, shape, eps):
    import torch
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=None, eps=eps).launch([torch.zeros(shape, device="cuda")])
    assert torch.equal(o, torch.zeros_like(o))
    ctx.poll()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ratio", [1.0, 1e-2, 1e-3, 1e-4])
def test_a_gradient_below_eps(ctx, shape, ratio):
    """|d| / eps = ratio: X starts that much smaller, in f16 steps of 2^-24 whose root mean square is 1.7e-8.  The weakest singular
    directions, ten times below the gradient's size, grow like the others: ten times 1.7e-8 / ratio, and a margin of two."""
    g = _matrix(shape, 5)
    eps = float(g.double().norm()) / ratio
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=None, eps=eps).launch([g])
    eps = ctypes.c_float(eps).value
    want, _ = _reference(g, None, None, False, 5, eps=eps)
    tol = _tolerance(ir.BF16, 5, g, eps=eps) + 20 * 1.7e-8 * (1 + ratio) / ratio
    _check(o, want, tol, f"{shape} {ratio}")
    ctx.poll()
