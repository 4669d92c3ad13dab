"""he_sgd_momentum on f16 gradients, and on the f16 updates that he_plan_muon writes."""
import ctypes as C

import pytest

import helium_b200 as hb
from helium_b200 import ir
from helium_b200._lib import check, lib

pytestmark = pytest.mark.gpu

u = 2.0 ** -24


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _step(w, avg, g, dt, w16, lr, momentum, first):
    import torch
    check(lib.he_sgd_momentum(_p(w), _p(avg), _p(g), dt, _p(w16), w.numel(), lr, momentum, first, C.c_void_p(torch.cuda.current_stream().cuda_stream)))


@pytest.mark.parametrize("first", [1, 0])
@pytest.mark.parametrize("n", [1, 255, 1003, 700001])
def test_momentum(n, first):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    w, avg, g = rand(), rand(), rand().half()
    g[0] = 2.0 ** -24                                     # f16's smallest
    w16 = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    a = g.double() if first else 0.25 * g.double() + 0.75 * avg.double()
    want, size = w.double() - 0.5 * a, avg.double().abs() + g.double().abs()
    _step(w, avg, g, ir.F16, w16, 0.5, 0.75, first)
    assert bool(((avg.double() - a).abs() <= 3 * u * size).all())     # two products and their sum
    assert bool(((w.double() - want).abs() <= 3 * u * size + u * want.abs()).all())
    assert torch.equal(w16, w.bfloat16())


def test_an_f16_update_of_muon(ctx):
    import torch
    shape = (130, 290)
    gen = torch.Generator(device="cuda").manual_seed(4)
    w, g = torch.randn(shape, generator=gen, device="cuda"), torch.randn(shape, generator=gen, device="cuda").half()
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F16, out_dtype=ir.F16, momentum=None).launch([g])
    want = w.double() - 0.125 * o.double()
    _step(w, None, o, ir.F16, None, 0.125, 0.0, 0)
    assert bool(((w.double() - want).abs() <= u * (want.abs() + 0.125 * o.double().abs())).all())
