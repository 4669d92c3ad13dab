"""he_sgd_momentum without an average (plain SGD), on the first step and on later ones: w -= lr * g, no average read."""
import ctypes as C

import pytest

from helium_b200 import ir
from helium_b200._lib import check, lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("first_step", [1, 0])
def test_no_average(dt, first_step):
    import torch
    n = 1003
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(n, generator=gen, device="cuda")
    g = torch.randn(n, generator=gen, device="cuda").to(torch.bfloat16 if dt == ir.BF16 else torch.float32)
    w16 = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    want = w.double() - 0.1 * g.double()
    check(lib.he_sgd_momentum(C.c_void_p(w.data_ptr()), None, C.c_void_p(g.data_ptr()), dt, C.c_void_p(w16.data_ptr()), n, 0.1, 0.0, first_step,
                              C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    # lr is the f32 nearest 0.1; one product, one difference
    assert bool(((w.double() - want).abs() <= 3 * 2.0 ** -24 * (want.abs() + 0.1 * g.double().abs())).all())
    assert torch.equal(w16, w.bfloat16())
