"""he_plan_muon without a device: what it plans and what it refuses."""
import ctypes as C

import pytest

import helium_b200 as hb
from helium_b200 import ir
from helium_b200._abi import HeMuonParams
from helium_b200._lib import lib


def _params(**change):
    args = dict(count=2, rows=[64, 300], cols=[288, 7], grad_dtype=ir.BF16, out_dtype=ir.BF16, steps=5, coef=(3.4445, -4.775, 2.0315), eps=1e-7,
                use_momentum=1, momentum=0.95, nesterov=1, scales=None)
    args.update(change)
    n = len(args["rows"])
    for k, t in (("rows", C.c_int64), ("cols", C.c_int64), ("scales", C.c_float)):
        if args[k] is not None:
            args[k] = (t * n)(*args[k])
    args["coef"] = (C.c_float * 3)(*args["coef"])
    return HeMuonParams(**{k: v for k, v in args.items() if v is not None})


def test_planning_without_a_device():
    p = hb.Plan.muon(None, [(64, 288), (1000, 512)], momentum=0.9)
    assert p.out_shapes == [(64, 288), (1000, 512)] * 2 and p.out_dtypes == [ir.BF16] * 2 + [ir.F32] * 2 and p.n_inputs == 4
    assert "2 matrices" in p.description and "5 Newton-Schulz steps" in p.description
    p = hb.Plan.muon(None, [(4096, 4096)], momentum=None, out_dtype=ir.F16)
    # X twice and its low half, S and B: five 4096 x 4096 tensors of two bytes
    assert p.n_inputs == 1 and 5 * 2 * 4096 ** 2 <= p.workspace_bytes <= 5 * 2 * 4096 ** 2 + (1 << 20)


@pytest.mark.parametrize("change,match", [
    (dict(count=0), "no matrices"), (dict(count=-1), "no matrices"), (dict(count=5000), "4096"),
    (dict(rows=[0, 300]), "empty"), (dict(cols=[288, -7]), "empty"), (dict(rows=[40000, 1], cols=[40000, 1]), "32768"),
    (dict(cols=[1 << 21, 7]), "32768"), (dict(grad_dtype=ir.U32), "gradients"), (dict(out_dtype=ir.F32), "updates"), (dict(steps=0), "steps"),
    (dict(steps=65), "steps"), (dict(coef=(1.0, float("nan"), 0.0)), "coefficients"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(momentum=1.0), "momentum"), (dict(momentum=-0.1), "momentum"), (dict(momentum=float("nan")), "momentum"),
    (dict(scales=[1.0, float("inf")]), "scale"),
])
def test_refusals(change, match):
    h = C.c_void_p(1)
    rc = lib.he_plan_muon(None, C.byref(_params(**change)), C.byref(h))
    assert rc in (-1, -2) and match.encode() in lib.he_last_error_string() and not h.value


def test_refused_calls():
    h = C.c_void_p()
    prm = _params()
    assert lib.he_plan_muon(None, None, C.byref(h)) == -1
    assert lib.he_plan_muon(None, C.byref(prm), None) == -1
    prm.rows = None
    assert lib.he_plan_muon(None, C.byref(prm), C.byref(h)) == -1
    with pytest.raises(ValueError, match="scales"):
        hb.Plan.muon(None, [(4, 4)], scales=[1.0, 2.0])
    p = hb.Plan.muon(None, [(4, 4)], momentum=None)
    assert lib.he_launch(p._h, None, None, None, None) == -1      # planned without a context: no CPU path


@pytest.mark.parametrize("coefs,steps,fits", [
    ((3.4445, -4.775, 2.0315), 64, True), ((1.5, -0.5, 0.0), 64, True), ((1.875, -1.25, 0.375), 64, True), ((2.0, -1.5, 0.5), 64, True),
    ((1.0, 0.0, 0.0), 64, True),
    ((4.0, 0.0, 0.0), 1, True),          # the step itself starts inside the range, what it makes is only written out
    ((4.0, 0.0, 0.0), 2, False),         # X past its f16 range
    ((0.0, 70.0, -70.0), 1, False),      # B past its f16 range at once
    ((3.4445, -4.775, 3.0), 5, False),   # runs away
    ((3e38, -3e38, 3e38), 5, False),
])
def test_coefficients_that_leave_the_products_range_are_refused(coefs, steps, fits):
    h = C.c_void_p()
    rc = lib.he_plan_muon(None, C.byref(_params(coef=coefs, steps=steps)), C.byref(h))
    assert (rc == 0) == fits, lib.he_last_error_string()
    if fits:
        lib.he_plan_destroy(h)
    else:
        assert rc == -2 and b"range" in lib.he_last_error_string() and not h.value
