"""he_plan_group_norm without a device: what it plans and what it refuses."""
import ctypes as C

import pytest

import helium_b200 as hb
from helium_b200 import ir
from helium_b200._abi import HeGroupNormParams
from helium_b200._lib import lib


def test_planning_without_a_device():
    p = hb.Plan.group_norm(None, "fwd", 8, 784, 128, 32, activation="silu")
    assert p.out_shapes == [(8, 784, 128), (8, 32), (8, 32)] and p.out_dtypes == [ir.BF16, ir.F32, ir.F32] and p.n_inputs == 3
    assert "group norm forward: " in p.description and "[8,784,128] in 32 groups" in p.description and "silu" in p.description
    p = hb.Plan.group_norm(None, "bwd", 8, 784, 128, 32, dtype=ir.F32)
    assert p.out_shapes == [(8, 784, 128), (128,), (128,)] and p.n_inputs == 6 and p.workspace_bytes >= 8 * 2 * 128 * 4


@pytest.mark.parametrize("change,match", [
    (dict(batch=0), "empty"), (dict(positions=0), "empty"), (dict(channels=0), "empty"), (dict(batch=-1), "empty"),
    (dict(groups=0), "groups"), (dict(groups=5), "groups"), (dict(groups=-2), "groups"), (dict(dtype=ir.U32), "f16, bf16 or f32"),
    (dict(dtype=ir.BOOL), "f16, bf16 or f32"), (dict(dtype=99), "f16, bf16 or f32"), (dict(activation=4), "activation"),
    (dict(activation=-1), "activation"), (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(batch=70000), "65535"), (dict(positions=1 << 31), "positions"), (dict(channels=1 << 17, groups=1), "channels"),
])
def test_refusals(change, match):
    args = dict(batch=2, channels=16, positions=9, groups=4, dtype=ir.BF16, activation=2, eps=1e-5)
    args.update(change)
    prm = HeGroupNormParams(**args)
    h = C.c_void_p(1)
    rc = lib.he_plan_group_norm(None, 0, C.byref(prm), C.byref(h))
    assert rc in (-1, -2) and match.encode() in lib.he_last_error_string() and not h.value


def test_refused_calls():
    prm = HeGroupNormParams(batch=2, channels=16, positions=9, groups=4, dtype=ir.BF16, activation=2, eps=1e-5)
    h = C.c_void_p()
    assert lib.he_plan_group_norm(None, 2, C.byref(prm), C.byref(h)) == -1
    assert lib.he_plan_group_norm(None, 0, None, C.byref(h)) == -1
    assert lib.he_plan_group_norm(None, 0, C.byref(prm), None) == -1
    assert lib.he_plan_group_norm(None, 0, C.byref(prm), C.byref(h)) == 0
    assert lib.he_launch(h, None, None, None, None) == -1      # planned without a context: no CPU path
    lib.he_plan_destroy(h)
    with pytest.raises(KeyError):
        hb.Plan.group_norm(None, "sideways", 1, 1, 8, 1)
    with pytest.raises(KeyError):
        hb.Plan.group_norm(None, "fwd", 1, 1, 8, 1, activation="swish")
