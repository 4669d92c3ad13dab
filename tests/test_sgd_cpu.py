"""he_sgd_momentum without a device: refused calls."""
import ctypes as C

import pytest

from helium_b200 import ir
from helium_b200._lib import lib


@pytest.mark.parametrize("dt", [ir.U32, ir.BOOL, 99, -1])
def test_gradient_types(dt):
    w = C.c_void_p(256)      # refused before anything is read
    assert lib.he_sgd_momentum(w, None, w, dt, None, 4, 0.1, 0.0, 1, None) == -2
    assert b"f32, bf16 or f16" in lib.he_last_error_string()


def test_null_and_empty():
    w = C.c_void_p(256)
    assert lib.he_sgd_momentum(None, None, w, ir.F16, None, 4, 0.1, 0.0, 1, None) == -1
    assert lib.he_sgd_momentum(w, None, None, ir.F16, None, 4, 0.1, 0.0, 1, None) == -1
    assert lib.he_sgd_momentum(w, None, w, ir.F16, None, 0, 0.1, 0.0, 1, None) == -1
