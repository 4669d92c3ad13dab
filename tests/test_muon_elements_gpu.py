"""he_plan_muon, every element of the update for itself: a wrong value in a tile's corner or in the columns behind the last vector
is nothing beside the 2-norm of a large update.

The arithmetic's error is spread over the update like noise: its root mean square is at most the 2-norm's tolerance (test_muon_gpu.py)
times the update's, and the largest of n independent normal values lies below 8 deviations for any n here (16 million: 5.4).
Beside it every element has its own rounding to the output's type, half a step.  For rows and columns the same with the norm
of a row (column): of k such values it is within (1 + 8 / sqrt(k)) of the root mean square times sqrt(k)."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_muon_gpu import _matrix, _reference, _tolerance

pytestmark = pytest.mark.gpu

HALF_STEP = {ir.BF16: 2.0 ** -8, ir.F16: 2.0 ** -11}


def _check_elements(o, want, out_dt, tol):
    err, rms = (o.double() - want).abs(), float(want.square().mean().sqrt())
    assert bool((err <= HALF_STEP[out_dt] * want.abs() + 8 * tol * rms + 2.0 ** -25).all()), float((err / (HALF_STEP[out_dt] * want.abs() + 8 * tol * rms)).max())
    for dim in (0, 1):
        k = err.shape[dim]
        bound = HALF_STEP[out_dt] * want.norm(dim=dim) + (1 + 8 / k ** 0.5) * tol * rms * k ** 0.5
        assert bool((err.norm(dim=dim) <= bound).all()), (dim, float((err.norm(dim=dim) / bound).max()))


# single CTAs and pairs, sums of S split and not, matrices of one SM, odd rows and columns at the edges of tiles
@pytest.mark.parametrize("shape", [(128, 320), (97, 301), (301, 97), (129, 65), (130, 1030), (333, 1037), (1037, 333), (512, 4608), (520, 4099), (4099, 520),
                                   (1025, 1031), (2048, 2050), (2050, 2047), (2049, 4104), (4096, 4100)])
@pytest.mark.parametrize("out_dt", [ir.BF16, ir.F16])
def test_elements(ctx, shape, out_dt):
    g = _matrix(shape, seed=shape[0] + shape[1], kind="noise")
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, out_dtype=out_dt, momentum=None).launch([g])
    want, _ = _reference(g, None, None, False, 5)
    _check_elements(o, want, out_dt, _tolerance(out_dt, 5, g))
    ctx.poll()


def test_elements_of_a_list(ctx):
    """Sizes side by side in one list, on pairs: the border of one matrix is the beginning of the next in the workspace."""
    shapes = [(2048, 2200), (129, 1000), (1000, 129), (64, 4096), (300, 301), (2200, 700)]
    grads = [_matrix(s, 50 + i, "noise") for i, s in enumerate(shapes)]
    for o, g in zip(hb.Plan.muon(ctx, shapes, grad_dtype=ir.F32, momentum=None).launch(grads), grads):
        want, _ = _reference(g, None, None, False, 5)
        _check_elements(o, want, ir.BF16, _tolerance(ir.BF16, 5, g))
    ctx.poll()
