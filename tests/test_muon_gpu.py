"""The Muon update (he_plan_muon) against the same steps in 64 bits.

Tolerance of an update, relative, 2-norm.  Rounding to the output type: at most half a step, 2^-8 (bf16) or 2^-11 (f16), of
each value; spread evenly over the half step and over the binade its root mean square is 0.42 of that.  Arithmetic: a step
rounds three operands to f16 (X, S and B off its diagonal), each 0.42 * 2^-11 = 2.1e-4 relative in the same sense, in terms
no larger than |b S X|: it adds sqrt(3) * 2.1e-4 * |b| |S X|.  Later steps multiply an error between the singular directions
i and j by the divided differences of p(v) = a v + b v^3 + c v^5 (its part symmetric in i, j by (p(vi) - p(vj)) / (vi - vj), the
other by (p(vi) + p(vj)) / (vi + vj), directions outside the matrix having v = 0).  `_tolerance` takes the singular values, follows
them through the steps and adds the steps' contributions as independent errors spread over all pairs, with a margin of
3 / sqrt(m) for matrices of few directions.  (A first form of this took the mean slope as 1, which three singular values
need not keep to: a 7 x 3 matrix was 6 % over it.)
The averages are f32, two roundings of products and one of the sum."""
import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_guard_bands_gpu import Guarded

pytestmark = pytest.mark.gpu

COEFS = (3.4445, -4.7750, 2.0315)
u = 2.0 ** -24


def _dtype(dt):
    import torch
    return {ir.BF16: torch.bfloat16, ir.F16: torch.float16, ir.F32: torch.float32}[dt]


def _tolerance(out_dt, steps, d, coefs=COEFS, eps=1e-7):
    import torch
    half = {ir.BF16: 2.0 ** -8, ir.F16: 2.0 ** -11}[out_dt]
    a, b, c = coefs
    p = lambda v: a * v + b * v ** 3 + c * v ** 5  # noqa: E731
    d = d.double()
    v = torch.linalg.svdvals(d / (d.norm() + eps))
    m = v.numel()
    if d.shape[0] != d.shape[1]:
        v = torch.cat([v, torch.zeros(1, dtype=v.dtype, device=v.device)])
    noise, slopes = [], []
    for _ in range(steps):
        noise.append(3 ** 0.5 * 2.1e-4 * abs(b) * (v ** 3).norm())
        w = p(v)
        diff, total = v[:m, None] - v[None, :], v[:m, None] + v[None, :]
        near = diff.abs() <= 1e-9 * (total + 1e-300)
        deriv = (a + 3 * b * v ** 2 + 5 * c * v ** 4)[:m, None].expand_as(diff)
        minus = torch.where(near, deriv, (w[:m, None] - w[None, :]) / torch.where(near, torch.ones_like(diff), diff))
        plus = torch.where(total > 0, (w[:m, None] + w[None, :]) / torch.where(total > 0, total, torch.ones_like(total)), torch.full_like(total, a))
        slopes.append((minus, plus))
        v = w
    tol2, size = (0.42 * half) ** 2, float(v.norm())
    minus, plus = torch.ones_like(slopes[0][0]), torch.ones_like(slopes[0][0])
    for k in reversed(range(steps)):
        grow = ((minus ** 2 + plus ** 2) / 2).mean().sqrt()      # of an error made in step k, by the steps behind it
        tol2 += float(noise[k] * grow / size) ** 2
        minus, plus = minus * slopes[k][0], plus * slopes[k][1]
    return (1 + 3 / m ** 0.5) * tol2 ** 0.5


def _reference(g, avg, momentum, nesterov, steps, coefs=COEFS, eps=1e-7, scale=1.0):
    d, new = g.double(), None
    if momentum is not None:
        new = momentum * avg.double() + (1 - momentum) * d
        d = momentum * new + (1 - momentum) * d if nesterov else new
    x = d / (d.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        s = x @ x.t()
        x = coefs[0] * x + (coefs[1] * s + coefs[2] * (s @ s)) @ x
    return (x.t() if tall else x) * scale, new


def _matrix(shape, seed, kind="gradient"):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    r, c = shape
    a = torch.randn(r, c, generator=g, device="cuda")
    if kind == "gradient":
        q = max(1, min(r, c) // 8)
        a = a + 4 * torch.randn(r, q, generator=g, device="cuda") @ torch.randn(q, c, generator=g, device="cuda") / q ** 0.5
    return a * 1e-3


def _check(got, want, tol, what):
    err = float((got.double() - want).norm() / want.norm())
    assert err <= tol, f"{what}: {err:.2e} > {tol:.2e}"


SHAPES = [(1, 1), (1, 777), (777, 1), (7, 3), (64, 288), (128, 128), (129, 65), (65, 129), (127, 640), (333, 1037), (1037, 333), (512, 512), (1000, 512),
          (256, 2304), (520, 520), (40, 20000), (5, 320), (320, 128), (128, 321), (320, 129), (2048, 2050)]


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_matrix(ctx, shape, dt):
    g = _matrix(shape, seed=shape[0] + shape[1]).to(_dtype(dt))
    for steps, out_dt in ((5, ir.BF16), (1, ir.F16)):
        (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=dt, out_dtype=out_dt, momentum=None, steps=steps).launch([g])
        want, _ = _reference(g, None, None, False, steps)
        _check(o, want, _tolerance(out_dt, steps, g), f"{shape} {steps} steps")
    ctx.poll()


@pytest.mark.parametrize("nesterov", [True, False])
def test_a_list_with_momentum(ctx, nesterov):
    """70 matrices (two rounds of launches) of mixed shapes, scales of their own, averages updated in place, three steps in a row."""
    import torch
    shapes = [SHAPES[i % 11] for i in range(70)]
    scales = [0.2 + 0.1 * (i % 5) for i in range(70)]
    plan = hb.Plan.muon(ctx, shapes, grad_dtype=ir.BF16, momentum=0.95, nesterov=nesterov, scales=scales)
    avgs = [torch.zeros(s, device="cuda") for s in shapes]
    outs = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    for step in range(3):
        grads = [_matrix(s, seed=1000 * step + i).bfloat16() for i, s in enumerate(shapes)]
        old = [a.clone() for a in avgs]
        plan.launch(grads + avgs, outs + avgs)
        for i in range(len(shapes)):
            want, new = _reference(grads[i], old[i], 0.95, nesterov, 5, scale=scales[i])
            tol = 4 * u * (0.95 * old[i].double().abs() + 0.05 * grads[i].double().abs()) + 1e-40
            # 0.05 and 0.95 themselves are f32 values of the plan
            tol = tol + 2 * u * (old[i].double().abs() + grads[i].double().abs())
            assert bool(((avgs[i].double() - new).abs() <= tol).all()), i
            d = (0.95 * new + 0.05 * grads[i].double()) if nesterov else new
            _check(outs[i], want, _tolerance(ir.BF16, 5, d), f"matrix {i} {shapes[i]}")
    ctx.poll()


def test_singular_values_land_around_one(ctx):
    import torch
    for shape in ((256, 1024), (700, 300)):
        (o,) = hb.Plan.muon(ctx, [shape], momentum=None, out_dtype=ir.F16).launch([_matrix(shape, 3, "noise").bfloat16()])
        s = torch.linalg.svdvals(o.double())
        assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("coefs,steps", [((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 8), (COEFS, 6)])
def test_other_coefficients(ctx, coefs, steps):
    """Cubic and quintic steps that converge to the orthogonal factor."""
    shape = (96, 200)
    g = _matrix(shape, 4, "noise").bfloat16()
    (o,) = hb.Plan.muon(ctx, [shape], momentum=None, coefs=coefs, steps=steps).launch([g])
    want, _ = _reference(g, None, None, False, steps, coefs)
    _check(o, want, _tolerance(ir.BF16, steps, g, coefs), f"{coefs}")


@pytest.mark.parametrize("size", [1e-18, 1e-4, 1e4, 1e30])
def test_gradients_of_any_size(ctx, size):
    shape = (130, 190)
    g = _matrix(shape, 5) * size
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=None, eps=0.0).launch([g])
    want, _ = _reference(g, None, None, False, 5, eps=0.0)
    _check(o, want, _tolerance(ir.BF16, 5, g, eps=0.0), f"{size}")


@pytest.mark.parametrize("shape", [(64, 64), (333, 257), (1024, 2048)])
def test_a_gradient_of_one_entry(ctx, shape):
    """The norm is one entry: X's largest value is as far from its root-mean-square as it can be.

    Nothing averages over one value v, so half steps add up: X's high half twice in S and S itself are each 2^-11 off, 3 2^-11
    in v^2 and twice that in v^4, so a step is |b| v^3 3 2^-11 + |c| v^5 6 2^-11 off (B's diagonal and the term a X are f32
    and the pair's 2^-22), the later steps multiply that by their slopes, and the update is rounded once, 2^-8."""
    import torch
    g = torch.zeros(shape, device="cuda")
    g[shape[0] // 2, 3] = -0.37
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=None).launch([g])
    want, _ = _reference(g, None, None, False, 5)
    (a, b, c), v, off = COEFS, 1.0, 0.0
    for _ in range(5):
        off = off * abs(a + 3 * b * v ** 2 + 5 * c * v ** 4) + (abs(b) * v ** 3 * 3 + abs(c) * v ** 5 * 6) * 2.0 ** -11
        v = a * v + b * v ** 3 + c * v ** 5
    _check(o, want, 2.0 ** -8 + 1.1 * off / v, f"{shape}")    # 1.1: second order, f32 roundings
    assert int((o != 0).sum()) == 1


def test_a_zero_gradient_gives_a_zero_update_and_nan_stays_in_its_matrix(ctx):
    import torch
    shapes = [(100, 200), (130, 70), (64, 64)]
    g = [torch.zeros(shapes[0], device="cuda"), _matrix(shapes[1], 6), _matrix(shapes[2], 7)]
    g[1][5, 6] = float("nan")
    a, b, c = hb.Plan.muon(ctx, shapes, grad_dtype=ir.F32, momentum=None).launch(g)
    assert torch.equal(a, torch.zeros_like(a)) and bool(torch.isnan(b).all())
    want, _ = _reference(g[2], None, None, False, 5)
    _check(c, want, _tolerance(ir.BF16, 5, g[2]), "the matrix beside")


@pytest.mark.parametrize("shapes", [[(1, 1), (129, 65), (65, 131)], [(300, 520), (64, 288)], [(64, 288), (77, 3)], [(2050, 2047)]])
def test_writes_only_its_outputs(ctx, shapes):
    import torch
    plan = hb.Plan.muon(ctx, shapes, momentum=0.9)
    grads = [_matrix(s, 8).bfloat16() for s in shapes]
    avgs = [_matrix(s, 9) for s in shapes]
    outs = [Guarded(s[0] * s[1] * k) for k in (2, 4) for s in shapes]
    ws = Guarded(plan.workspace_bytes) if plan.workspace_bytes else None
    for _ in range(2):
        plan.launch_ptrs([t.data_ptr() for t in grads + avgs], [o.ptr for o in outs], ws.ptr if ws else 0)
    torch.cuda.synchronize()
    ctx.poll()
    for i, o in enumerate(outs):
        o.assert_bands(f"output {i}")
    if ws:
        ws.assert_bands("workspace")
    for o, w in zip(outs, plan.launch(grads + avgs)):
        assert torch.equal(o.payload(), w.reshape(-1).view(torch.uint8))   # the same bits, every time


@pytest.mark.parametrize("shapes", [[(256, 2304), (333, 1037), (1000, 512)], [(64, 288), (3, 7)], [(2048, 2304)]])
def test_streams_and_captured_graphs(ctx, shapes):
    import torch
    plan = hb.Plan.muon(ctx, shapes, momentum=0.9)
    data = [[_matrix(s, 10 + k).bfloat16() for s in shapes] + [_matrix(s, 20 + k) for s in shapes] for k in range(2)]
    want = [[t.clone() for t in plan.launch(d)] for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = plan.launch(data[0], stream=side)
    got2 = plan.launch(data[1])
    torch.cuda.synchronize()
    for a, b in zip(got + got2, want[0] + want[1]):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(plan.launch(d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    ctx.poll()
    for o, w in zip(outs, want):
        for a, b in zip(o, w):
            assert torch.equal(a, b)


def test_refused_launches(ctx):
    import torch
    plan = hb.Plan.muon(ctx, [(64, 64), (32, 8)], momentum=0.9)
    g = [_matrix((64, 64), 1).bfloat16(), _matrix((32, 8), 2).bfloat16()]
    a = [torch.zeros(64, 64, device="cuda"), torch.zeros(32, 8, device="cuda")]
    with pytest.raises(ValueError, match="4 inputs"):
        plan.launch(g)
    with pytest.raises(ValueError, match="input 1"):
        plan.launch([g[0], g[1].t().contiguous()] + a)
    with pytest.raises(ValueError, match="input 2"):
        plan.launch(g + [a[0].bfloat16(), a[1]])
    o = [torch.empty_like(v) for v in g]
    n = [torch.empty_like(v) for v in a]
    for ins, outs in (([*g, *a], [g[0], o[1], *n]), ([*g, *a], [*o, n[0], n[0][:4].view(32, 8)]), ([*g, *a], [o[0], o[0][:4].view(32, 8), *n])):
        with pytest.raises(hb.HeliumError, match="overlaps"):
            plan.launch(ins, outs)
    room = torch.empty(64 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(hb.HeliumError, match="16-byte aligned"):
        plan.launch([room[1:1 + 64 * 64].view(64, 64), g[1]] + a)


@pytest.mark.parametrize("shape", [(200, 300), (1024, 2304), (64, 288)])
def test_operand_wait_runs_out_and_context_survives(ctx, shape):
    """The producers stay silent (host-side injection): every wait ends at its limit, the poll reports it, the plan still works."""
    import torch
    g = _matrix(shape, 30).bfloat16()
    plan = hb.Plan.muon(ctx, [shape], momentum=None, steps=1)
    ctx.poll()
    plan.fault_injection(wait_limit_us=20_000, withhold_loads=True)
    plan.launch([g])
    torch.cuda.synchronize()
    with pytest.raises(hb.HeliumError) as ei:
        ctx.poll()
    assert ei.value.status == -5
    ctx.poll()
    plan.fault_injection()
    (o,) = plan.launch([g])
    ctx.poll()
    _check(o, _reference(g, None, None, False, 1)[0], _tolerance(ir.BF16, 1, g), "after the injection")
