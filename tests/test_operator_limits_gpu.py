"""Group norm and Muon at the ends of what their entry points allow: the first launch of a process under capture, one plan from two
host threads, the longest and thinnest matrices, lists of thousands, 65535 pictures, the same tensor twice."""
import os
import subprocess
import sys
import threading

import pytest

import helium_b200 as hb
from helium_b200 import ir
from test_group_norm_gpu import _check_forward, _inputs
from test_muon_gpu import _check, _matrix, _reference, _tolerance

pytestmark = pytest.mark.gpu

CAPTURE_FIRST = """
import torch
import helium_b200 as hb
ctx = hb.Context(0)
gen = torch.Generator(device="cuda").manual_seed(1)
rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
plans = [(hb.Plan.group_norm(ctx, "fwd", 2, 700, 64, 8, activation="silu"), [rand(2, 700, 64).bfloat16(), rand(64), rand(64)]),
         (hb.Plan.group_norm(ctx, "fwd", 1, 70001, 40, 8, activation="gelu"), [rand(1, 70001, 40).bfloat16(), rand(40), rand(40)]),
         (hb.Plan.group_norm(ctx, "bwd", 3, 437, 320, 32), [rand(3, 437, 320).bfloat16(), rand(3, 437, 320).bfloat16(), rand(320), rand(320),
                                                            rand(3, 32), rand(3, 32).abs()]),
         (hb.Plan.group_norm(ctx, "bwd", 1, 70001, 40, 8), [rand(1, 70001, 40).bfloat16(), rand(1, 70001, 40).bfloat16(), rand(40), rand(40),
                                                            rand(1, 8), rand(1, 8).abs()]),
         (hb.Plan.muon(ctx, [(64, 288)], momentum=None), [rand(64, 288).bfloat16()]),
         (hb.Plan.muon(ctx, [(300, 520), (64, 32)], momentum=0.9), [rand(300, 520).bfloat16(), rand(64, 32).bfloat16(), rand(300, 520), rand(64, 32)]),
         (hb.Plan.muon(ctx, [(2048, 2304)], momentum=None), [rand(2048, 2304).bfloat16()])]
torch.cuda.synchronize()
got = []
for plan, ins in plans:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = plan.launch(ins)
    got.append((graph, outs))
for graph, _ in got:
    graph.replay()
    graph.replay()
torch.cuda.synchronize()
ctx.poll()
for (plan, ins), (_, outs) in zip(plans, got):
    for a, b in zip(plan.launch(ins), outs):
        assert torch.equal(a, b), plan.description
torch.cuda.synchronize()
ctx.poll()
print("same bits")
"""


def test_first_launches_of_a_process_under_capture():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE_FIRST], capture_output=True, text=True, timeout=300, env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and "same bits" in r.stdout, r.stderr[-2000:]


def test_one_plan_from_two_host_threads(ctx):
    import torch
    cases = []
    for size in ((3, 437, 320, 32), (1, 70001, 40, 8)):
        x, gamma, beta, dy = _inputs(*size[:3], ir.BF16, 3)
        cases.append((hb.Plan.group_norm(ctx, "fwd", *size, activation="silu"), [x, gamma, beta]))
        st = [torch.zeros(size[0], size[3], device="cuda"), torch.ones(size[0], size[3], device="cuda")]
        cases.append((hb.Plan.group_norm(ctx, "bwd", *size, activation="silu"), [dy, x, gamma, beta] + st))
    for shapes in ([(300, 520), (129, 65)], [(64, 288)]):
        cases.append((hb.Plan.muon(ctx, shapes, momentum=None), [_matrix(s, 7).bfloat16() for s in shapes]))
    want = [[t.clone() for t in plan.launch(ins)] for plan, ins in cases]
    torch.cuda.synchronize()
    got, errors = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    for k, (plan, ins) in enumerate(cases):
                        got.append((k, plan.launch(ins)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001 -- handed to the test's thread
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(got) == 2 * 20 * len(cases)
    for k, outs in got:
        for a, b in zip(outs, want[k]):
            assert torch.equal(a, b)
    ctx.poll()


@pytest.mark.parametrize("shape", [(1, 1 << 20), (1 << 20, 1), (2, 1 << 19), (3, 1048573), (200, 99991)])
def test_long_thin_matrices(ctx, shape):
    g = _matrix(shape, 3, "noise")
    (o,) = hb.Plan.muon(ctx, [shape], grad_dtype=ir.F32, momentum=None).launch([g])
    want, _ = _reference(g, None, None, False, 5)
    _check(o, want, _tolerance(ir.BF16, 5, g if shape[0] <= shape[1] else g.t()), f"{shape}")
    ctx.poll()


@pytest.mark.parametrize("tall", [False, True])
def test_muon_offsets_past_32_bits(ctx, tall):
    """2.4e9 elements.  Row i has values in the columns k with k mod m = i only, all v_i: its singular value is v_i sqrt(n / m), S and
    B are diagonal and the update is v_i times a factor of its own, zero elsewhere.  Half steps add up for one singular value as
    in test_muon_gpu.test_a_gradient_of_one_entry: X's high half twice in S, S itself."""
    import torch
    m, n = 2304, 1 << 20
    g = torch.zeros((n, m) if tall else (m, n), dtype=torch.bfloat16, device="cuda")
    v = (1.0 + torch.arange(m, device="cuda") % 7) / 8 * torch.where(torch.arange(m, device="cuda") % 2 == 0, 1.0, -1.0)
    cols = torch.arange(n, device="cuda")
    rows = cols % m
    index = (cols, rows) if tall else (rows, cols)
    g[index] = v[rows].bfloat16()
    (o,) = hb.Plan.muon(ctx, [tuple(g.shape)], momentum=None).launch([g])
    ctx.poll()
    count = torch.bincount(rows, minlength=m).double()
    del g
    norm = (v.double() ** 2 * count).sum().sqrt()
    s = v.double().abs() * count.sqrt() / norm
    a, b, c = 3.4445, -4.7750, 2.0315
    off = torch.zeros_like(s)
    s0 = s.clone()
    for _ in range(5):
        off = off * (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs() + (abs(b) * s ** 3 * 3 + abs(c) * s ** 5 * 6) * 2.0 ** -11
        s = a * s + b * s ** 3 + c * s ** 5
    factor = s / s0 / norm                                   # update / gradient
    want = (v.double() * factor)[rows]
    tol = want.abs() * (2.0 ** -8 + 1.1 * (off / s.abs())[rows] + 2.0 ** -20)
    assert bool(((o[index].double() - want).abs() <= tol).all())
    o[index] = 0
    assert not bool(o.any())


def test_four_thousand_matrices(ctx):
    import torch
    shapes = [((3, 5), (17, 9), (40, 40), (129, 33))[i % 4] for i in range(4096)]
    grads = [_matrix(s, i, "noise").bfloat16() for i, s in enumerate(shapes)]
    outs = hb.Plan.muon(ctx, shapes, momentum=None).launch(grads)
    ctx.poll()
    for i in (0, 1, 2, 3, 62, 63, 64, 65, 2047, 2048, 4093, 4094, 4095):
        want, _ = _reference(grads[i], None, None, False, 5)
        _check(outs[i], want, _tolerance(ir.BF16, 5, grads[i]), f"{i}")
    # the same matrix at two places of the list comes out alike
    again = hb.Plan.muon(ctx, shapes, momentum=None).launch([grads[i % 4] for i in range(4096)])
    for i in range(4096):
        assert torch.equal(again[i], again[i % 4])


def test_the_same_tensor_twice(ctx):
    import torch
    g = _matrix((200, 300), 1).bfloat16()
    a = torch.randn(200, 300, device="cuda")
    plan = hb.Plan.muon(ctx, [(200, 300)] * 2, momentum=0.9)
    o1, o2, n1, n2 = plan.launch([g, g, a, a])
    assert torch.equal(o1, o2) and torch.equal(n1, n2)
    with pytest.raises(hb.HeliumError, match="overlaps"):
        plan.launch([g, g, a, a], [o1, o2, a, a])
    x, gamma, _, _ = _inputs(2, 50, 64, ir.BF16, 1)
    y, mean, rstd = hb.Plan.group_norm(ctx, "fwd", 2, 50, 64, 8).launch([x, gamma, gamma])
    _check_forward(plan, x, gamma, gamma, 8, "none", ir.BF16, y, mean, rstd)
    bwd = hb.Plan.group_norm(ctx, "bwd", 2, 50, 64, 8)
    for p, q in zip(bwd.launch([x, x, gamma, gamma, mean, rstd]), bwd.launch([x.clone(), x, gamma, gamma.clone(), mean, rstd])):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("size", [(65535, 1, 3, 1), (65535, 5, 16, 4), (65535, 1, 64, 64)])
def test_the_largest_batch(ctx, size, dt):
    import torch
    n, p, c, groups = size
    x, gamma, beta, dy = _inputs(n, p, c, dt, 5)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation="silu")
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "silu", dt, y, mean, rstd)
    # dbeta without an activation is the sum of dy
    dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt).launch([dy, x, gamma, beta, mean, rstd])
    want, size_of = dy.double().sum((0, 1)), dy.double().abs().sum((0, 1))
    assert bool(((dbeta.double() - want).abs() <= 64 * 2.0 ** -24 * size_of).all()) and not bool(torch.isnan(dx).any())


def test_a_closed_plan_is_refused(ctx):
    x, gamma, beta, _ = _inputs(1, 9, 16, ir.BF16, 1)
    plan = hb.Plan.group_norm(ctx, "fwd", 1, 9, 16, 4)
    plan.close()
    with pytest.raises(hb.HeliumError, match="null"):
        plan.launch([x, gamma, beta])


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("size", [(1, 4, 65536, 1), (2, 301, 65536, 2), (3, 5, 65535, 1), (1, 2, 65536, 32768), (1, 1, 65521, 1)])
def test_the_most_channels(ctx, size, dt):
    import torch
    n, p, c, groups = size
    x, gamma, beta, dy = _inputs(n, p, c, dt, 6)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation="gelu")
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "gelu", dt, y, mean, rstd)
    dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt).launch([dy, x, gamma, beta, mean, rstd])
    want, size_of = dy.double().sum((0, 1)), dy.double().abs().sum((0, 1))
    assert bool(((dbeta.double() - want).abs() <= 64 * 2.0 ** -24 * size_of).all()) and not bool(torch.isnan(dx).any())


@pytest.mark.parametrize("p,c,groups", [((1 << 31) - 1, 1, 1), ((1 << 31) - 3, 2, 2)])
def test_the_most_positions(ctx, p, c, groups):
    """Values -1, 0 and 1 (and 1 to 3 forward): sums of whole numbers.  Forward, the largest sum is 2^32: f32 adds partial sums beyond
    2^24 with half steps of 2^-24 each, some twenty of them behind one another: 32 u."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.empty(1, p, c, dtype=torch.bfloat16, device="cuda").random_(1, 4, generator=gen)
    sums = [0.0, 0.0]
    for k in range(0, p, 1 << 28):
        v = x[0, k:k + (1 << 28)].float()                # whole numbers below 2^24 a block of sum()'s own
        sums[0] = sums[0] + v.sum(0, dtype=torch.float64)
        sums[1] = sums[1] + (v * v).sum(0, dtype=torch.float64)
    mean64 = sums[0] / p
    rstd64 = 1 / (sums[1] / p - mean64 ** 2 + 1e-5).sqrt()
    one, zero = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    y, mean, rstd = hb.Plan.group_norm(ctx, "fwd", 1, p, c, groups).launch([x, one, zero])
    u = 2.0 ** -24
    assert bool(((mean[0].double() / mean64 - 1).abs() <= 32 * u).all()) and bool(((rstd[0].double() / rstd64 - 1).abs() <= 128 * u).all())
    for rows in (slice(0, 4096), slice(p // 2, p // 2 + 4096), slice(p - 4096, p)):
        want = (x[0, rows].double() - mean64) * rstd64
        assert bool(((y[0, rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()), rows
    del y
    dy = torch.empty_like(x).random_(-1, 2, generator=gen)
    m, r = torch.full((1, groups), 2.0, device="cuda"), torch.ones(1, groups, device="cuda")
    dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", 1, p, c, groups).launch([dy, x, one, zero, m, r])
    wb, wg = 0.0, 0.0
    for k in range(0, p, 1 << 28):
        d = dy[0, k:k + (1 << 28)].float()
        wb = wb + d.sum(0, dtype=torch.float64)
        wg = wg + (d * (x[0, k:k + (1 << 28)].float() - 2)).sum(0, dtype=torch.float64)
    assert torch.equal(dbeta.double(), wb) and torch.equal(dgamma.double(), wg)
    for rows in (slice(0, 4096), slice(p // 2, p // 2 + 4096), slice(p - 4096, p)):
        want = dy[0, rows].double() - wb / p - (x[0, rows].double() - 2) * wg / p
        assert bool(((dx[0, rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()), rows
