"""Group normalisation with an activation (he_plan_group_norm) against a plain implementation in 64 bits.

Tolerances, with u = 2^-24 (half a step of f32) and U the half step of the tensor's type: an output is rounded once, at
most U |value|; what is computed before that is f32.  A sum here passes at most 64 additions in a thread, 64 in the row
lanes, 70 in a group and the slices' fold, so a sum of t_i is at most 256 u sum |t_i| off, and each value takes fewer than
16 + 4 |z| further roundings (exp's argument alone makes |z| of them).  So an output is within
  U |y| + 512 u (1 + |z|) S,   S = what the value is made of, summed without signs (written out at each check)."""
import ctypes as C

import pytest

import helium_b200 as hb
from helium_b200 import ir
from helium_b200._lib import lib
from test_guard_bands_gpu import Guarded

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
HALF_STEP = {ir.BF16: 2.0 ** -8, ir.F16: 2.0 ** -11, ir.F32: 2.0 ** -24}
# f16 values below the normal range are rounded to multiples of 2^-24
FLOOR = {ir.BF16: 1e-38, ir.F16: 2.0 ** -25, ir.F32: 1e-38}
EPS = 1e-5


def _dtype(dt):
    import torch
    return {ir.BF16: torch.bfloat16, ir.F16: torch.float16, ir.F32: torch.float32}[dt]


def _act(z, act):
    import torch
    return {"none": z, "relu": z.clamp(min=0), "silu": z * torch.sigmoid(z), "gelu": z * torch.special.ndtr(z)}[act]


def _slope(z, act):
    import torch
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327


def _inputs(n, p, c, dt, seed, offset=0.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(n, p, c, generator=g, device="cuda") * (0.5 + torch.rand(c, generator=g, device="cuda")) +
         torch.randn(c, generator=g, device="cuda") + offset).to(_dtype(dt))
    gamma = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    beta = 0.3 * torch.randn(c, generator=g, device="cuda")
    dy = torch.randn(n, p, c, generator=g, device="cuda").to(_dtype(dt))
    return x, gamma, beta, dy


def _per_channel(v, c):
    """[n, groups] -> [n, 1, c]"""
    return v.repeat_interleave(c // v.shape[1], dim=1)[:, None, :]


def _forward64(x, gamma, beta, groups, act, eps=EPS):
    n, p, c = x.shape
    xg = x.double().reshape(n, p, groups, c // groups)
    mean = xg.mean((1, 3))
    var = (xg - mean[:, None, :, None]).square().mean((1, 3))
    rstd = 1.0 / (var + eps).sqrt()
    z = (x.double() - _per_channel(mean, c)) * _per_channel(rstd, c) * gamma.double() + beta.double()
    return _act(z, act), mean, rstd, z


def _check_forward(plan, x, gamma, beta, groups, act, dt, y, mean, rstd, eps=EPS):
    c = x.shape[2]
    want, wm, wr, z = _forward64(x, gamma, beta, groups, act, eps)
    size = _per_channel(x.double().abs().reshape(x.shape[0], x.shape[1], groups, -1).mean((1, 3)), c)
    # the sum of squares is taken about the mean: its relative error is that of the sum, halved by the square root
    # and the mean's own error enters squared (256 u size rstd)^2, far below it unless the spread is nothing next to the mean
    spread = 1 + (256 * u * size * _per_channel(wr, c)) ** 2 / u
    assert bool(((mean.double() - wm).abs() <= 256 * u * size[:, 0, ::c // groups] + 1e-38).all()), "mean"
    assert bool(((rstd.double() - wr).abs() <= 512 * u * wr * spread[:, 0, ::c // groups]).all()), "rstd"
    parts = gamma.double().abs() * (x.double().abs() + size) * _per_channel(wr, c) * spread + beta.double().abs()
    tol = HALF_STEP[dt] * want.abs() + 512 * u * (1 + z.abs()) * parts + FLOOR[dt]
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), (plan.description, float((err / tol).max()))


# (batch, positions, channels, groups): one position and one channel; channel counts that a 16-byte vector divides, meets
# halfway and does not divide; positions that end inside a super-row; one group and a group per channel; more vector
# columns than a CTA has threads; pictures of several slices and pictures that a cluster's shared memory holds
SIZES = [(1, 1, 1, 1), (3, 1, 5, 5), (2, 1, 512, 32), (1, 49, 512, 32), (4, 49, 64, 8), (5, 37, 60, 6), (3, 101, 77, 7), (7, 13, 3, 1),
         (2, 64, 24, 24), (3, 50, 320, 32), (1, 5000, 8, 1), (2, 777, 1, 1), (2, 9, 1023, 11), (1, 3, 8200, 8), (2, 4099, 96, 3),
         (1, 70001, 40, 8), (2, 33000, 64, 32), (130, 6, 16, 2),
         (2, 700001, 3, 1), (1, 120001, 77, 7), (2, 9001, 1023, 11), (1, 200000, 64, 8), (1, 5, 4096, 1), (2, 3, 2049, 3)]


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES)
def test_forward(ctx, size, dt):
    n, p, c, groups = size
    for act in ("none", "silu") if p * c > 100000 else ("none", "relu", "silu", "gelu"):
        x, gamma, beta, _ = _inputs(n, p, c, dt, seed=p + c)
        plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation=act, eps=EPS)
        y, mean, rstd = plan.launch([x, gamma, beta])
        _check_forward(plan, x, gamma, beta, groups, act, dt, y, mean, rstd)


@pytest.mark.parametrize("dt", [ir.BF16, ir.F16, ir.F32])
@pytest.mark.parametrize("size", SIZES)
def test_backward(ctx, size, dt):
    import torch
    n, p, c, groups = size
    for act in ("none", "silu") if p * c > 100000 else ("none", "relu", "silu", "gelu"):
        x, gamma, beta, dy = _inputs(n, p, c, dt, seed=2 * p + c)
        _, m64, r64, _ = _forward64(x, gamma, beta, groups, act)
        mean, rstd = m64.float(), r64.float()
        m, r = _per_channel(mean.double(), c), _per_channel(rstd.double(), c)
        xh = (x.double() - m) * r
        z = xh * gamma.double() + beta.double()
        if act == "relu":
            dy = torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)   # at the border two roundings are a gradient apart
        plan = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=dt, activation=act, eps=EPS)
        dx, dgamma, dbeta = plan.launch([dy, x, gamma, beta, mean, rstd])
        g = dy.double() * _slope(z, act)
        # a value's own error: the activation's slope, 512 u (1 + |z|) |dy|, and that of x - mean relative to xh
        eg = 512 * u * (1 + z.abs()) * dy.double().abs() * (1 + (x.double().abs() + m.abs()) * r * gamma.double().abs())
        ex = 4 * u * (x.double().abs() + m.abs()) * r
        tol_b = eg.sum((0, 1)) + 512 * u * g.abs().sum((0, 1))
        tol_g = (eg * xh.abs() + ex * g.abs()).sum((0, 1)) + 512 * u * (g * xh).abs().sum((0, 1))
        assert bool(((dbeta.double() - g.sum((0, 1))).abs() <= tol_b + 1e-38).all()), plan.description
        assert bool(((dgamma.double() - (g * xh).sum((0, 1))).abs() <= tol_g + 1e-38).all()), plan.description
        t = g * gamma.double()
        mean_of = lambda v: _per_channel(v.reshape(n, p, groups, -1).mean((1, 3)), c)  # noqa: E731
        want = r * (t - mean_of(t) - xh * mean_of(t * xh))
        ga = gamma.double().abs()
        tol = HALF_STEP[dt] * want.abs() + FLOOR[dt] + r * (
            ga * eg + mean_of(ga * eg) + 512 * u * (t.abs() + mean_of(t.abs())) +
            xh.abs() * (mean_of(ga * (eg * xh.abs() + ex * g.abs())) + 512 * u * mean_of((t * xh).abs())) + ex * mean_of((t * xh).abs()))
        err = (dx.double() - want).abs()
        assert bool((err <= tol).all()), (plan.description, float((err / tol).max()))


# A group per channel beyond what shared memory could list; columns are cut into blocks there, forward and backward alike.
MANY_GROUPS = [(1, 4, 65535, 65535), (2, 3, 50001, 50001), (1, 4, 65536, 65536)]


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
@pytest.mark.parametrize("size", MANY_GROUPS)
def test_many_groups(ctx, size, dt):
    test_forward(ctx, size, dt)
    test_backward(ctx, size, dt)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_backward_against_differences(ctx, act):
    """d/dt of sum(w y) along random directions of x, gamma and beta: central differences of the 64-bit forward."""
    import torch
    n, p, c, groups = 2, 21, 24, 4
    x, gamma, beta, dy = _inputs(n, p, c, ir.F32, seed=5)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=ir.F32, activation=act)
    _, mean, rstd = plan.launch([x, gamma, beta])
    dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, dtype=ir.F32, activation=act).launch([dy, x, gamma, beta, mean, rstd])
    gen = torch.Generator(device="cuda").manual_seed(6)
    h = 1e-5
    for which, grad in ((0, dx), (1, dgamma), (2, dbeta)):
        v = torch.randn(grad.shape, generator=gen, device="cuda", dtype=torch.float64)
        at = lambda s: _forward64(*[t.double() + (s * v if i == which else 0) for i, t in enumerate((x, gamma, beta))], groups, act)[0]  # noqa: E731,B023
        num = float((dy.double() * (at(h) - at(-h))).sum() / (2 * h))
        size = float((grad.double() * v).abs().sum())
        # third derivatives of the 64-bit forward are O(1): h^2 = 1e-10; the kernel's sums are f32
        assert abs(num - float((grad.double() * v).sum())) <= 2e-5 * size, which


@pytest.mark.parametrize("dt", [ir.BF16, ir.F32])
def test_mean_far_from_zero(ctx, dt):
    """The spread is 1/1000 of the mean (f32) or a few steps of the type (bf16): no cancellation in the variance."""
    n, p, c, groups = 2, 500, 64, 8
    x, gamma, beta, _ = _inputs(n, p, c, dt, seed=9, offset=1000.0 if dt == ir.F32 else 30.0)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=dt, activation="none")
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "none", dt, y, mean, rstd)


@pytest.mark.parametrize("size", [(64, 49, 512, 32), (40, 101, 77, 7)])
def test_a_mean_next_to_zero_keeps_its_digits(ctx, size):
    """Groups of spread 1 and mean ~0 whose first value is 3.  n values added as they come (a few in a thread, then a tree of some
    ten levels) leave an error of u sqrt(20 / 3n) by root mean square, 0.1 u at n = 784 and 0.08 u at n = 1111; a sum about the
    first value would leave about 2 u, the rounding of 3.  Allowed: 0.5 u."""
    import torch
    n, p, c, groups = size
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(n, p, c, generator=g, device="cuda")
    x = x - _per_channel(x.reshape(n, p, groups, -1).mean((1, 3)), c)
    x[:, 0, ::c // groups] = 3.0
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=ir.F32)
    assert "one pass" in plan.description
    _, mean, _ = plan.launch([x, torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")])
    want = x.double().reshape(n, p, groups, -1).mean((1, 3))
    assert float((mean.double() - want).square().mean().sqrt()) <= 0.5 * u


def test_an_outlier_first_and_a_constant_group(ctx):
    import torch
    n, p, c, groups = 2, 300, 32, 4
    x, gamma, beta, _ = _inputs(n, p, c, ir.F32, seed=10)
    x[0, 0, 0] = 1e4          # the first value a thread sees, far from all the others
    x[1, :, 8:16] = 3.25      # no spread at all: rstd = 1 / sqrt(eps), y = act(beta)
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, dtype=ir.F32, activation="silu")
    y, mean, rstd = plan.launch([x, gamma, beta])
    _check_forward(plan, x, gamma, beta, groups, "silu", ir.F32, y, mean, rstd)
    assert torch.equal(mean[1, 1], torch.tensor(3.25, device="cuda"))
    want = _act(beta[8:16].double(), "silu")
    assert bool(((y[1, :, 8:16].double() - want).abs() <= 64 * u * (1 + want.abs())).all())


@pytest.mark.parametrize("size", [(3, 100, 64, 8), (3, 101, 77, 7), (2, 33000, 64, 32)])
def test_a_nan_stays_in_its_group(ctx, size):
    import torch
    n, p, c, groups = size
    for bad in (float("nan"), float("inf")):
        x, gamma, beta, dy = _inputs(n, p, c, ir.BF16, seed=11)
        x[1, p - 1, 0] = bad
        y, mean, rstd = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, activation="relu").launch([x, gamma, beta])
        hit = torch.zeros(n, p, c, dtype=torch.bool, device="cuda")
        hit[1, :, :c // groups] = True
        assert bool(torch.isnan(y[hit]).all()) and not bool(torch.isnan(y[~hit]).any())
        dx, dgamma, dbeta = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, activation="silu").launch([dy, x, gamma, beta, mean, rstd])
        assert bool(torch.isnan(dx[hit]).all()) and not bool(torch.isnan(dx[~hit]).any())
        assert not bool(torch.isnan(dgamma[c // groups:]).any())


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("size,dt", [((3, 101, 77, 7), ir.BF16), ((2, 13, 3, 1), ir.F32), ((1, 7001, 40, 8), ir.F16), ((2, 33000, 64, 32), ir.BF16),
                                     ((3, 19, 320, 32), ir.BF16)])
def test_writes_only_its_outputs(ctx, size, dt, direction):
    import torch
    n, p, c, groups = size
    x, gamma, beta, dy = _inputs(n, p, c, dt, seed=12)
    st = [torch.zeros(n, groups, device="cuda"), torch.ones(n, groups, device="cuda")]
    ins = [x, gamma, beta] if direction == "fwd" else [dy, x, gamma, beta] + st
    plan = hb.Plan.group_norm(ctx, direction, n, p, c, groups, dtype=dt, activation="silu")
    size_of = {ir.BF16: 2, ir.F16: 2, ir.F32: 4}
    outs = []
    for shape, d in zip(plan.out_shapes, plan.out_dtypes):
        k = size_of[d]
        for v in shape:
            k *= v
        outs.append(Guarded(k))
    ws = Guarded(plan.workspace_bytes) if plan.workspace_bytes else None
    for _ in range(2):
        plan.launch_ptrs([t.data_ptr() for t in ins], [o.ptr for o in outs], ws.ptr if ws else 0)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        o.assert_bands(f"output {i}")
    if ws:
        ws.assert_bands("workspace")
    want = plan.launch(ins)
    for o, w in zip(outs, want):
        assert torch.equal(o.payload(), w.reshape(-1).view(torch.uint8))   # the same bits, every time


def test_offsets_past_32_bits(ctx):
    """More than 2^32 bytes and 2^31 elements; the last picture is checked."""
    import torch
    n, p, c, groups = 3, 11_500_003, 64, 8
    x = torch.empty(n, p, c, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(13)
    for i in range(n):
        x[i].normal_(generator=g)
    gamma, beta = torch.full((c,), 1.5, device="cuda"), torch.full((c,), 0.25, device="cuda")
    y, mean, rstd = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, activation="none").launch([x, gamma, beta])
    v = x[2].double().view(p, groups, c // groups)
    m = v.mean((0, 2))
    r = 1 / ((v - m[None, :, None]).square().mean((0, 2)) + EPS).sqrt()
    del v
    assert float((mean[2].double() - m).abs().max()) < 1e-6 and float((rstd[2].double() / r - 1).abs().max()) < 1e-5
    tail = x[2, -1000:].double()
    want = (tail - m.repeat_interleave(8)) * r.repeat_interleave(8) * 1.5 + 0.25
    assert bool(((y[2, -1000:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all())


def test_streams_and_captured_graphs(ctx):
    """Another stream than the current one, and two captured graphs of one plan replayed at the same time."""
    import torch
    n, p, c, groups = 2, 33000, 64, 32
    plan = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, activation="silu")
    data = []
    for seed in (20, 21):
        x, gamma, beta, dy = _inputs(n, p, c, ir.BF16, seed)
        _, m, r, _ = _forward64(x, gamma, beta, groups, "silu")
        data.append([dy, x, gamma, beta, m.float(), r.float()])
    want = [[t.clone() for t in plan.launch(d)] for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = plan.launch(data[0], stream=side)
    got2 = plan.launch(data[1])
    side.synchronize()
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
    for o, w in zip(outs, want):
        for a, b in zip(o, w):
            assert torch.equal(a, b)


def test_refused_launches(ctx):
    import torch
    n, p, c, groups = 2, 10, 16, 4
    plan = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups)
    x, gamma, beta, _ = _inputs(n, p, c, ir.BF16, 1)
    with pytest.raises(ValueError, match="3 inputs"):
        plan.launch([x, gamma])
    with pytest.raises(ValueError, match="input 0"):
        plan.launch([x.float(), gamma, beta])
    with pytest.raises(ValueError, match="input 1"):
        plan.launch([x, gamma[:8].contiguous(), beta])
    with pytest.raises(ValueError, match="contiguous"):
        plan.launch([x.transpose(0, 1).contiguous().transpose(0, 1), gamma, beta])
    st = torch.empty(n, groups, device="cuda")
    with pytest.raises(hb.HeliumError, match="overlaps"):
        plan.launch([x, gamma, beta], [x, st, st.clone()])
    room = torch.empty(x.numel() + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(hb.HeliumError, match="16-byte aligned"):
        plan.launch([room[1:1 + x.numel()].view(n, p, c), gamma, beta])
    ins = (C.c_void_p * 3)(x.data_ptr(), None, beta.data_ptr())
    outs = (C.c_void_p * 3)(room.data_ptr(), st.data_ptr(), st.data_ptr())
    big = torch.empty(plan.workspace_bytes + 256, dtype=torch.uint8, device="cuda")
    rc = lib.he_launch(plan._h, ins, outs, C.c_void_p((big.data_ptr() + 255) // 256 * 256), C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == -1 and b"input 1 is null" in lib.he_last_error_string()


@pytest.mark.parametrize("p", [10, 300000])   # one pass and two
def test_outputs_that_overlap_are_refused(ctx, p):
    import torch
    n, c, groups = 1, 16, 16
    x, gamma, beta, dy = _inputs(n, p, c, ir.BF16, 1)
    st = lambda: torch.ones(n, groups, device="cuda")  # noqa: E731
    vec = lambda: torch.ones(c, device="cuda")  # noqa: E731
    fwd = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups)
    s = st()
    for outs in ([x, st(), st()], [torch.empty_like(x), s, s], [torch.empty_like(x), st(), gamma.view(n, groups)],
                 [torch.empty_like(x), beta.view(n, groups), st()]):
        with pytest.raises(hb.HeliumError, match="overlaps"):
            fwd.launch([x, gamma, beta], outs)
    bwd = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups)
    mean, rstd, v = st(), st(), vec()
    for outs in ([x, vec(), vec()], [dy, vec(), vec()], [torch.empty_like(x), gamma, vec()], [torch.empty_like(x), vec(), beta],
                 [torch.empty_like(x), v, v], [torch.empty_like(x), mean.view(c), vec()]):
        with pytest.raises(hb.HeliumError, match="overlaps"):
            bwd.launch([dy, x, gamma, beta, mean, rstd], outs)


@pytest.mark.parametrize("size", [(3, 437, 320, 32), (1, 200000, 77, 7), (2, 33000, 64, 32), (2, 3, 2049, 3)])
def test_chains_on_two_streams_at_once(ctx, size):
    """Launches back to back on two streams, whose kernels overlap within a chain and between the streams: same bits each time."""
    import torch
    n, p, c, groups = size
    fwd = hb.Plan.group_norm(ctx, "fwd", n, p, c, groups, activation="silu")
    bwd = hb.Plan.group_norm(ctx, "bwd", n, p, c, groups, activation="silu")
    sets, want = [], []
    for seed in range(2):
        x, gamma, beta, dy = _inputs(n, p, c, ir.BF16, seed)
        y, mean, rstd = fwd.launch([x, gamma, beta])
        sets.append((x, gamma, beta, dy, mean, rstd))
        want.append([y, mean, rstd] + bwd.launch([dy, x, gamma, beta, mean, rstd]))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(20):
        for k, (x, gamma, beta, dy, mean, rstd) in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                got.append((k, fwd.launch([x, gamma, beta]) + bwd.launch([dy, x, gamma, beta, mean, rstd])))
    torch.cuda.synchronize()
    for k, outs in got:
        for a, b in zip(outs, want[k]):
            assert torch.equal(a, b)
