"""One training step of a normalised convolution, the new operators together with the ones around them: convolution, group
norm + SiLU, the gradients of both, the filter gradient through Muon, he_sgd_momentum applying the update.

Every stage is held to 64 bits from the tensors that entered it.  Tolerances, relative, 2-norm: a bf16 tensor that was
rounded once is 0.42 * 2^-8 = 1.7e-3 off (half a step, spread over it and over the binade); a convolution's f32 sums add
2^-24 times the square root of their length, nothing beside it; f32 outputs of sums over bf16 values 1e-5; an update
1.7e-3 and at most 2e-3 of arithmetic (test_muon_gpu.py computes it from the singular values; the 64 x 288 filter's noise has
condition 10).  Weights: three roundings of f32."""
import ctypes as C

import pytest

import helium_b200 as hb
from helium_b200 import ir
from helium_b200._lib import check, lib
from test_muon_gpu import _reference, _tolerance

pytestmark = pytest.mark.gpu

N, HW, CIN, COUT, GROUPS, LR = 4, 14, 32, 64, 8, 0.02


class Step:
    def __init__(self, ctx):
        import torch
        g = torch.Generator(device="cuda").manual_seed(1)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        p = HW * HW
        self.conv = hb.Plan.conv2d(ctx, "fwd", batch=N, in_hw=(HW, HW), in_channels=CIN, out_channels=COUT, kernel=(3, 3), bias=True)
        self.wgrad = hb.Plan.conv2d(ctx, "bwd_filter", batch=N, in_hw=(HW, HW), in_channels=CIN, out_channels=COUT, kernel=(3, 3))
        self.fwd = hb.Plan.group_norm(ctx, "fwd", N, p, COUT, GROUPS, activation="silu")
        self.bwd = hb.Plan.group_norm(ctx, "bwd", N, p, COUT, GROUPS, activation="silu")
        self.muon = hb.Plan.muon(ctx, [(COUT, 9 * CIN)], momentum=0.9, scales=[0.5])
        self.w = rand(COUT, 3, 3, CIN) / (9 * CIN) ** 0.5
        self.w16 = self.w.bfloat16()
        self.bias, self.gamma, self.beta = 0.1 * rand(COUT), 1 + 0.1 * rand(COUT), 0.1 * rand(COUT)
        self.avg = torch.zeros(COUT, 9 * CIN, device="cuda")
        self.x = rand(N, HW, HW, CIN).bfloat16()
        self.da = rand(N, p, COUT).bfloat16()
        f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        b16 = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.y, self.dw, self.update = b16(N, HW, HW, COUT), b16(COUT, 3, 3, CIN), b16(COUT, 9 * CIN)
        self.a, self.mean, self.rstd = b16(N, p, COUT), f32(N, GROUPS), f32(N, GROUPS)
        self.dy, self.dgamma, self.dbeta = b16(N, p, COUT), f32(COUT), f32(COUT)

    def run(self):
        import torch
        p = HW * HW
        self.conv.launch([self.x, self.w16, self.bias], [self.y])
        self.fwd.launch([self.y.view(N, p, COUT), self.gamma, self.beta], [self.a, self.mean, self.rstd])
        self.bwd.launch([self.da, self.y.view(N, p, COUT), self.gamma, self.beta, self.mean, self.rstd], [self.dy, self.dgamma, self.dbeta])
        self.wgrad.launch([self.dy.view(N, HW, HW, COUT), self.x], [self.dw])
        self.muon.launch([self.dw.view(COUT, 9 * CIN), self.avg], [self.update, self.avg])
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        check(lib.he_sgd_momentum(C.c_void_p(self.w.data_ptr()), None, C.c_void_p(self.update.data_ptr()), ir.BF16, C.c_void_p(self.w16.data_ptr()),
                                  self.w.numel(), LR, 0.0, 0, st))


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_two_steps_against_64_bits(ctx):
    import torch
    s = Step(ctx)
    p = HW * HW
    for _ in range(2):
        w16, w, avg = s.w16.double(), s.w.clone(), s.avg.clone()
        s.run()
        torch.cuda.synchronize()
        ctx.poll()
        nchw = lambda t: t.double().view(N, HW, HW, -1).permute(0, 3, 1, 2)  # noqa: E731
        y = torch.nn.functional.conv2d(nchw(s.x), w16.permute(0, 3, 1, 2), s.bias.double(), padding=1).permute(0, 2, 3, 1)
        assert _rel(s.y, y) <= 2e-3
        # group norm from the y that it read
        yy = s.y.double().view(N, p, COUT).requires_grad_()
        gamma, beta = s.gamma.double().requires_grad_(), s.beta.double().requires_grad_()
        yg = yy.view(N, p, GROUPS, COUT // GROUPS)
        mean = yg.mean((1, 3), keepdim=True)
        rstd = 1 / ((yg - mean).square().mean((1, 3), keepdim=True) + 1e-5).sqrt()
        z = ((yg - mean) * rstd).view(N, p, COUT) * gamma + beta
        a = z * torch.sigmoid(z)
        assert _rel(s.a, a) <= 2e-3
        a.backward(s.da.double())
        assert _rel(s.dy, yy.grad) <= 2e-3
        assert _rel(s.dgamma, gamma.grad) <= 1e-5 and _rel(s.dbeta, beta.grad) <= 1e-5
        # filter gradient from the dy that it read, the update from the gradient
        dw = torch.nn.grad.conv2d_weight(nchw(s.x), (COUT, CIN, 3, 3), nchw(s.dy), padding=1).permute(0, 2, 3, 1)
        assert _rel(s.dw, dw) <= 2e-3
        g = s.dw.view(COUT, 9 * CIN)
        want, new = _reference(g, avg, 0.9, True, 5, scale=0.5)
        assert _rel(s.avg, new) <= 1e-6
        assert _rel(s.update, want) <= _tolerance(ir.BF16, 5, 0.9 * new + 0.1 * g.double())
        assert bool(((s.w - (w - LR * s.update.float().view_as(w))).abs() <= 3 * 2.0 ** -24 * (w.abs() + 1)).all())
        assert torch.equal(s.w16, s.w.bfloat16())


def test_captured_steps_match_eager_ones(ctx):
    import torch
    a, b = Step(ctx), Step(ctx)
    for _ in range(4):
        a.run()
    b.run()                                  # kernels' one-time set-up stays outside the capture
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    ctx.poll()
    for name in ("w", "w16", "avg", "a", "dy", "dgamma", "update"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
