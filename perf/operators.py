"""Cases, plain forms and definitions of the operators that are measured: group normalisation with an activation over
channels-last tensors (forward and backward), and the orthogonalised update of the Muon optimiser (Newton-Schulz products,
with or without the momentum average in front of them).

A case is a dict of plain values.  `run` computes it in its plain form, with elementary torch operations in f32, or
(`own`) through the framework's own entry points; `exact` computes the same from the definition in 64 bits."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
COEFS = (3.4445, -4.7750, 2.0315)   # the quintic of the Muon optimiser
NORM_EPS = 1e-7                     # added to the Frobenius norm of an update before it divides
EPS = 1e-5                          # added to the variance of a group


def _gn(name, direction, batch, height, width, channels, groups, dtype, activation):
    return {"name": name, "op": "group_norm", "direction": direction, "batch": batch, "height": height, "width": width,
            "channels": channels, "groups": groups, "dtype": dtype, "activation": activation}


def _muon(name, shapes, dtype, momentum, nesterov=True, steps=5):
    return {"name": name, "op": "muon", "shapes": shapes, "dtype": dtype, "momentum": momentum, "nesterov": nesterov, "steps": steps}


def _conv_filters():
    """Filters of the conv net's 22 convolutions as matrices: output channels x (taps * input channels)."""
    s, c = ["32x152"], 32
    for _ in range(4):
        o = 2 * c
        s += ["%dx%d" % (o, 9 * c), "%dx%d" % (o, 9 * o), "%dx%d" % (o, c), "%dx%d" % (o, 9 * o), "%dx%d" % (o, 9 * o)]
        c = o
    return ",".join(s + ["1000x512"])


def listed():
    return [
        # one picture through the last segment: 7 x 7 positions of 512 channels, where the call's latency is all there is
        _gn("gn_fwd_one_picture", "fwd", 1, 7, 7, 512, 32, "bf16", "silu"),
        # a training batch of the conv net's second segment
        _gn("gn_fwd_segment", "fwd", 128, 28, 28, 128, 32, "bf16", "relu"),
        # the activation tensor of the pointwise benchmark, [64, 56, 56, 256]
        _gn("gn_fwd_wide", "fwd", 64, 56, 56, 256, 32, "bf16", "silu"),
        # odd sizes in f32: channels that no 16-byte vector divides, an odd number of positions, 11 channels a group
        _gn("gn_fwd_odd_f32", "fwd", 5, 37, 53, 77, 7, "f32", "gelu"),
        # gradients of the second segment's normalisation
        _gn("gn_bwd_segment", "bwd", 128, 28, 28, 128, 32, "bf16", "silu"),
        # gradients at image resolution: few pictures, each larger than any one multiprocessor's memory by far
        _gn("gn_bwd_picture_512", "bwd", 2, 512, 512, 128, 32, "f16", "silu"),
        # a small ragged batch: groups of 10 channels, so that a 16-byte vector meets two groups
        _gn("gn_bwd_ragged", "bwd", 3, 19, 23, 320, 32, "bf16", "gelu"),
        # one filter of the first segment, alone
        _muon("muon_one_filter", "64x288", "bf16", 0.0),
        # the whole optimiser step of the conv net: momentum and direction of all 22 filters
        _muon("muon_conv_net", _conv_filters(), "bf16", 0.95),
        # odd sizes, both orientations, f32 gradients
        _muon("muon_odd_f32", "333x1037,1037x333,1x777,129x65", "f32", 0.9, nesterov=False),
        # a square projection of the transformer block's width
        _muon("muon_square", "4096x4096", "bf16", 0.0),
        # the transformer block's two weight gradients, [4096, 16384] and [16384, 4096]
        _muon("muon_mlp_block", "4096x16384,16384x4096", "bf16", 0.95),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        direction = rng.choice(["fwd", "bwd"])
        while True:
            groups = rng.choice([1, 2, 3, 4, 7, 8, 16, 32, 32, 32])
            channels = groups * _log(rng, 1, 64)
            batch, height, width = _log(rng, 1, 128), _log(rng, 1, 512), _log(rng, 1, 512)
            if 2 <= height * width * channels // groups and 256 <= batch * height * width * channels <= 24_000_000 and channels <= 1024:
                break
        # the rectifier's gradient jumps where its argument is zero, and there two roundings of one sum differ by all of it:
        # backward cases have the activations whose gradients are continuous
        acts = ["none", "relu", "silu", "gelu"] if direction == "fwd" else ["none", "silu", "gelu"]
        c = _gn("", direction, batch, height, width, channels, groups, rng.choice(["bf16", "f16", "f32"]), rng.choice(acts))
    else:
        shapes = []
        for _ in range(rng.choice([1, 1, 2, 3, 6])):
            shapes.append("%dx%d" % (_log(rng, 4, 2048), _log(rng, 4, 4096)))
        c = _muon("", ",".join(shapes), rng.choice(["bf16", "f16", "f32"]), rng.choice([0.0, 0.9, 0.95]), rng.random() < 0.5,
                  rng.choice([3, 5, 5, 6]))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------

def _gn_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, p, ch, gr = c["batch"], c["height"] * c["width"], c["channels"], c["groups"]
    dt = DTYPES[c["dtype"]]
    rand = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    # activations whose channels have means and spreads of their own, as a convolution with a bias leaves them
    x = (rand(n, p, ch) * (0.5 + rand(ch).abs()) + rand(ch)).to(dt)
    s = {"x": x, "gamma": 1.0 + 0.2 * rand(ch), "beta": 0.2 * rand(ch)}
    if c["direction"] == "bwd":
        s["dy"] = rand(n, p, ch).to(dt)
        xg = x.view(n, p, gr, ch // gr).double()
        mean = xg.mean(dim=(1, 3))
        var = (xg - mean[:, None, :, None]).square().mean(dim=(1, 3))
        s["mean"], s["rstd"] = mean.float(), (1.0 / torch.sqrt(var + EPS)).float()
    return s


def _shapes(c):
    return [tuple(int(v) for v in s.split("x")) for s in c["shapes"].split(",")]


def _muon_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731

    def gradient(r, k):
        # a few strong directions over a floor of noise: the spectrum that weight gradients have
        q = max(1, min(r, k, 64) // 4)
        decay = torch.arange(1, q + 1, device="cuda", dtype=torch.float32) ** -0.5
        return (rand(r, q) * decay) @ rand(q, k) / math.sqrt(q) + rand(r, k)

    s = {"grads": [(1e-3 * gradient(r, k)).to(DTYPES[c["dtype"]]) for r, k in _shapes(c)]}
    if c["momentum"]:
        s["averages"] = [5e-4 * gradient(r, k) for r, k in _shapes(c)]
    return s


def _context():
    import helium_b200

    if not hasattr(_context, "ctx"):
        _context.ctx = helium_b200.Context(torch.cuda.current_device())
    return _context.ctx


def _plan(c):
    import helium_b200
    from helium_b200 import ir

    dtype = {"bf16": ir.BF16, "f16": ir.F16, "f32": ir.F32}[c["dtype"]]
    if c["op"] == "group_norm":
        return helium_b200.Plan.group_norm(_context(), c["direction"], c["batch"], c["height"] * c["width"], c["channels"], c["groups"],
                                           dtype=dtype, activation=c["activation"], eps=EPS)
    return helium_b200.Plan.muon(_context(), _shapes(c), grad_dtype=dtype, out_dtype=ir.BF16, momentum=c["momentum"] or None,
                                 nesterov=c["nesterov"], steps=c["steps"], coefs=COEFS, eps=NORM_EPS)


def prepare(case, seed):
    s = _gn_inputs(case, seed) if case["op"] == "group_norm" else _muon_inputs(case, seed)
    s["case"] = case
    if own:
        s["plan"] = _plan(case)   # what a program makes once for a layer, or for its list of weights
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def _activate(z, activation):
    if activation == "relu":
        return torch.clamp(z, min=0.0)
    if activation == "silu":
        return z / (1.0 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, activation):
    if activation == "relu":
        return (z > 0).to(z.dtype)
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if activation == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(z)


def _gn_fwd_plain(c, s):
    n, p, ch, gr = c["batch"], c["height"] * c["width"], c["channels"], c["groups"]
    x = s["x"].float().view(n, p, gr, ch // gr)
    mean = x.mean(dim=(1, 3), keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    z = (d * rstd).view(n, p, ch) * s["gamma"] + s["beta"]
    return [_activate(z, c["activation"]).to(s["x"].dtype), mean.view(n, gr), rstd.view(n, gr)]


def _gn_bwd_plain(c, s):
    n, p, ch, gr = c["batch"], c["height"] * c["width"], c["channels"], c["groups"]
    xh = ((s["x"].float().view(n, p, gr, ch // gr) - s["mean"][:, None, :, None]) * s["rstd"][:, None, :, None]).view(n, p, ch)
    g = s["dy"].float() * _slope(xh * s["gamma"] + s["beta"], c["activation"])
    dgamma, dbeta = (g * xh).sum(dim=1).sum(dim=0), g.sum(dim=1).sum(dim=0)
    t = (g * s["gamma"]).view(n, p, gr, ch // gr)
    xg = xh.view(n, p, gr, ch // gr)
    dx = s["rstd"][:, None, :, None] * (t - t.mean(dim=(1, 3), keepdim=True) - xg * (t * xg).mean(dim=(1, 3), keepdim=True))
    return [dx.view(n, p, ch).to(s["x"].dtype), dgamma, dbeta]


def _muon_plain(c, s):
    updates, averages = [], []
    m = c["momentum"]
    for i, g in enumerate(s["grads"]):
        d = g.float()
        if m:
            avg = m * s["averages"][i] + (1.0 - m) * d
            averages.append(avg)
            d = m * avg + (1.0 - m) * d if c["nesterov"] else avg
        x = d / (torch.sqrt((d * d).sum()) + NORM_EPS)
        x = x.t() if d.shape[0] > d.shape[1] else x
        for _ in range(c["steps"]):
            a = x @ x.t()
            x = COEFS[0] * x + (COEFS[1] * a + COEFS[2] * (a @ a)) @ x
        updates.append((x.t() if d.shape[0] > d.shape[1] else x).to(torch.bfloat16))
    return updates + averages


def run(state):
    c = state["case"]
    if c["op"] == "group_norm":
        if own:
            names = ("x", "gamma", "beta") if c["direction"] == "fwd" else ("dy", "x", "gamma", "beta", "mean", "rstd")
            return state["plan"].launch([state[k] for k in names])
        return (_gn_fwd_plain if c["direction"] == "fwd" else _gn_bwd_plain)(c, state)
    if own:
        return state["plan"].launch(state["grads"] + state.get("averages", []))
    return _muon_plain(c, state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    if case["op"] == "group_norm":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["batch"] * case["height"] * case["width"] * case["channels"]
        stats, params = 8 * case["batch"] * case["groups"], 8 * case["channels"]
        fwd = case["direction"] == "fwd"
        # forward: x in, y and the statistics out; backward: dy, x, the statistics in, dx and the parameters' gradients out
        return {"bytes": (2 * n * size + params + stats) if fwd else (3 * n * size + 2 * params + stats), "flops": (8 if fwd else 16) * n}
    byts = flops = 0
    for r, k in _shapes(case):
        m, n = min(r, k), max(r, k)
        # the gradient in and the update out, and the average in and out; of the symmetric products x x^T and a a one half is
        # enough: m^2 n + m^3 operations, and 2 m^2 n for the last product of a step
        byts += m * n * ((4 if case["dtype"] == "f32" else 2) + 2 + (8 if case["momentum"] else 0))
        flops += case["steps"] * (3 * m * m * n + m ** 3)
    return {"bytes": byts, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _gn_exact(c, s):
    """A picture at a time: the moments of each group, then the map of each value; the backward pass by the chain rule through
    the mean and the variance rather than by its closed form."""
    n, p, ch, gr = c["batch"], c["height"] * c["width"], c["channels"], c["groups"]
    per = ch // gr
    gamma, beta = s["gamma"].double().view(gr, 1, per), s["beta"].double().view(gr, 1, per)
    count = p * per
    act = c["activation"]
    outs, first, second = [], [], []
    for i in range(n):
        x = s["x"][i].double().view(p, gr, per).transpose(0, 1)              # [group, position, channel in it]
        if c["direction"] == "fwd":
            mean = x.sum((1, 2)) / count
            var = (x * x).sum((1, 2)) / count - mean * mean
            rstd = (var.clamp(min=0.0) + EPS).rsqrt()
        else:
            mean, rstd = s["mean"][i].double(), s["rstd"][i].double()
        dev = x - mean.view(gr, 1, 1)
        z = dev * rstd.view(gr, 1, 1) * gamma + beta
        if c["direction"] == "fwd":
            y = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.special.expit(v),
                 "gelu": lambda v: v * torch.special.ndtr(v)}[act](z)
            outs.append(y.transpose(0, 1).reshape(p, ch))
            first.append(mean)
            second.append(rstd)
            continue
        if act == "none":
            slope = torch.ones_like(z)
        elif act == "relu":
            slope = torch.heaviside(z, torch.zeros_like(z))
        elif act == "silu":
            e = torch.special.expit(z)
            slope = e + z * e * torch.special.expit(-z)
        else:
            slope = torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * (0.5 * math.sqrt(2 / math.pi))
        g = s["dy"][i].double().view(p, gr, per).transpose(0, 1) * slope
        first.append((g * dev * rstd.view(gr, 1, 1)).sum(1).reshape(ch))
        second.append(g.sum(1).reshape(ch))
        h = g * gamma                                                        # d loss / d normalised value
        dvar = -0.5 * (h * dev).sum((1, 2)) * rstd ** 3
        dmean = -(h.sum((1, 2)) * rstd)
        dx = h * rstd.view(gr, 1, 1) + (2.0 / count) * dvar.view(gr, 1, 1) * dev + (dmean / count).view(gr, 1, 1)
        outs.append(dx.transpose(0, 1).reshape(p, ch))
    first, second = torch.stack(first), torch.stack(second)
    return [torch.stack(outs), first, second] if c["direction"] == "fwd" else [torch.stack(outs), first.sum(0), second.sum(0)]


def _muon_exact(c, s):
    """Through the eigenvectors of the Gram matrix: a step multiplies the singular value v by a + b v^2 + c v^4."""
    updates, averages = [], []
    for i, g in enumerate(s["grads"]):
        d = g.double()
        if c["momentum"]:
            avg = s["averages"][i].double() + (1.0 - c["momentum"]) * (d - s["averages"][i].double())
            averages.append(avg)
            d = d + c["momentum"] * (avg - d) if c["nesterov"] else avg
        norm = torch.linalg.vector_norm(d) + NORM_EPS
        tall = d.shape[0] > d.shape[1]
        w = d.mT if tall else d
        lam, u = torch.linalg.eigh(w @ w.mT)
        v2 = lam.clamp(min=0.0) / norm ** 2
        factor = torch.ones_like(v2)
        for _ in range(c["steps"]):
            f = COEFS[0] + COEFS[1] * v2 + COEFS[2] * v2 * v2
            factor, v2 = factor * f, v2 * f * f
        o = (u * factor) @ (u.mT @ w) / norm
        updates.append(o.mT.contiguous() if tall else o)
    return updates + averages


def exact(case, seed):
    if case["op"] == "group_norm":
        return _gn_exact(case, _gn_inputs(case, seed))
    return _muon_exact(case, _muon_inputs(case, seed))
