"""Plan.launch on another stream than the current one: memory that is let go while that stream still works on it."""
import pytest

import helium_b200 as hb
from helium_b200 import ir

pytestmark = pytest.mark.gpu

WAIT = 100_000_000      # cycles: some 50 ms


def _cases(ctx):
    import torch
    x = torch.randn(2, 700, 64, device="cuda").bfloat16()
    yield hb.Plan.group_norm(ctx, "fwd", 2, 700, 64, 8, activation="silu"), [x, torch.rand(64, device="cuda"), torch.rand(64, device="cuda")]
    yield hb.Plan.muon(ctx, [(200, 300), (64, 288)], momentum=0.9), [torch.randn(200, 300, device="cuda").bfloat16(),
                                                                      torch.randn(64, 288, device="cuda").bfloat16(),
                                                                      torch.randn(200, 300, device="cuda"), torch.randn(64, 288, device="cuda")]


@pytest.mark.parametrize("raw", [False, True])
def test_inputs_let_go_behind_the_launch(ctx, raw):
    import torch
    for plan, data in _cases(ctx):
        want = plan.launch(data)
        side = torch.cuda.Stream()
        for given in (False, True):
            ins = [t.clone() for t in data]
            outs = [torch.empty_like(t) for t in want] if given else None
            keep = [torch.zeros_like(t) for t in want]
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                torch.cuda._sleep(WAIT)
            got = plan.launch(ins, outs, stream=side.cuda_stream if raw else side)
            with torch.cuda.stream(side):
                for k, t in zip(keep, got):
                    k.copy_(t)
            del ins, outs, got
            junk = [torch.full_like(t, float("nan")) for t in list(data) + list(want) for _ in range(4)]   # takes what is free
            torch.cuda.synchronize()
            for a, b in zip(keep, want):
                assert torch.equal(a, b)
            del junk
    ctx.poll()


def test_outputs_read_by_the_current_stream_and_let_go(ctx):
    import torch
    for plan, data in _cases(ctx):
        want = plan.launch(data)
        other = [-t for t in data]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = plan.launch(data, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(WAIT)
        copies = [t.clone() for t in got]
        del got
        for _ in range(8):
            plan.launch(other, stream=side)      # allocates on that stream
        torch.cuda.synchronize()
        for a, b in zip(copies, want):
            assert torch.equal(a, b)


def test_the_current_stream_given(ctx):
    import torch
    for plan, data in _cases(ctx):
        for s in (torch.cuda.current_stream(), torch.cuda.current_stream().cuda_stream):
            for a, b in zip(plan.launch(data, stream=s), plan.launch(data)):
                assert torch.equal(a, b)


def test_captured_on_a_side_stream(ctx):
    """The launch's stream joins a capture through an event, as any other stream does."""
    import torch
    for plan, data in _cases(ctx):
        want = plan.launch(data)
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            side.wait_stream(torch.cuda.current_stream())
            got = plan.launch(data, stream=side)
            torch.cuda.current_stream().wait_stream(side)
        for _ in range(2):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
