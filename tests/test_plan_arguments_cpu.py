"""Arguments of Plan.group_norm and Plan.muon that their C structures cannot hold, or only in part."""
import pytest

import helium_b200 as hb

BIG = 1 << 32


@pytest.mark.parametrize("change", [dict(batch=BIG + 1), dict(channels=BIG + 16), dict(groups=BIG + 4), dict(positions=(1 << 64) + 9),
                                    dict(dtype=BIG + 1), dict(batch=-BIG + 1)])
def test_group_norm_sizes_beyond_their_fields(change):
    args = dict(batch=1, positions=9, channels=16, groups=4)
    args.update(change)
    with pytest.raises(ValueError, match="does not fit"):
        hb.Plan.group_norm(None, "fwd", **args)


@pytest.mark.parametrize("change", [dict(steps=BIG + 5), dict(shapes=[((1 << 64) + 4, 4)]), dict(shapes=[(4, (1 << 64) + 4)]), dict(grad_dtype=BIG + 1),
                                    dict(out_dtype=BIG + 1)])
def test_muon_sizes_beyond_their_fields(change):
    args = dict(shapes=[(4, 4)])
    args.update(change)
    with pytest.raises(ValueError, match="does not fit"):
        hb.Plan.muon(None, **args)


@pytest.mark.parametrize("coefs", [(), (1.5,), (1.5, -0.5), (1.0, 0.0, 0.0, 0.0)])
def test_muon_takes_three_coefficients(coefs):
    with pytest.raises(ValueError, match="coefs"):
        hb.Plan.muon(None, [(4, 4)], coefs=coefs)


@pytest.mark.parametrize("shape", [(4,), (), (4, 4, 4), (64, 3, 3, 32)])
def test_muon_takes_matrices(shape):
    """A filter is given as its K x RSC matrix: of [K, R, S, C] the first two sizes alone would be another matrix."""
    with pytest.raises(ValueError, match="two sizes"):
        hb.Plan.muon(None, [(8, 8), shape])


def test_a_stream_of_another_device_is_refused():
    import torch

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0

    plan = hb.Plan.group_norm(None, "fwd", 1, 9, 16, 4)
    x = torch.zeros(1, 9, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        plan.launch([x, torch.zeros(16), torch.zeros(16)], stream=Stream())
