"""dropout + activation of values that the scaling carries out of range: an activation that gives zero gives zero of an infinity
too.  The definition is written with selections, act(v) = v where v > 0 (or NaN), else 0 (relu) / v / 10 (leaky), and likewise its
derivative; the comparison is bit for bit where there is a value, NaN for NaN elsewhere (NaN * 0 and inf * 0 on the CPU's side
never arise)."""
import math

import numpy as np
import pytest
import torch

from philox_ref import pieces

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def want(x, dy, p, seed, offset, act):
    t = int(p * 65536 + 0.5)
    keep = torch.from_numpy(pieces(np.arange(x.numel()), seed, offset) >= np.uint64(t)).view(x.shape)
    f = torch.tensor(65536.0) / torch.tensor(float(65536 - t))
    v, g = x.float() * f, dy.float() * f
    if act == "relu":
        v, g = torch.where(v < 0, torch.zeros(()), v), torch.where(x.float() > 0, g, torch.zeros(()))
    elif act == "leaky":
        v, g = torch.where(v < 0, v * torch.tensor(0.1), v), torch.where(x.float() > 0, g, g * torch.tensor(0.1))
    return torch.where(keep, v, torch.zeros(())).to(x.dtype), torch.where(keep, g, torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", [None, "relu", "leaky"])
def test_values_out_of_range(dt, act):
    from trace_amd import autograd as tag
    ends = [math.inf, -math.inf, math.nan, 3e38, -3e38, 1.0, -1.0, 0.0, -0.0, 1e-38, -1e-38]
    x = torch.tensor(ends).repeat_interleave(len(ends)).repeat(9).to(dt)       # every pair of a value and a gradient, 9 masks each
    dy = torch.tensor(ends).repeat(len(ends)).repeat(9).to(dt)
    for p, seed in ((0.5, 3), (0.0, 4), (0.9, 5)):
        y, dx = want(x, dy, p, seed, 1, act)
        leaf = x.to(DEV).requires_grad_(True)
        got = tag.dropout_act(leaf, p, seed, 1, act)
        got.backward(dy.to(DEV))
        for a, b, name in ((got.detach().cpu(), y, "y"), (leaf.grad.cpu(), dx, "dx")):
            assert torch.equal(a.isnan(), b.isnan()), (name, p, x[a.isnan() != b.isnan()][:4], dy[a.isnan() != b.isnan()][:4])
            assert torch.equal(a.nan_to_num(7.0, math.inf, -math.inf), b.nan_to_num(7.0, math.inf, -math.inf)), (name, p)
