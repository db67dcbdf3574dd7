"""ops.group_norm_act of samples without positions."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 0, 24), (3, 4, 0, 5, 24)])
def test_group_norm_statistics_without_positions(dt, shape):
    """mean 0 and 1 / sqrt(0 + eps): what the sums over nothing leave, and not what the memory held"""
    from trace_amd import autograd as tag, ops
    torch.full((2, 4, 2), 77.0, device=DEV), torch.full((3, 4, 2), 77.0, device=DEV)     # freed again: blocks the call may get
    x = torch.zeros(shape, dtype=dt, device=DEV)
    y, stats = ops.group_norm_act(x, 4, eps=0.25, return_stats=True)
    assert y.shape == x.shape
    assert torch.equal(stats.cpu(), torch.tensor([0.0, 2.0]).expand(shape[0], 4, 2))
    leaf, w = x.clone().requires_grad_(True), torch.ones(24, device=DEV, requires_grad=True)
    tag.group_norm_act(leaf, 4, w).float().sum().backward()
    assert leaf.grad.shape == x.shape and not w.grad.any()
