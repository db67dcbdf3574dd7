"""dbeta of a wide group over many chunks of rows.  With dy = d everywhere it is d P, and every partial sum is a multiple of d: what
is lost are the roundings of the sums alone, one more for every term that is added behind another.  csrc/norm_ops.hip adds a
thread's rows (8 or 16 of them here), pairs of rows side by side, lists of chunks / 32 chunks, those 32 in five steps, the samples:
each sum is half a step, 2^-24 of it, off at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("d", [0.3, 0.1, 1.0 / 3.0])
@pytest.mark.parametrize("N,P,C,G,rows,lists", [(1, 25088, 512, 1, 8 + 1, 49), (1, 25088, 512, 2, 8 + 1, 49), (2, 25088, 1024, 1, 16 + 1, 25)])
def test_dbeta_of_equal_gradients(d, N, P, C, G, rows, lists):
    from trace_amd import ops
    x = torch.randn((N, P, C), device=DEV)
    dy = torch.full_like(x, d)
    _, st = ops.group_norm_act(x, G, return_stats=True)
    _, _, db = ops.group_norm_act_backward(dy, x, st, G)
    want = N * P * float(dy[0, 0, 0])
    terms = rows + lists + 5 + (N - 1)
    assert float((db.double() - want).abs().max()) <= terms * 2.0 ** -24 * want * (1 + 1e-4)
