"""ops.dropout_act / autograd.dropout_act against the counter-based definition: masks and values are equal, bit for bit (one
product in 32 bits, one rounding - the CPU's arithmetic is the same)."""
import math

import numpy as np
import pytest
import torch

from philox_ref import pieces

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def want(x, p, seed, offset, act, dy=None):
    t = int(p * 65536 + 0.5)
    keep = torch.from_numpy(pieces(np.arange(x.numel()), seed, offset) >= np.uint64(t)).view(x.shape)
    f = torch.tensor(65536.0) / torch.tensor(float(65536 - t)) if t < 65536 else torch.tensor(0.0)
    low = {None: 1.0, "relu": 0.0, "leaky": 0.1}[act]
    v = x.float() * f
    y = torch.where(keep, torch.where(v < 0, v * torch.tensor(low), v), torch.zeros(()))
    if dy is None:
        return y.to(x.dtype)
    g = dy.float() * f
    g = torch.where(x.float() > 0, g, g * torch.tensor(low))
    return y.to(x.dtype), torch.where(keep, g, torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2049, 100003])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", [None, "relu", "leaky"])
def test_values_and_gradients(n, dt, act):
    from trace_amd import autograd as tag, ops
    g = torch.Generator().manual_seed(n)
    x, dy = torch.randn(n, generator=g).to(dt), torch.randn(n, generator=g).to(dt)
    for p, seed, off in ((0.5, 1, 0), (0.1, (1 << 64) - 3, (1 << 40) + 5), (0.9, 77, (1 << 64) - 1)):
        y, dx = want(x, p, seed, off, act, dy)
        leaf = x.to(DEV).requires_grad_(True)
        got = tag.dropout_act(leaf, p, seed, off, act)
        got.backward(dy.to(DEV))
        assert torch.equal(got.detach().cpu(), y) and torch.equal(leaf.grad.cpu(), dx)
        assert torch.equal(ops.dropout_act(x.to(DEV), p, seed, off, act).cpu(), y)


def test_probabilities_ends_and_eval():
    from trace_amd import autograd as tag, ops
    x = torch.randn((64, 1024), device=DEV)
    x[0, 0], x[0, 1] = math.inf, math.nan
    assert torch.equal(ops.dropout_act(x, 0.0, 5).nan_to_num(1.5), x.nan_to_num(1.5))
    assert not ops.dropout_act(x, 1.0, 5).any()                      # nothing is kept, not even infinities
    y = tag.dropout_act(x, 0.7, 5, training=False)
    assert torch.equal(y.nan_to_num(1.5), x.nan_to_num(1.5))
    one = torch.ones(1 << 22, device=DEV)
    for p in (0.01, 0.3, 0.5):
        m = float(ops.dropout_act(one, p, 123).mean())
        assert abs(m - 1) < 6 * math.sqrt(p / (1 - p) / one.numel())     # six standard deviations of the mean
    a, b = (ops.dropout_act(one, 0.5, 9, o) for o in (0, 1))
    assert abs(float(((a > 0) == (b > 0)).float().mean()) - 0.5) < 6 * 0.5 / math.sqrt(one.numel())


def test_positions_past_32_bits_of_bytes():
    """element numbers behind 2^31: the last elements of a 2^31 + 13 long map"""
    from trace_amd import ops
    n = (1 << 31) + 13
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = ops.dropout_act(x, 0.5, 42, 7)
    i = np.concatenate([np.arange(64), np.arange((1 << 31) - 40, n)])
    keep = pieces(i, 42, 7) >= np.uint64(32768)
    got = y[torch.from_numpy(i).to(DEV)].float().cpu().numpy()
    assert np.array_equal(got, np.where(keep, 2.0, 0.0))


def test_views_and_steps_and_replays():
    from trace_amd import autograd as tag, ops
    x = torch.randn((40, 70), device=DEV)
    assert torch.equal(ops.dropout_act(x.t(), 0.5, 3), ops.dropout_act(x.t().contiguous(), 0.5, 3))
    odd = torch.randn(1001, device=DEV)[1:]
    assert torch.equal(ops.dropout_act(odd, 0.5, 3), ops.dropout_act(odd.clone(), 0.5, 3))
    step = torch.tensor([4], device=DEV)
    assert torch.equal(ops.dropout_act(x, 0.5, 3, 10, step=step), ops.dropout_act(x, 0.5, 3, 14))
    leaf = x.clone().requires_grad_(True)
    y = tag.dropout_act(leaf, 0.5, 3, 10, step=step)
    step += 1
    with pytest.raises(RuntimeError):          # the mask of the forward pass could not be drawn again
        y.sum().backward()

    def one():
        a = x.detach().requires_grad_(True)
        y = tag.dropout_act(a, 0.5, 3, 10, "leaky", step)
        return y.detach(), torch.autograd.grad(y, a, x)[0]
    one()
    gr = torch.cuda.CUDAGraph()
    with ops.capture(gr):
        res = one()
    seen = []
    for rep in range(4):
        step.fill_(rep)
        x.normal_()
        w = one()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, w)), rep
        seen.append(res[0] != 0)
    assert not torch.equal(seen[0], seen[1])


def test_relation_logits_train():
    """the model's path: both relation MLPs with their dropout, against torch in 64 bits with the same masks, and their gradients"""
    from trace_amd.config import TraceConfig
    from trace_amd.model_builder_rel import Generalized_RCNN
    torch.manual_seed(0)
    m = Generalized_RCNN(TraceConfig(RESIZE_HIDDEN_DIM=4), conv_bodies=False)
    P, K = 57, m.relation_infer_sem[2].in_features
    sem, spa, part = torch.randn(P, K), torch.randn(P, K), torch.randn(P, m.cfg.NUM_PRD_CLASSES)
    m.relation_infer_sem.to(DEV)
    m.relation_infer_spa.to(DEV)
    m.train()
    a, b = (t.bfloat16().to(DEV).requires_grad_(True) for t in (sem, spa))
    out = m.relation_logits_train(a, b, 11, 3, part.to(DEV))
    r = torch.randn(out.shape).bfloat16().float()
    (out * r.to(DEV)).sum().backward()
    ref, leaves = part.double(), []
    for x, seq, key in ((sem, m.relation_infer_sem, 11), (spa, m.relation_infer_spa, 11 + (1 << 63))):
        keep = torch.from_numpy(pieces(np.arange(P * K), key, 3) >= np.uint64(32768)).view(P, K).double()
        x = x.bfloat16().double().requires_grad_(True)
        w = seq[2].weight.detach().cpu().bfloat16().double().requires_grad_(True)
        h = torch.nn.functional.leaky_relu(x * keep * 2, 0.1)
        ref = ref + h @ w.t() + seq[2].bias.detach().cpu().double()
        leaves.append((x, w))
    (ref * r.double()).sum().backward()

    def rel(g, w):
        return float((g.detach().double().cpu() - w.detach()).norm() / w.detach().norm())
    assert rel(out, ref) < 2e-2
    for (x, w), got, seq in zip(leaves, (a, b), (m.relation_infer_sem, m.relation_infer_spa)):
        assert rel(got.grad, x.grad) < 2e-2 and rel(seq[2].weight.grad, w.grad) < 2e-2
    m.eval()
    e1, e2 = m.relation_logits_train(a, b, 11, 3), m.relation_logits_train(a, b, 12, 4)
    assert torch.equal(e1, e2)


def test_refusals():
    from trace_amd import ops
    x = torch.zeros(10, device=DEV)
    for args, kw in (((x, -0.1, 0), {}), ((x, 1.1, 0), {}), ((x, float("nan"), 0), {}), ((x, 0.5, -1), {}), ((x, 0.5, 1 << 64), {}),
                     ((x, 0.5, 0, -1), {}), ((x.half(), 0.5, 0), {}), ((x.cpu(), 0.5, 0), {}), ((x, 0.5, 0), dict(act="silu")),
                     ((x, 0.5, 0), dict(step=torch.zeros(1, dtype=torch.int64))), ((x, 0.5, 0), dict(step=torch.zeros(1, device=DEV)))):
        with pytest.raises(RuntimeError):
            ops.dropout_act(*args, **kw)
    for args, kw in (((x, None, 0.5, 0), dict(act="relu")), ((x, x[:5], 0.5, 0), dict(act="relu")), ((x, x.bfloat16(), 0.5, 0), dict(act="relu"))):
        with pytest.raises(RuntimeError):
            ops.dropout_act_backward(*args, **kw)
