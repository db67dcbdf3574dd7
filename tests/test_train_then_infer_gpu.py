"""The inference path after a training step computes with the trained weights, not with copies folded before it: what a training loop
with validation passes in between sees."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NORMS = {"BN": dict(type='BN3d'), "GN": dict(type='GN', num_groups=8)}


def modules(norm, which):
    from trace_amd.resnet3d import Bottleneck3d, ConvModule, NonLocal3d
    cfg = NORMS[norm]
    if which == "conv":
        return ConvModule(64, 64, 1, norm_cfg=cfg)
    if which == "bottleneck":
        return Bottleneck3d(64, 32, downsample=ConvModule(64, 128, 1, bias=False, norm_cfg=cfg, act_cfg=None), norm_cfg=cfg)
    return NonLocal3d(64, sub_sample=True, use_scale=True, mode=which, norm_cfg=cfg, reduction=1)


@pytest.mark.parametrize("norm", ["BN", "GN"])
@pytest.mark.parametrize("which", ["conv", "bottleneck", "dot_product", "embedded_gaussian"])
def test_modules(norm, which):
    torch.manual_seed(3)
    m = modules(norm, which).to(DEV)
    x = torch.randn((2, 2, 6, 6, 64), device=DEV).bfloat16()
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    for _ in range(2):
        m.eval()
        with torch.no_grad():
            before = m.run(x)
        m.train()
        m.run_train(x).float().square().mean().backward()
        opt.step()
        opt.zero_grad()
        m.eval()
        with torch.no_grad():
            after = m.run(x)
        other = modules(norm, which).to(DEV).eval()
        other.load_state_dict(m.state_dict())
        with torch.no_grad():
            want = other.run(x)
        assert torch.equal(after, want) and not torch.equal(after, before)


@pytest.mark.parametrize("norm", ["BN", "GN"])
def test_network_and_its_graph(norm):
    from trace_amd.resnet3d import ResNet3d, i3d_dc5_config
    cfg = i3d_dc5_config()
    cfg["norm_cfg"] = dict(NORMS[norm], num_groups=32) if norm == "GN" else NORMS[norm]
    cfg["non_local_cfg"] = dict(cfg["non_local_cfg"], norm_cfg=cfg["norm_cfg"])
    torch.manual_seed(0)
    m = ResNet3d(**cfg)
    clip = torch.randn((1, 3, 8, 64, 64)) * 50
    if norm == "BN":
        m.calibrate_bn(clip)
    m.to(DEV)
    clip = clip.to(DEV)
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    m.eval()
    before = m.forward_ndhwc_graphed(clip).clone()
    m.train()
    m.forward_train(clip).float().square().mean().backward()
    opt.step()
    opt.zero_grad()
    m.eval()
    graphed, eager = m.forward_ndhwc_graphed(clip).clone(), m.forward_ndhwc(clip)
    other = ResNet3d(**cfg)
    other.load_state_dict(m.state_dict())
    other.to(DEV)
    other.eval()
    want = other.forward_ndhwc(clip)
    assert not torch.equal(want, before)
    assert torch.equal(eager, want) and torch.equal(graphed, want)


def test_captured_training_steps():
    """replays run no Python: entering train() is what drops the folded copies"""
    from trace_amd import ops
    m = modules("GN", "conv").to(DEV)
    x = torch.randn((2, 2, 6, 6, 64), device=DEV).bfloat16()

    def step():
        grads = torch.autograd.grad(m.run_train(x).float().square().mean(), list(m.parameters()))
        with torch.no_grad():
            for p, g in zip(m.parameters(), grads):
                p.sub_(0.5 * g)
    m.train()
    step()
    g = torch.cuda.CUDAGraph()
    with ops.capture(g):
        step()
    seen = []
    for _ in range(3):
        m.train()
        g.replay()
        m.eval()
        with torch.no_grad():
            seen.append((m.run(x), {k: v.clone() for k, v in m.state_dict().items()}))
    for after, state in seen:      # last: loading a state drops every folded copy
        other = modules("GN", "conv").to(DEV).eval()
        other.load_state_dict(state)
        with torch.no_grad():
            assert torch.equal(after, other.run(x))
    assert not torch.equal(seen[0][0], seen[2][0])


def test_frozen_stages_keep_their_folded_copies():
    """train() in every step costs no folding of what is not trained; a network that is thawed is folded again"""
    from trace_amd.resnet3d import ResNet3d, i3d_dc5_config
    cfg = dict(i3d_dc5_config(), norm_cfg=dict(type='GN', num_groups=32), frozen_stages=1)
    cfg["non_local_cfg"] = dict(cfg["non_local_cfg"], norm_cfg=cfg["norm_cfg"])
    torch.manual_seed(0)
    m = ResNet3d(**cfg).to(DEV)
    clip = torch.randn((1, 3, 8, 64, 64), device=DEV) * 50
    m.eval()
    m.forward_ndhwc(clip)
    frozen, live = m.layer1[0].conv2, m.layer2[0].conv2
    assert live._packed is not None
    m.train()
    m.forward_train(clip)
    assert live._packed is None
    kept = frozen.packed()[0]
    for _ in range(2):
        m.train()
        m.forward_train(clip)
        assert frozen.packed()[0] is kept and live._packed is None
    m.frozen_stages = 0
    m.train()
    assert frozen._packed is None
