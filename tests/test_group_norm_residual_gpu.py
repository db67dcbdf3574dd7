"""GroupNorm networks with an f32 residual stream (ResNet3d.res_f32_stages, Bottleneck3d.res_f32), which BatchNorm ones have."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CFG = dict(type='GN', num_groups=8)


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


def st(t):
    return t.bfloat16().double()


def conv(m, x, rnd=True):
    """m's convolution and norm in 64 bits on the CPU from operands rounded to bf16, its own convolution's output not rounded"""
    y = torch.nn.functional.conv3d(st(x), st(m.conv.weight), None, m.conv.stride, m.conv.padding, m.conv.dilation)
    return torch.nn.functional.group_norm(y, m.gn.num_groups, m.gn.weight.double(), m.gn.bias.double(), m.gn.eps)


@pytest.mark.parametrize("down", [False, True])
def test_bottleneck_keeps_the_sum_in_f32(down):
    from trace_amd.resnet3d import Bottleneck3d, ConvModule
    torch.manual_seed(7)
    ds = ConvModule(128, 128, 1, bias=False, norm_cfg=CFG, act_cfg=None) if down else None
    blk = Bottleneck3d(128, 32, downsample=ds, norm_cfg=CFG).eval()
    x32 = torch.randn((2, 128, 2, 6, 6)) * 4
    with torch.no_grad():
        h = torch.relu(conv(blk.conv2, torch.relu(conv(blk.conv1, x32))))
        branch = conv(blk.conv3, h)
        want = torch.relu(branch + (conv(ds, x32) if down else x32.double()))
    blk.to(DEV)
    x = x32.permute(0, 2, 3, 4, 1).contiguous().to(DEV)
    xb = x.bfloat16()
    xb._res32 = x
    with torch.no_grad():
        blk.res_f32 = False
        assert not hasattr(blk.run(xb), "_res32")
        blk.res_f32 = True
        out = blk.run(xb)
    assert out.dtype == torch.bfloat16 and out._res32.dtype == torch.float32
    assert torch.equal(out._res32.bfloat16(), out)
    e32, e16 = (rel(t.permute(0, 4, 1, 2, 3), want) for t in (out._res32, out))
    # what is left are the roundings of h (twice, u / sqrt(3) each in the root mean square) on the way through the branch
    assert e32 < 2.0 ** -8 and e32 < e16, (e32, e16)


@pytest.mark.parametrize("main,side", [("GN", "BN"), ("BN", "GN")])
def test_bottleneck_of_both_norms(main, side):
    """a block whose downsample has the other norm: the f32 sum rounds to what the bf16 stream gives, but for that stream's roundings"""
    from trace_amd.resnet3d import Bottleneck3d, ConvModule
    torch.manual_seed(9)
    cfg = {"GN": CFG, "BN": dict(type='BN3d')}
    blk = Bottleneck3d(64, 32, downsample=ConvModule(64, 128, 1, bias=False, norm_cfg=cfg[side], act_cfg=None), norm_cfg=cfg[main]).eval().to(DEV)
    x = torch.randn((2, 2, 6, 6, 64), device=DEV).bfloat16()
    with torch.no_grad():
        plain = blk.run(x)
        blk.res_f32 = True
        out = blk.run(x)
    assert torch.equal(out._res32.bfloat16(), out)
    # the plain stream rounds both branches, the convolution under a GroupNorm and the sum: four roundings of u / sqrt(3) each
    assert rel(plain, out._res32) < 4 * 2.0 ** -8 / 3 ** 0.5


@pytest.mark.parametrize("mode", ["embedded_gaussian", "dot_product"])
@pytest.mark.parametrize("sub", [False, True])
def test_nonlocal_keeps_the_sum_in_f32(mode, sub):
    from trace_amd import ops
    from trace_amd.resnet3d import NonLocal3d
    torch.manual_seed(6)
    nl = NonLocal3d(128, sub_sample=sub, use_scale=True, mode=mode, norm_cfg=CFG).eval().to(DEV)
    heads, run_f32 = [], nl.conv_out.run_f32
    nl.conv_out.run_f32 = lambda h, *a: (heads.append(h), run_f32(h, *a))[1]
    with torch.no_grad():
        x32 = torch.randn((2, 2, 6, 6, 128), device=DEV) * 4
        x = x32.bfloat16()
        plain = nl.run(x)
        assert not hasattr(plain, "_res32") and not heads
        x._res32 = x32
        out = nl.run(x)
        assert torch.equal(out._res32.bfloat16(), out)
        c = ops.conv3d(heads[0], *nl.conv_out.packed(), (1, 1, 1), out_f32=True)
    # y in 64 bits from the convolution's own f32 output c: the norm's sums lose E of the magnitudes they add, the sum 2^-24 of itself
    u, E = 2.0 ** -8, 64 * 2.0 ** -24
    c = c.double().view(2, -1, 8, 16)
    red = (1, 3)
    mean = c.mean(red, keepdim=True)
    dev = c - mean
    rstd = (dev.square().mean(red, keepdim=True) + nl.conv_out.gn.eps).rsqrt()
    y = dev * rstd

    def moved(e):      # what an error of e |c| in every element of c does to y: through the element, the mean, the spread
        ec = e * c.abs()
        em = ec.mean(red, keepdim=True)
        return rstd * (ec + em) + y.abs() * (dev.abs() * (ec + em)).mean(red, keepdim=True) * rstd ** 2
    y, e32, e16 = (t.reshape(x.shape) for t in (y, moved(E), moved(u)))
    want = x32.double() + y
    assert bool(((out._res32.double() - want).abs() <= e32 + E * y.abs() + 2.0 ** -23 * want.abs()).all())
    # without the f32 stream: x, c, y and the sum are rounded
    plain = plain.double()
    assert bool(((plain - (x.double() + y)).abs() <= (e16 + u * y.abs() + u * plain.abs()) * 1.01 + 1e-5).all())


def test_stages_of_a_network():
    from trace_amd.resnet3d import ResNet3d, i3d_dc5_config
    cfg = i3d_dc5_config()
    cfg["norm_cfg"] = dict(type='GN', num_groups=32)
    cfg["non_local_cfg"] = dict(sub_sample=True, use_scale=True, norm_cfg=dict(type='GN', num_groups=32), mode='embedded_gaussian')
    torch.manual_seed(0)
    m = ResNet3d(**cfg)
    m.eval()
    clip = torch.randn((1, 3, 8, 64, 64)) * 50
    with torch.no_grad():
        want = m.forward_torch(clip).permute(0, 2, 3, 4, 1)
    m.to(DEV)
    with torch.no_grad():
        plain = m.forward_ndhwc(clip.to(DEV))
        m.res_f32_stages = (1, 2, 3)
        got = m.forward_ndhwc(clip.to(DEV))
        graphed = m.forward_ndhwc_graphed(clip.to(DEV))
    assert hasattr(got, "_res32") and torch.equal(got._res32.bfloat16(), got) and torch.equal(graphed, got)
    assert rel(got, want) < 5e-2 and rel(plain, want) < 5e-2       # 50 layers of bf16 operands against f32
