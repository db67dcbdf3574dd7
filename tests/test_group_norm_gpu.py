"""ops.group_norm_act / group_norm_act_backward / autograd.group_norm_act against the definition in 64 bits on the CPU.

Bounds per element, from first-order error propagation.  E = 64 x 2^-24 covers a sum: at most 16 pieces or GN_U rows in a row,
then trees of at most 9 + 8 + 8 levels and 128 chunks merged four at a time, all in 32 bits; u is half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = 2.0 ** -24
E = 64 * F
LEAKY = 0.1


def u_of(dt):
    return torch.finfo(dt).eps / 2


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "leaky":
        return torch.where(z > 0, z, LEAKY * z), torch.where(z > 0, 1.0, LEAKY).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def reference(x, dy, G, gamma, beta, eps, act):
    N, C = x.shape[0], x.shape[-1]
    dt = x.dtype
    u = u_of(dt)
    xs = x.double().reshape(N, -1, G, C // G)
    red = (1, 3)
    ga = torch.ones(C).double() if gamma is None else gamma.double()
    be = torch.zeros(C).double() if beta is None else beta.double()
    ga, be = ga.view(1, 1, G, -1), be.view(1, 1, G, -1)
    mean = xs.mean(red, keepdim=True)
    dev = xs - mean
    var = dev.square().mean(red, keepdim=True)
    rstd = (var + eps).rsqrt()
    # errors of mean, of 1 / sqrt(var + eps) (relative), of xh, of z
    em = E * xs.abs().mean(red, keepdim=True)
    ed = em + F * (xs.abs() + mean.abs())                       # of a deviation
    evar = 2 * E * var + (2 * dev.abs() * ed + ed * ed).mean(red, keepdim=True)
    er = 0.5 * evar / (var + eps) + 4 * F
    xh = dev * rstd
    exh = ed * rstd + xh.abs() * er
    z = xh * ga + be
    ez = exh * ga.abs() + 4 * F * ((xh * ga).abs() + be.abs())
    y, d1 = act64(z, act)
    # |silu'| <= 1.1, |silu''| <= 0.5; exp through exp2: relative 2^-21 + 2 |z| 2^-24 of a sigmoid
    eexp = 2.0 ** -20 * (1 + z.abs()) if act == "silu" else torch.zeros_like(z)
    ey = 1.1 * ez + z.abs() * eexp + u * y.abs()
    out = {"y": (y, ey)}
    if dy is not None:
        g = dy.double().reshape(xs.shape)
        dz = g * d1
        ed1 = {None: 0 * z, "silu": 0.5 * ez + (1 + z.abs()) * eexp,
               "relu": (z.abs() <= ez).double(), "leaky": (z.abs() <= ez).double()}[act]       # a kink inside the error: either side
        edz = g.abs() * ed1 + 4 * F * dz.abs()
        t, et = dz * ga, edz * ga.abs() + 2 * F * (dz * ga).abs()
        S1, S2 = t.mean(red, keepdim=True), (t * xh).mean(red, keepdim=True)
        eS1 = et.mean(red, keepdim=True) + E * t.abs().mean(red, keepdim=True)
        eS2 = (et * xh.abs() + t.abs() * exh).mean(red, keepdim=True) + E * (t * xh).abs().mean(red, keepdim=True)
        dx = rstd * (t - S1 - xh * S2)
        edx = rstd * (et + eS1 + xh.abs() * eS2 + exh * S2.abs() + 8 * F * (t.abs() + S1.abs() + (xh * S2).abs())) * (1 + er) + dx.abs() * (er + u)
        out["dx"] = (dx, edx)
        out["dbeta"] = (dz.sum((0, 1)), (edz + E * dz.abs()).sum((0, 1)))
        out["dgamma"] = ((dz * xh).sum((0, 1)), (edz * xh.abs() + dz.abs() * exh + E * (dz * xh).abs()).sum((0, 1)))
    return {k: (a.reshape(x.shape if k in ("y", "dx") else (C,)), (b * (1 + 1e-6)).reshape(x.shape if k in ("y", "dx") else (C,))) for k, (a, b) in out.items()}


def check(got, ref, name):
    val, bnd = ref
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), name
    bad = (got - val).abs() - bnd
    assert float(bad.max()) <= 1e-30, "%s: off by %.3g where %.3g is allowed" % (name, float((got - val).abs().flatten()[bad.argmax()]), float(bnd.flatten()[bad.argmax()]))


def run_case(shape, G, act, dt, affine=True, eps=1e-5, shift=1.0, scale=1.0, seed=0):
    from trace_amd import ops
    g = torch.Generator().manual_seed(seed + sum(shape) + G)
    C = shape[-1]
    x = ((torch.randn(shape, generator=g) * (0.3 + torch.rand(C, generator=g)) + shift * torch.randn(C, generator=g)) * scale).to(dt)
    dy = torch.randn(shape, generator=g).to(dt)
    gamma = 1 + 0.3 * torch.randn(C, generator=g) if affine else None
    beta = 0.3 * torch.randn(C, generator=g) if affine else None
    ref = reference(x, dy, G, gamma, beta, eps, act)
    xd, dyd = x.to(DEV), dy.to(DEV)
    gd, bd = (None, None) if gamma is None else (gamma.to(DEV), beta.to(DEV))
    y, st = ops.group_norm_act(xd, G, gd, bd, eps, act, return_stats=True)
    assert y.dtype == dt and y.shape == x.shape
    check(y, ref["y"], "y")
    dx, dg, db = ops.group_norm_act_backward(dyd, xd, st, G, gd, bd, act)
    check(dx, ref["dx"], "dx")
    check(db, ref["dbeta"], "dbeta")
    check(dg, ref["dgamma"], "dgamma")
    y2, st2 = ops.group_norm_act(xd, G, gd, bd, eps, act, return_stats=True)
    again = ops.group_norm_act_backward(dyd, xd, st2, G, gd, bd, act)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip((dx, dg, db), again))


# (P rows, C, G): one pass with 1 .. 16 pieces per thread, groups inside and across an access, two passes, one group, groups of one
SHAPES = [((2, 1, 8), 1), ((1, 2, 3, 32), 4), ((2, 49, 64), 8), ((3, 77, 60), 12), ((2, 100, 30), 6), ((2, 33, 7), 7), ((1, 31, 5), 1),
          ((2, 784, 256), 32), ((1, 900, 2048), 32), ((2, 2100, 64), 32), ((1, 4097, 32), 8), ((2, 3000, 60), 12), ((1, 5000, 24), 1),
          ((1, 700, 2056), 8), ((1, 300, 4104), 3), ((3, 2500, 9), 3), ((1, 1300, 257), 257), ((2, 260, 264), 1), ((17, 64, 16), 2),
          ((1, 40, 8192), 1), ((1, 20000, 1), 1), ((1, 6, 5, 4, 48), 3)]


@pytest.mark.parametrize("shape,G", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_shapes(shape, G, dt):
    run_case(shape, G, None, dt)


@pytest.mark.parametrize("act", ["relu", "leaky", "silu"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,G", [((2, 100, 64), 8), ((2, 3000, 64), 8), ((1, 2600, 30), 5)])
def test_activations(act, dt, shape, G):
    run_case(shape, G, act, dt)


@pytest.mark.parametrize("shape,G", [((2, 200, 64), 8), ((1, 3000, 64), 8)])
def test_far_mean_no_affine_and_eps(shape, G):
    run_case(shape, G, None, torch.float32, shift=3000.0)          # mean far outside the spread
    run_case(shape, G, "silu", torch.bfloat16, affine=False)
    run_case(shape, G, None, torch.float32, eps=0.1, scale=1e-3)   # eps dominates


def test_constant_map_and_nan():
    from trace_amd import ops
    x = torch.full((2, 50, 16), 3.0, device=DEV)
    y, st = ops.group_norm_act(x, 2, None, torch.arange(16.0, device=DEV), return_stats=True)
    assert torch.equal(y, torch.arange(16.0, device=DEV).expand_as(y))
    x[1, 7, 3] = float("nan")
    y = ops.group_norm_act(x, 2, act="relu")
    assert not y[0].isnan().any() and y[1, :, :8].isnan().all() and not y[1, :, 8:].isnan().any()


def test_views_other_memory_and_empty():
    from trace_amd import ops
    g = torch.Generator().manual_seed(0)
    x = torch.randn((2, 10, 12, 24), generator=g).to(DEV).bfloat16()
    want = ops.group_norm_act(x, 3)
    assert torch.equal(ops.group_norm_act(x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), 3), want)     # channels first in memory
    wide = torch.zeros((2, 10, 12, 25), device=DEV, dtype=torch.bfloat16)
    wide[..., 1:] = x
    assert torch.equal(ops.group_norm_act(wide[..., 1:], 3), want)
    e = torch.zeros((0, 5, 8), device=DEV)
    y, st = ops.group_norm_act(e, 2, return_stats=True)
    dx, dg, db = ops.group_norm_act_backward(e, e, st, 2)
    assert y.shape == e.shape and dx.shape == e.shape and not dg.any() and not db.any()
    e = torch.zeros((2, 0, 8), device=DEV)
    assert ops.group_norm_act(e, 2).shape == e.shape


def test_autograd_differences_and_partial_needs():
    from trace_amd import autograd as tag
    g = torch.Generator().manual_seed(3)
    x, r = torch.randn((2, 40, 24), generator=g), torch.randn((2, 40, 24), generator=g)
    ga, be = 1 + 0.2 * torch.randn(24, generator=g), 0.2 * torch.randn(24, generator=g)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, ga, be)]
    tag.group_norm_act(leaves[0], 4, leaves[1], leaves[2], 1e-5, "silu").backward(r.to(DEV))

    def loss(x, ga, be):
        return float((torch.nn.functional.silu(torch.nn.functional.group_norm(x.transpose(1, 2), 4, ga, be, 1e-5)).transpose(1, 2) * r.double()).sum())
    base = [t.double() for t in (x, ga, be)]
    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=g).double()
        hi, lo = ([t + (s * 1e-5 * d if j == i else 0) for j, t in enumerate(base)] for s in (1, -1))
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        got = leaf.grad.double().cpu()
        assert abs(float((got * d).sum()) - diff) <= 2.0 ** -18 * float((got.abs() * d.abs()).sum()) + 1e-6
    b2 = be.to(DEV).requires_grad_(True)
    y = tag.group_norm_act(x.to(DEV), 4, ga.to(DEV), b2, 1e-5, "silu")
    (gb,) = torch.autograd.grad(y, b2, r.to(DEV))
    assert torch.equal(gb, leaves[2].grad)


def test_graph_replays():
    from trace_amd import autograd as tag, ops
    for shape, G in (((2, 100, 64), 8), ((2, 3000, 64), 8)):
        x = torch.randn(shape, device=DEV)
        dy = torch.randn(shape, device=DEV)
        ga = torch.ones(shape[-1], device=DEV)

        def step():
            a, w = x.detach().requires_grad_(True), ga.detach().requires_grad_(True)
            y = tag.group_norm_act(a, G, w, None, 1e-5, "silu")
            return (y.detach(),) + torch.autograd.grad(y, (a, w), dy)
        step()
        gr = torch.cuda.CUDAGraph()
        with ops.capture(gr):
            res = step()
        for rep in range(3):
            x.normal_()
            want = step()
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want)), rep


def test_conv_module_with_group_norm():
    """ConvModule(norm_cfg GN): run and run_train against nn.Conv3d + nn.GroupNorm in f32 on the CPU, as the batch-norm tests do"""
    from trace_amd.resnet3d import Bottleneck3d, ConvModule, NonLocal3d
    torch.manual_seed(5)
    cfg = dict(type='GN', num_groups=8)
    ds = ConvModule(64, 128, 1, bias=False, norm_cfg=cfg, act_cfg=None)
    blk = Bottleneck3d(64, 32, downsample=ds, norm_cfg=cfg)
    assert blk.conv1.norm is blk.conv1.gn and not hasattr(blk.conv1, "bn")
    x = torch.randn((2, 64, 3, 8, 8))
    xr = x.bfloat16().float().requires_grad_(True)

    def st(t):
        return t + (t.bfloat16().float() - t).detach()

    def ref_conv(m, t, relu):
        y = st(torch.nn.functional.conv3d(t, st(m.conv.weight), None, m.conv.stride, m.conv.padding, m.conv.dilation))
        y = m.gn(y)
        return st(torch.relu(y) if relu else y)
    out = torch.relu(st(ref_conv(blk.conv3, ref_conv(blk.conv2, ref_conv(blk.conv1, xr, True), True), False) + ref_conv(ds, xr, False)))
    r = torch.randn(out.shape).bfloat16().float()
    (out * r).sum().backward()
    ref = {n: p.grad.clone() for n, p in blk.named_parameters()}
    blk.zero_grad()
    blk.to(DEV)
    xh = x.bfloat16().permute(0, 2, 3, 4, 1).contiguous().to(DEV).requires_grad_(True)

    def rel(a, b):
        a, b = a.detach().float().cpu(), b.detach().float().cpu()
        return float((a - b).norm() / b.norm())
    with torch.no_grad():
        assert rel(blk.run(xh.detach()).permute(0, 4, 1, 2, 3), out) < 2e-2
    got = blk.run_train(xh)
    assert rel(got.permute(0, 4, 1, 2, 3), out) < 2e-2
    (got.float() * r.permute(0, 2, 3, 4, 1).to(DEV)).sum().backward()
    assert rel(xh.grad.permute(0, 4, 1, 2, 3), xr.grad) < 3e-2
    for n, p in blk.named_parameters():
        assert rel(p.grad, ref[n]) < 3e-2, n
    frozen = ConvModule(8, 16, 1, norm_cfg=dict(type='GN', num_groups=4, eps=1e-3, requires_grad=False))
    assert frozen.gn.eps == 1e-3 and not frozen.gn.weight.requires_grad


def test_resnet3d_and_nonlocal_with_group_norm_and_softmax_attention():
    """the operators together, as a user trains the clip backbone without batch statistics and with softmax non-local blocks:
    inference path against the module's own torch path in f32, then a training step that reaches every parameter"""
    from trace_amd.resnet3d import ResNet3d, i3d_dc5_config
    cfg = i3d_dc5_config()
    cfg["norm_cfg"] = dict(type='GN', num_groups=32)
    cfg["non_local_cfg"] = dict(sub_sample=True, use_scale=True, norm_cfg=dict(type='GN', num_groups=32), mode='embedded_gaussian')
    torch.manual_seed(0)
    m = ResNet3d(**cfg)
    m.eval()
    clip = torch.randn((2, 3, 8, 64, 64)) * 50
    with torch.no_grad():
        want = m.forward_torch(clip).permute(0, 2, 3, 4, 1)
    m.to(DEV)
    with torch.no_grad():
        got = m.forward_ndhwc(clip.to(DEV)).float().cpu()
    err = float((got - want).norm() / want.norm())
    assert got.shape == want.shape and err < 5e-2, err      # 50 layers of bf16 operands against f32
    m.train()
    out = m.forward_train(clip.to(DEV))
    assert float((out.detach().float().cpu() - want).norm() / want.norm()) < 5e-2
    out.float().square().mean().backward()
    for n, p in m.named_parameters():
        if n.startswith("conv1."):
            assert p.grad is None, n
        else:
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n


@pytest.mark.parametrize("sub", [False, True])
@pytest.mark.parametrize("use_scale", [False, True])
def test_nonlocal_embedded_gaussian(sub, use_scale):
    from trace_amd.resnet3d import NonLocal3d
    torch.manual_seed(2)
    nl = NonLocal3d(128, sub_sample=sub, use_scale=use_scale, mode='embedded_gaussian', norm_cfg=dict(type='BN3d'))
    with torch.no_grad():
        bn = nl.conv_out.bn
        bn.weight.uniform_(0.5, 1.5)
        bn.bias.normal_(0, 0.1)
        bn.running_mean.normal_(0, 0.1)
        bn.running_var.uniform_(0.5, 1.5)
    nl.eval()
    x = torch.randn((2, 128, 2, 6, 6)) * 2
    xr = x.bfloat16().float().requires_grad_(True)

    # the reference rounds what the path stores (weights and activations, straight-through): unscaled scores of ten units turn
    # an unmatched rounding of theta and phi, 2^-9 relative, into percents of a probability, which says nothing about the kernels
    def st(t):
        return t + (t.bfloat16().float() - t).detach()

    def conv(m, t):
        w = m.conv.weight
        b = m.conv.bias
        if m.with_norm:
            sc = m.bn.weight / torch.sqrt(m.bn.running_var + m.bn.eps)
            w, b = w * sc.view(-1, 1, 1, 1, 1), m.bn.bias - m.bn.running_mean * sc
        return st(torch.nn.functional.conv3d(t, st(w), b))
    pool = (lambda t: torch.nn.functional.max_pool3d(t, (1, 2, 2))) if sub else (lambda t: t)
    th, ph, gg = (f(conv(nl._conv(m), xr)).flatten(2) for m, f in ((nl.theta, lambda t: t), (nl.phi, pool), (nl.g, pool)))
    att = torch.softmax(th.transpose(1, 2) @ ph * (64 ** -0.5 if use_scale else 1.0), -1) @ gg.transpose(1, 2)
    out = xr + conv(nl.conv_out, st(att).transpose(1, 2).reshape(2, 64, 2, 6, 6))
    with torch.no_grad():       # the module's own torch path computes the same function
        own = float((nl(xr) - out).norm() / out.norm())
    assert own < 2e-2
    r = torch.randn(out.shape).bfloat16().float()
    (out * r).sum().backward()
    ref = {n: p.grad.clone() for n, p in nl.named_parameters()}
    nl.zero_grad()
    nl.to(DEV)

    def rel(a, b):
        a, b = a.detach().float().cpu(), b.detach().float().cpu()
        return float((a - b).norm() / b.norm().clamp_min(1e-6))
    xh = x.bfloat16().permute(0, 2, 3, 4, 1).contiguous().to(DEV).requires_grad_(True)
    with torch.no_grad():
        e_run = rel(nl.run(xh.detach()).permute(0, 4, 1, 2, 3), out)
    got = nl.run_train(xh)
    e_train = rel(got.permute(0, 4, 1, 2, 3), out)
    (got.float() * r.permute(0, 2, 3, 4, 1).to(DEV)).sum().backward()
    e_x = rel(xh.grad.permute(0, 4, 1, 2, 3), xr.grad)
    assert max(e_run, e_train, e_x) < 2e-2, (e_run, e_train, e_x)
    for n, p in nl.named_parameters():
        if n == "phi.conv.bias" or n == "phi.0.conv.bias":
            continue       # shifts every score of a row alike: its gradient is zero but for rounding
        # pooled phi / g: near-ties of the max-pool move whole entries, as in the dot_product test
        assert rel(p.grad, ref[n]) < (5e-2 if n.startswith(("phi.", "g.", "theta.")) else 2e-2), (n, rel(p.grad, ref[n]))


def test_nonlocal_embedded_gaussian_keeps_the_f32_residual_stream():
    from trace_amd.resnet3d import NonLocal3d
    torch.manual_seed(6)
    nl = NonLocal3d(128, sub_sample=True, use_scale=True, mode='embedded_gaussian', norm_cfg=dict(type='BN3d')).eval().to(DEV)
    with torch.no_grad():
        nl.conv_out.bn.weight.fill_(1.0)
        x32 = torch.randn((2, 2, 6, 6, 128), device=DEV) * 4
        x = x32.bfloat16()
        plain = nl.run(x)
        assert not hasattr(plain, "_res32")
        x._res32 = x32
        out = nl.run(x)
        assert out.dtype == torch.bfloat16 and torch.equal(out._res32.bfloat16(), out)
        # plain is x + y rounded to bf16, out x32 + y; x itself is half a bf16 step from x32
        step = 2.0 ** -8 * (plain.float().abs() + x32.abs()) + 1e-5
        assert bool(((out._res32 - x32) - (plain.float() - x.float())).abs().le(step).all())


def test_refusals():
    from trace_amd import ops
    x = torch.zeros((2, 10, 16), device=DEV)
    ga = torch.ones(16, device=DEV)
    for args, kw in (((x, 3), {}), ((x, 0), {}), ((x.half(), 2), {}), ((x.cpu(), 2), {}), ((x, 2, ga[:8]), {}), ((x, 2, ga.cpu()), {}),
                     ((x, 2), dict(act="gelu")), ((x, 2), dict(eps=-1.0)), ((x, 2), dict(eps=float("nan"))), ((x[0, 0], 2), {}),
                     ((torch.zeros((1, 2, 8200), device=DEV), 1), {})):
        with pytest.raises(RuntimeError):
            ops.group_norm_act(*args, **kw)
    y, st = ops.group_norm_act(x, 2, return_stats=True)
    for args in ((x[:1], x, st, 2), (x.bfloat16(), x, st, 2), (x, x, st[:1], 2), (x, x, st.double(), 2), (x, x, st, 4)):
        with pytest.raises(RuntimeError):
            ops.group_norm_act_backward(*args)


def test_offsets_past_32_bits():
    """2^31 + elements; the last sample by itself gives the same bits"""
    from trace_amd import ops
    x = torch.empty((3, 2800001, 256), dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 1 << 31
    x.normal_()
    x[2] += 3
    y, st = ops.group_norm_act(x, 32, act="silu", return_stats=True)
    assert abs(float(st[2, :, 0].mean()) - 3) < 1e-2 and abs(float(st[0, :, 0].mean())) < 1e-2
    tail = x[2, -4:].float()
    z = (tail - st[2, :, 0].repeat_interleave(8)) * st[2, :, 1].repeat_interleave(8)
    want = z * torch.sigmoid(z)
    assert float((y[2, -4:].float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1e-5
    del y
    dx, dg, db = ops.group_norm_act_backward(x, x, st, 32)
    # dy = x: dbeta = sum of x, dgamma = sum of x xh; xh has mean 0 and variance 1 over a group, so dx is near 0
    assert float(dx[2, -1000:].float().abs().max()) < 0.1
    n = x.shape[1]
    assert abs(float(db.mean()) / n - 3) < 0.05
