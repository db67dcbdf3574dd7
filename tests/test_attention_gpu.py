"""ops.attention / ops.attention_backward / autograd.attention against the definition in 64 bits on the CPU.

Tolerances are bounds per element, from the roundings the kernels make (u = eps / 2 of bf16 = 2^-8, relative):
  out   u |out|  (the result)  +  u sum_j P_j |v_j|  (P is rounded to bf16 for the product)
  dv    u |dv| + u sum_i P_ij |dout_i|
  dS    u |dS|  (rounded for the product)  +  P_ij e_i,  e_i = sum_d |dout_id| 2 u^2 (|out_id| + sum_j P_j |v_jd|): delta is formed
        from out + rest, each rounding of which leaves u of what the first one left
  dq    u |dq| + scale sum_j (bound of dS)_ij |k_j|;  dk likewise over i
and what 32-bit sums lose: a score is off by (D + 2) 2^-24 sum_d |q_d k_d| scale, its exponential by that, by the rounding of
lse (2^-23 |lse|) and by the hardware's exp2 (2^-20 taken), relative to P; dP by (D + 2) 2^-24 sum_d |dout_d v_d|; sums over
n rows by n 2^-24 of the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = torch.finfo(torch.bfloat16).eps / 2
F = 2.0 ** -24


def lens(mode, B, Nq, Nk, which):
    """[(q_len, kv_len)] of a padded batch; entry 1 has no keys, entry 2 no queries."""
    out = []
    for b in range(B):
        lq, lk = Nq, Nk
        if mode != "none":
            lk = 0 if b == 1 else max(1, Nk - (b * Nk) // B)
        if mode == "both":
            lq = 0 if b == 2 else max(1, Nq - (b * Nq * 2) // (3 * B))
        out.append((lq, lk))
    return out


def reference(q, k, v, do, scale, causal, ln):
    """f64 results and bounds: dict name -> (value, bound); rows nothing is defined for are zero with bound 0."""
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1:3]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    res = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64))
           for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape))}
    lse_all = torch.full((B, H, Nq), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros((B, H, Nq), dtype=torch.float64)
    for b in range(B):
        lq, lk = ln[b]
        for h in range(H):
            hk = h // (H // Hk)
            qq, kk, vv, dd = q[b, :lq, h], k[b, :lk, hk], v[b, :lk, hk], do[b, :lq, h]
            if lq == 0 or lk == 0:
                continue
            s = qq @ kk.t() * scale
            if causal:
                s = s.masked_fill(torch.ones(lq, lk).triu(lk - lq + 1).bool(), -math.inf)
            live = (s > -math.inf).any(1)
            lse = torch.logsumexp(s, 1)
            P = torch.where(live[:, None], torch.exp(s - torch.where(live, lse, torch.zeros_like(lse))[:, None]), torch.zeros_like(s))
            s_err = (D + 2) * F * scale * (qq.abs() @ kk.abs().t())
            l_abs = torch.where(live, lse, torch.zeros_like(lse)).abs()
            # relative error of a recomputed / normalised probability; in the forward the maximum is scaled once more (2^-23)
            p_rel = 2 * s_err.max(1).values + 2 ** -20 + (l_abs + s.masked_fill(s == -math.inf, 0).abs().max(1).values) * 2 ** -22 + lk * F
            o = P @ vv
            A = P @ vv.abs()
            e_o = U * o.abs() + (U + p_rel[:, None] + lk * F) * A * (1 + U)
            res["out"][0][b, :lq, h], res["out"][1][b, :lq, h] = o, e_o
            lse_all[b, h, :lq] = lse
            lse_bound[b, h, :lq] = torch.where(live, p_rel + l_abs * 2 ** -22 + 1e-6, torch.zeros_like(lse))
            dp = dd @ vv.t()
            delta = (dd * o).sum(1, keepdim=True)
            ds = P * (dp - delta)
            e_fine = 2 * U * U * (o.abs() + A) + (p_rel[:, None] + lk * F) * A
            e_ds = P * ((dd.abs() * e_fine).sum(1, keepdim=True) + (D + 2) * F * (dd.abs() @ vv.abs().t() + (dd.abs() * o.abs()).sum(1, keepdim=True)))
            e_ds = e_ds + (p_rel[:, None] + U) * (ds.abs() + e_ds)
            e_p = (p_rel[:, None] + U) * P
            dq = scale * ds @ kk
            res["dq"][0][b, :lq, h] = dq
            res["dq"][1][b, :lq, h] = U * dq.abs() + scale * (1 + U) * (e_ds + lk * F * ds.abs()) @ kk.abs()
            res["dk"][0][b, :lk, hk] += scale * ds.t() @ qq
            res["dk"][1][b, :lk, hk] += scale * (1 + U) * (e_ds + lq * F * ds.abs()).t() @ qq.abs()
            res["dv"][0][b, :lk, hk] += P.t() @ dd
            res["dv"][1][b, :lk, hk] += (1 + U) * (e_p + lq * F * P).t() @ dd.abs()
    for n in ("dk", "dv"):
        val, bnd = res[n]
        res[n] = (val, bnd + U * val.abs())
    return res, lse_all, lse_bound


def check(got, ref, name):
    val, bnd = ref
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), "%s: not finite" % name
    worst = float(((got - val).abs() - bnd).max())
    if worst > 1e-12:
        r = (got - val).abs() / bnd.clamp_min(1e-30)
        raise AssertionError("%s: %.3g times its bound, off by %.3g" % (name, float(r.max()), float((got - val).abs().max())))


def make(B, Nq, Nk, H, Hk, D, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((B, Nq, H, D), generator=g) * spread).bfloat16()
    k = (torch.randn((B, Nk, Hk, D), generator=g) * spread).bfloat16()
    v = torch.randn((B, Nk, Hk, D), generator=g).bfloat16()
    do = torch.randn((B, Nq, H, D), generator=g).bfloat16()
    return q, k, v, do


def run_case(B, Nq, Nk, H, Hk, D, causal, mode, scale=None, spread=1.0, seed=0, q_view=None):
    from trace_amd import ops
    q, k, v, do = make(B, Nq, Nk, H, Hk, D, seed + B + Nq + Nk + D, spread)
    ln = lens(mode, B, Nq, Nk, None)
    ref, lse_ref, lse_bnd = reference(q, k, v, do, D ** -0.5 if scale is None else scale, causal, ln)
    # nothing behind a length may be read
    for b, (lq, lk) in enumerate(ln):
        q[b, lq:], do[b, lq:] = math.nan, math.inf
        k[b, lk:], v[b, lk:] = math.nan, math.inf
    q, k, v, do = (t.to(DEV) for t in (q, k, v, do))
    kw = dict(scale=scale, causal=causal)
    if mode == "both":
        kw["q_len"] = torch.tensor([a for a, _ in ln], dtype=torch.int32, device=DEV)
    if mode != "none":
        kw["kv_len"] = torch.tensor([b for _, b in ln], dtype=torch.int32, device=DEV)
    out, lse, rest = ops.attention(q, k, v, for_backward=True, **kw)
    check(out, ref["out"], "out")
    dead = lse_ref == -math.inf
    lse_c = lse.double().cpu()
    assert torch.equal(lse_c == -math.inf, dead)
    assert float(((lse_c - lse_ref).abs() - lse_bnd)[~dead].max() if (~dead).any() else 0.0) <= 0.0
    dq, dk, dv = ops.attention_backward(do, q, k, v, out, lse, rest, **kw)
    check(dv, ref["dv"], "dv")
    check(dq, ref["dq"], "dq")
    check(dk, ref["dk"], "dk")
    # the forward pass alone: one product, its probabilities rounded
    plain, plain_lse = ops.attention(q, k, v, return_lse=True, **kw)
    check(plain, ref["out"], "out alone")
    assert torch.equal(plain_lse, lse)
    # equal calls, equal bits
    out2, lse2, rest2 = ops.attention(q, k, v, for_backward=True, **kw)
    again = ops.attention_backward(do, q, k, v, out2, lse2, rest2, **kw)
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip((dq, dk, dv), again))


@pytest.mark.parametrize("D", [8, 24, 64, 72, 128, 200, 256, 264, 512])
@pytest.mark.parametrize("causal", [False, True])
def test_head_sizes(D, causal):
    run_case(2, 77, 93, 2, 1, D, causal, "none")


@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 2), (2, 1), (1, 31), (1, 513), (15, 16), (16, 17), (17, 15), (33, 64), (64, 65),
                                   (128, 32), (129, 200), (300, 7), (257, 257)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(Nq, Nk, causal):
    run_case(1, Nq, Nk, 4, 2, 64, causal, "none")


@pytest.mark.parametrize("D", [40, 128, 256, 512])
@pytest.mark.parametrize("mode", ["keys", "both"])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batches(D, mode, causal):
    run_case(5, 70, 100, 2, 2, D, causal, mode)
    run_case(4, 100, 37, 2, 1, D, causal, mode)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (8, 2), (12, 4), (16, 16)])
@pytest.mark.parametrize("Nq", [1, 2, 50])
def test_shared_heads(H, Hk, Nq):
    run_case(3, Nq, 130, H, Hk, 64, False, "keys")
    run_case(3, Nq, 130, H, Hk, 128, True, "both")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_split_keys(D):
    """few rows over many keys: the keys are split over workgroups and joined; lengths leave whole splits empty"""
    run_case(3, 1, 4000, 4, 2, D, False, "keys")
    run_case(1, 40, 3000, 1, 1, D, True, "none")
    run_case(1, 1500, 33, 1, 1, D, False, "none")      # dk / dv split over the queries


@pytest.mark.parametrize("D,causal", [(24, False), (64, True), (128, False), (128, True), (256, False), (512, False), (512, True)])
def test_grids_that_fill_the_card(D, causal):
    """so many heads that whole tiles of rows are taken (the other tests' calls get half tiles)"""
    run_case(26, 130, 140, 10, 10, D, causal, "both")


def test_grids_that_fill_the_card_by_rows_or_by_splits():
    run_case(35, 130, 140, 8, 4, 128, False, "none")
    run_case(11, 120, 130, 6, 6, 512, False, "both")
    run_case(1, 200, 4500, 2, 2, 512, False, "keys")
    run_case(1, 100, 9000, 2, 1, 128, False, "none")    # long shares: whole tiles in splits
    run_case(1, 100, 9000, 1, 1, 128, True, "keys")


@pytest.mark.parametrize("spread,scale", [(6.0, None), (1.0, 3.0), (0.01, None), (1.0, 1e-6)])
def test_peaked_and_flat_rows(spread, scale):
    run_case(2, 65, 140, 2, 2, 64, False, "none", scale=scale, spread=spread)


@pytest.mark.parametrize("D", [8, 16, 32])
def test_dq_of_few_columns(D):
    """dq carries no more than its own rounding: at most u |dq| each, so u / sqrt(3) in the root mean square if spread evenly (a
    rounded dS would add as much again, and more the fewer the columns, because its rows sum to zero)"""
    from trace_amd import ops
    q, k, v, do = make(2, 300, 400, 4, 2, D, 21)
    ref, _, _ = reference(q, k, v, do, D ** -0.5, False, [(300, 400)] * 2)
    q, k, v, do = (t.to(DEV) for t in (q, k, v, do))
    dq, _, _ = ops.attention_backward(do, q, k, v, *ops.attention(q, k, v, for_backward=True))
    want = ref["dq"][0]
    assert float((dq.double().cpu() - want).norm() / want.norm()) < U / 3 ** 0.5


def test_no_keys_no_rows():
    from trace_amd import ops
    q, k, v, do = (t.to(DEV) for t in make(2, 5, 0, 2, 1, 64, 3))
    out, lse, rest = ops.attention(q, k, v, for_backward=True)
    assert not out.any() and not rest.any() and (lse == -math.inf).all()
    dq, dk, dv = ops.attention_backward(do, q, k, v, out, lse, rest)
    assert not dq.any() and dk.shape == k.shape and dv.shape == v.shape
    q, k, v, do = (t.to(DEV) for t in make(2, 0, 5, 2, 1, 64, 3))
    out, lse, rest = ops.attention(q, k, v, for_backward=True)
    assert out.shape == q.shape and lse.shape == (2, 2, 0)
    dq, dk, dv = ops.attention_backward(do, q, k, v, out, lse, rest)
    assert not dk.any() and not dv.any()
    q, k, v, do = (t.to(DEV) for t in make(0, 4, 5, 2, 1, 64, 3))
    assert ops.attention(q, k, v).shape == (0, 4, 2, 64)


@pytest.mark.parametrize("Nq,Nk", [(5, 0), (0, 5)])
def test_empty_views(Nq, Nk):
    """operands without elements, cut out of memory whose strides the kernels do not take"""
    from trace_amd import ops
    q, k, v, do = (torch.ones((2, n, h, 68), dtype=torch.bfloat16, device=DEV)[..., :64] for n, h in ((Nq, 2), (Nk, 1), (Nk, 1), (Nq, 2)))
    out, lse, rest = ops.attention(q, k, v, for_backward=True)
    assert out.shape == (2, Nq, 2, 64) and not out.any()
    for t, g in zip((q, k, v), ops.attention_backward(do, q, k, v, out, lse, rest)):
        assert g.shape == t.shape and not g.any()


def test_lengths_are_clamped():
    from trace_amd import ops
    q, k, v, _ = (t.to(DEV) for t in make(2, 9, 20, 2, 2, 64, 5))
    n = torch.tensor([-3, 1 << 30], dtype=torch.int32, device=DEV)
    out = ops.attention(q, k, v, kv_len=n)
    assert not out[0].any() and torch.equal(out[1], ops.attention(q[1:], k[1:], v[1:])[0])


def test_strided_and_broadcast_operands():
    from trace_amd import autograd as tag, ops
    g = torch.Generator().manual_seed(1)
    B, N, H, D = 2, 45, 3, 64
    qkv = torch.randn((B, N, 3, H, D), generator=g).bfloat16().to(DEV)
    q, k, v = qkv.unbind(2)
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(ops.attention(q, k, v), want)                                          # views of a packed projection
    hm = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]          # head-major memory
    assert torch.equal(ops.attention(*hm), want)
    odd = torch.randn((B, N, H, D + 4), generator=g).bfloat16().to(DEV)                       # rows that are not 16-byte aligned
    odd[..., 4:] = q
    assert torch.equal(ops.attention(odd[..., 4:], k, v), want)
    last = q.transpose(2, 3).contiguous().transpose(2, 3)                                     # last dimension not contiguous
    assert torch.equal(ops.attention(last, k, v), want)
    k1 = k[:1].expand(B, N, H, D)
    assert torch.equal(ops.attention(q, k1, v), ops.attention(q, k1.contiguous(), v))         # broadcast over the batch
    # gradient of a broadcast input, and an output gradient that is itself broadcast
    base = k[:1].detach().clone().requires_grad_(True)
    out = tag.attention(q, base.expand(B, N, H, D), v)
    (gb,) = torch.autograd.grad(out.float().sum(), base)
    kk = k1.detach().contiguous().requires_grad_(True)
    (gk,) = torch.autograd.grad(tag.attention(q, kk, v).float().sum(), kk)
    assert torch.equal(gb, gk.sum(0, keepdim=True))


def test_autograd_only_where_needed_and_differences():
    """gradients against differences of the 64-bit loss along random directions"""
    from trace_amd import autograd as tag
    B, Nq, Nk, H, D = 1, 24, 40, 2, 32
    q, k, v, r = make(B, Nq, Nk, H, H, D, 9)
    lq, lk, lv = (t.to(DEV).requires_grad_(True) for t in (q, k, v))
    out = tag.attention(lq, lk, lv, causal=True)
    out.backward(r.to(DEV))

    def loss(q, k, v):
        s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
        s = s.masked_fill(torch.ones(Nq, Nk).triu(Nk - Nq + 1).bool(), -math.inf)
        return float((torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v) * r.double()).sum())
    ops64 = [t.double() for t in (q, k, v)]
    for n, (leaf, i) in enumerate(zip((lq, lk, lv), range(3))):
        d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(n)).double()
        eps = 1e-4
        hi, lo = ([t + (s * eps * d if j == i else 0) for j, t in enumerate(ops64)] for s in (1, -1))
        diff = (loss(*hi) - loss(*lo)) / (2 * eps)
        got = leaf.grad.double().cpu()
        # three bf16 roundings (P or dS, out in delta, the result), each at most u of the terms summed
        assert abs(float((got * d).sum()) - diff) <= 3 * U * float((got.abs() * d.abs()).sum()) + 1e-3
    vv = v.to(DEV).requires_grad_(True)
    (gv,) = torch.autograd.grad(tag.attention(q.to(DEV), k.to(DEV), vv, causal=True), vv, r.to(DEV))
    assert torch.equal(gv, lv.grad)


def test_second_derivatives_are_refused():
    """a recorded backward pass gives the same gradients, and an error only where it is differentiated itself"""
    from trace_amd import autograd as tag
    q, k, v, do = (t.to(DEV) for t in make(1, 20, 30, 2, 2, 32, 4))
    w = torch.ones(32, device=DEV)
    for f in (lambda x: tag.attention(x, k, v), lambda x: tag.group_norm_act(x, 8, w, None, 1e-5, "silu"),
              lambda x: tag.dropout_act(x, 0.5, 1, 2, "leaky")):
        x = q.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(f(x), x, do)
        g = do.clone().requires_grad_(True)
        (got,) = torch.autograd.grad(f(x), x, g, create_graph=True)
        assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
        with pytest.raises(RuntimeError, match="differentiate twice"):
            got.float().sum().backward()


def test_graph_replays_and_streams():
    from trace_amd import autograd as tag, ops
    q, k, v, do = (t.to(DEV) for t in make(2, 100, 600, 2, 2, 64, 11))
    n = torch.tensor([600, 17], dtype=torch.int32, device=DEV)

    def step():
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = tag.attention(a, b, c, kv_len=n)
        return (out.detach(),) + torch.autograd.grad(out, (a, b, c), do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, step()))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with ops.capture(g):
            res = step()
        graphs.append((g, res))
    for rep in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        n.copy_(torch.tensor([600 - rep, rep], dtype=torch.int32))
        want = step()
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), rep


def test_refusals():
    from trace_amd import ops
    q, k, v, do = (t.to(DEV) for t in make(2, 5, 7, 4, 2, 64, 1))
    for args in ((q.float(), k, v), (q[0], k, v), (q, k[:, :6], v), (q[..., :60], k[..., :60], v[..., :60]), (q[:, :, :3], k, v),
                 (q, k[:1], v[:1]), (q.cpu(), k, v)):
        with pytest.raises(RuntimeError):
            ops.attention(*args)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(kv_len=torch.tensor([1, 2])),
               dict(kv_len=torch.tensor([1], dtype=torch.int32, device=DEV)), dict(q_len=torch.tensor([1, 2], device=DEV))):
        with pytest.raises(RuntimeError):
            ops.attention(q, k, v, **kw)
    big = torch.zeros((1, 4, 1, 520), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        ops.attention(big, big, big)
    out, lse, rest = ops.attention(q, k, v, for_backward=True)
    for args in ((do[:, :4], q, k, v, out, lse, rest), (do, q, k, v, out[:, :4], lse, rest), (do, q, k, v, out, lse[:, :2], rest),
                 (do, q, k, v, out.float(), lse, rest), (do, q, k, v, out, lse.double(), rest), (do, q, k, v, out, lse, rest[:1])):
        with pytest.raises(RuntimeError):
            ops.attention_backward(*args)


@pytest.mark.parametrize("Nq,Nk", [(1, 40), (1, 3000), (100, 60), (20, 3000)])
def test_nan_is_not_hidden(Nq, Nk):
    """a NaN that a row sees reaches its output and its lse, also where the keys are split; other rows do not notice"""
    from trace_amd import ops
    q, k, v, do = (t.to(DEV) for t in make(2, Nq, Nk, 2, 2, 64, 21))
    q[0, Nq // 2, 1] = math.nan
    for kw in (dict(return_lse=True), dict(for_backward=True)):
        out, lse = ops.attention(q, k, v, **kw)[:2]
        bad = torch.zeros((2, 2, Nq), dtype=torch.bool, device=DEV)
        bad[0, 1, Nq // 2] = True
        assert torch.equal(lse.isnan(), bad) and torch.equal(out.isnan().all(-1).transpose(1, 2), bad)
        assert torch.equal(out.isnan().any(-1).transpose(1, 2), bad)
    q[0, Nq // 2, 1] = 0
    k[1, Nk - 1, 0, 3] = math.nan
    out = ops.attention(q, k, v)
    assert out[1, :, 0].isnan().all() and not out[0].isnan().any() and not out[1, :, 1].isnan().any()
    # rows that a causal mask keeps from the key
    out, lse, rest = ops.attention(q, k, v, causal=True, for_backward=True)
    assert out[1, Nq - 1, 0].isnan().all() and not lse[1, 0, :Nq - 1].isnan().any()


def test_offsets_past_32_bits():
    """a cache of 2^31 + elements: the key that decides is its last one, in the last head and in the first"""
    from trace_amd import ops
    Nk, Hk, D = (1 << 20) + 37, 16, 128
    k = torch.zeros((1, Nk, Hk, D), dtype=torch.bfloat16, device=DEV)
    v = torch.ones((1, Nk, Hk, D), dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 1 << 31
    q = torch.full((1, 1, 2 * Hk, D), 1.0, dtype=torch.bfloat16, device=DEV)
    k[0, Nk - 1] = 10.0                                       # score 10 sqrt(128) = 113 against 0: nothing else is left
    v[0, Nk - 1] = torch.arange(Hk, device=DEV).view(Hk, 1).to(torch.bfloat16)
    out, lse, rest = ops.attention(q, k, v, for_backward=True)
    want = torch.arange(Hk, device=DEV).repeat_interleave(2).view(1, 1, 2 * Hk, 1).expand_as(out).float()
    assert torch.equal(out.float(), want)
    cut = torch.tensor([Nk - 1], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.attention(q, k, v, kv_len=cut), torch.ones_like(out))      # a mean of equal values
    del out, lse, rest
    # forty rows instead of one: the tiled form, and its backward pass over the same keys
    q = torch.full((1, 40, Hk, D), 1.0, dtype=torch.bfloat16, device=DEV)
    res = ops.attention(q, k, v, for_backward=True)
    assert torch.equal(res[0].float(), torch.arange(Hk, device=DEV).view(1, 1, Hk, 1).expand_as(q).float())
    dq, dk, dv = ops.attention_backward(torch.ones_like(q), q, k, v, *res)
    assert torch.equal(dv[0, Nk - 1], torch.full((Hk, D), 40.0, dtype=torch.bfloat16, device=DEV)) and not dv[0, :Nk - 1].any()
    assert not dk[0, :Nk - 1].any()


def test_calls_at_once_on_two_streams():
    """split calls have partial results in scratch: two at once on two streams give what they give alone"""
    from trace_amd import ops
    sets = [[t.to(DEV) for t in make(2, 40, 3000, 2, 2, 128, s)] for s in (31, 32)]
    want = []
    for q, k, v, do in sets:
        res = ops.attention(q, k, v, for_backward=True)
        want.append(res + ops.attention_backward(do, q, k, v, *res))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, (q, k, v, do) in zip(streams, sets):
            with torch.cuda.stream(st):
                res = ops.attention(q, k, v, for_backward=True)
                got.append(res + ops.attention_backward(do, q, k, v, *res))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
