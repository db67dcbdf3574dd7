"""Operators of a training step, as cases that can be timed and checked: softmax attention (forward, and forward +
backward), group normalisation with an activation over channels-last maps, and dropout from a counter-based generator.

A case is a dict of plain values.  `listed()` gives the named ones, `draw(rng)` another one of the same ranges, `prepare`
the inputs a caller has in hand, `run` one pass (`own` false: the operator written out in elementary torch operations;
true: the calls of trace_amd), `work` what a pass has to read, write and compute, `exact` its outputs in 64 bits.

attention   q (B, Nq, H, D), k / v (B, Nk, Hkv, D) bf16, H a multiple of Hkv (query head h reads head h // (H / Hkv));
            out[i] = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that query i sees: j < kv_len[b], and with
            `causal` also j <= i + kv_len[b] - q_len[b].  Rows at or behind q_len[b] and rows that see no key are zero
            and have no gradient; keys at or behind kv_len[b] are not read and have no gradient.
group norm  x (N, P, C): per sample and group of C / G channels, z = (x - mean) / sqrt(var + eps) * gamma + beta over the
            P * C / G elements, y = act(z).
dropout     y = act(x * keep / q) with q the probability of keep: element i takes the i % 8-th 16-bit piece of
            Philox4x32-10(counter = (i // 8, offset), key = seed) and is dropped where that piece < round(p * 65536).
"""
import math
import random

import torch

own = False

LEAKY = 0.1
EPS = 1e-5
DEVICE = "cuda"


# ---------------------------------------------------------------------------------------------------------- cases
def _attn(name, train, batch, q_rows, k_rows, heads, kv_heads, head_dim, causal, ragged):
    c = dict(op="attention", train=train, batch=batch, q_rows=q_rows, k_rows=k_rows, heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, causal=causal, ragged=ragged)
    return dict(c, name=name) if name else c


def _norm(name, train, samples, positions, channels, groups, act, dtype):
    c = dict(op="group_norm", train=train, samples=samples, positions=positions, channels=channels, groups=groups, act=act,
             dtype=dtype)
    return dict(c, name=name) if name else c


def _drop(name, rows, width, p, act, dtype):
    c = dict(op="dropout", rows=rows, width=width, p=p, act=act, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one query per tracked box over its 8 frames, 20 boxes in each of 8 clips, some of them seen in fewer frames: the
        # smallest call, where latency counts
        _attn("attn_frames", False, 160, 1, 8, 4, 4, 64, False, "keys"),
        # single tokens against long histories of unequal length, four query heads to a key head: bytes of the cache
        _attn("attn_token", False, 4, 1, 16384, 32, 8, 128, False, "keys"),
        # softmax non-local block behind layer2 at 8 clips of 32 x 224 x 224: 4 x 28 x 28 positions against their
        # (1, 2, 2)-pooled ones, 256 channels in one head
        _attn("attn_nonlocal2", False, 8, 3136, 784, 1, 1, 256, False, "none"),
        # the block behind layer3 in a training step: 4 x 14 x 14 against pooled, 512 channels
        _attn("attn_nonlocal3_train", True, 8, 784, 196, 1, 1, 512, False, "none"),
        # causal self-attention over long sequences with shared key heads, a training step: the largest
        _attn("attn_causal_train", True, 2, 4096, 4096, 16, 4, 128, True, "none"),
        # padded batches of odd length whose rows are partly or wholly padding, a training step
        _attn("attn_ragged_train", True, 16, 197, 197, 12, 12, 64, False, "both"),
        # layer3's maps of one short clip, inference: a small call
        _norm("norm_clip", False, 1, 4 * 14 * 14, 256, 32, "relu", "bf16"),
        # layer1's maps at 8 clips (8 frames of 56 x 56, 256 channels), a training step: bytes
        _norm("norm_layer1_train", True, 8, 8 * 56 * 56, 256, 32, "silu", "bf16"),
        # f32 maps of odd extent, groups of 5 channels, a training step
        _norm("norm_odd_train", True, 3, 45 * 31, 60, 12, None, "f32"),
        # the widest maps, inference: layer4 at 8 clips
        _norm("norm_layer4", False, 8, 4 * 14 * 14, 2048, 32, "relu", "bf16"),
        # the relation MLP's input for 8 clips of 380 pairs, a training step: small
        _drop("drop_pairs", 3040, 256, 0.5, "leaky", "bf16"),
        # dropout over a layer's whole map, a training step: bytes
        _drop("drop_maps", 200704, 256, 0.1, None, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "group_norm", "group_norm", "dropout"])
    cap = {}
    for c in listed():
        w = work(c)
        for k in w:
            cap[c["op"], k] = max(cap.get((c["op"], k), 0), w[k])
    while True:
        if op == "attention":
            train = rng.random() < 0.5
            kv_heads = rng.choice([1, 1, 2, 4, 8, 12])
            heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
            head_dim = 8 * _log_int(rng, 1, 64)
            k_rows = _log_int(rng, 16, 4096) if train else _log_int(rng, 1, 16384)
            q_rows = rng.choice([1, k_rows, _log_int(rng, 1, 4096)])
            q_rows = min(q_rows, 4096)
            c = _attn(None, train, _log_int(rng, 1, 160), q_rows, k_rows, heads, kv_heads, head_dim, rng.random() < 0.4,
                      rng.choice(["none", "keys", "both"]))
        elif op == "group_norm":
            per = rng.choice([1, 2, 3, 5, 8, 16, 30, 64])
            groups = rng.choice([1, 4, 8, 12, 32])
            train = rng.random() < 0.5
            c = _norm(None, train, _log_int(rng, 1, 16), _log_int(rng, 16, 25088), min(per * groups, 2048) // groups * groups,
                      groups, rng.choice([None, "silu"] if train else [None, "relu", "leaky", "silu"]),
                      rng.choice(["bf16", "bf16", "f32"]))
        else:
            c = _drop(None, _log_int(rng, 1, 200704), _log_int(rng, 1, 2048), rng.choice([0.0, 0.1, 0.25, 0.5, rng.random()]),
                      rng.choice([None, "relu", "leaky"]), rng.choice(["bf16", "bf16", "f32"]))
        w = work(c)
        if all(w[k] <= cap[op, k] for k in w):
            return c


def _lens(case):
    """(q_len, kv_len) of a batch as lists, or None where all rows count.  Lengths fall from full to a small share over the
    batch; in a batch of three or more the second entry has none at all."""
    B = case["batch"]

    def fall(n):
        out = [max(1, n - (b * n * 7) // (8 * B)) for b in range(B)]
        if B > 2:
            out[1] = 0
        return out
    kv = fall(case["k_rows"]) if case["ragged"] in ("keys", "both") else None
    q = fall(case["q_rows"]) if case["ragged"] == "both" else None
    return q, kv


_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------ work
def _pairs(case):
    """Query-key pairs of the whole batch (per head), rows of queries and of keys that count."""
    q_len, kv_len = _lens(case)
    B, Nq, Nk = case["batch"], case["q_rows"], case["k_rows"]
    n = rq = rk = 0
    for b in range(B):
        lq = q_len[b] if q_len else Nq
        lk = kv_len[b] if kv_len else Nk
        rq += lq
        rk += lk
        if not case["causal"]:
            n += lq * lk
            continue
        # query i sees max(0, min(lk, i + lk - lq + 1)) keys
        first = max(0, lq - lk)
        m = lq - first
        if m > 0 and lk > 0:
            a = first + lk - lq + 1
            n += m * (a + lk) // 2
    return n, rq, rk


def work(case):
    if case["op"] == "attention":
        n, rq, rk = _pairs(case)
        H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
        full_q, full_k = case["batch"] * case["q_rows"] * H * D, case["batch"] * case["k_rows"] * Hk * D
        q, k = rq * H * D, rk * Hk * D
        if case["train"]:
            # read q, k, v and the output's gradient; write the output and three gradients
            return {"bytes": 2 * (2 * q + 2 * k + 2 * full_q + 2 * full_k), "flops": 14 * n * H * D}
        return {"bytes": 2 * (q + 2 * k + full_q), "flops": 4 * n * H * D}
    if case["op"] == "group_norm":
        e = case["samples"] * case["positions"] * case["channels"]
        s = 2 if case["dtype"] == "bf16" else 4
        # forward: x in, y out; a training step also reads the gradient and writes x's
        return {"bytes": e * s * (4 if case["train"] else 2), "flops": e * (24 if case["train"] else 8)}
    e = case["rows"] * case["width"]
    s = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": e * s * 4, "flops": 4 * e}


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    st = {"case": case}
    if case["op"] == "attention":
        B, D = case["batch"], case["head_dim"]
        q = (B, case["q_rows"], case["heads"], D)
        k = (B, case["k_rows"], case["kv_heads"], D)
        # projections of normalised features: scores of a few units, so that some rows are peaked and most are not
        st["q"] = (randn(*q) * 1.3).bfloat16()
        st["k"] = (randn(*k) * 1.3 + 0.2 * randn(1, 1, case["kv_heads"], D)).bfloat16()
        st["v"] = randn(*k).bfloat16()
        if case["train"]:
            st["do"] = (randn(*q) * 0.05).bfloat16()
        q_len, kv_len = _lens(case)
        st["q_len"] = torch.tensor(q_len, dtype=torch.int32, device=DEVICE) if q_len else None
        st["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=DEVICE) if kv_len else None
    elif case["op"] == "group_norm":
        dt, C = _DT[case["dtype"]], case["channels"]
        # a convolution's output: every channel with its own mean and spread
        st["x"] = (randn(case["samples"], case["positions"], C) * (0.3 + randn(C).abs()) + 1.5 * randn(C)).to(dt)
        st["gamma"] = 1.0 + 0.2 * randn(C)
        st["beta"] = 0.2 * randn(C)
        if case["train"]:
            st["dy"] = (randn(*st["x"].shape) * 0.05).to(dt)
    else:
        dt = _DT[case["dtype"]]
        st["x"] = randn(case["rows"], case["width"]).to(dt)
        st["dy"] = (randn(case["rows"], case["width"]) * 0.05).to(dt)
        r = random.Random(seed)
        st["seed"], st["offset"] = r.getrandbits(63), r.getrandbits(40)
    return st


# ------------------------------------------------------------------------------------------------------ plain forms
_CHUNK = 1 << 29     # scores formed at once


def _seen(case, q_len, kv_len, b0, b1):
    """(b1 - b0, Nq, Nk) bool: the pairs that count."""
    Nq, Nk, dev = case["q_rows"], case["k_rows"], DEVICE
    i = torch.arange(Nq, device=dev).view(1, Nq, 1)
    j = torch.arange(Nk, device=dev).view(1, 1, Nk)
    lq = q_len[b0:b1].view(-1, 1, 1) if q_len is not None else torch.full((b1 - b0, 1, 1), Nq, device=dev)
    lk = kv_len[b0:b1].view(-1, 1, 1) if kv_len is not None else torch.full((b1 - b0, 1, 1), Nk, device=dev)
    m = (i < lq) & (j < lk)
    if case["causal"]:
        m = m & (j <= i + lk - lq)
    return m


def _plain_attention(st):
    case = st["case"]
    B, Nq, Nk, H, Hk, D = (case[n] for n in ("batch", "q_rows", "k_rows", "heads", "kv_heads", "head_dim"))
    G = H // Hk
    scale = D ** -0.5
    out = torch.empty_like(st["q"])
    if case["train"]:
        dq, dk, dv = torch.empty_like(st["q"]), torch.empty_like(st["k"]), torch.empty_like(st["v"])
    step = max(1, _CHUNK // (Nq * Nk * G))       # (batch, key head) units per chunk
    bs = max(1, min(B, step // Hk))
    hs = Hk if step >= Hk else step

    def rows(t, b0, b1, h0, h1, n):              # (B, N, heads, D) -> f32 (units, rows, D) of the key heads h0 .. h1
        g = t.shape[2] // Hk
        t = t[b0:b1, :, h0 * g:h1 * g].float().permute(0, 2, 1, 3)
        return t.reshape((b1 - b0) * (h1 - h0), g * n, D)

    def back(t, b0, b1, h0, h1, n, dst):
        g = dst.shape[2] // Hk
        dst[b0:b1, :, h0 * g:h1 * g] = t.view(b1 - b0, (h1 - h0) * g, n, D).permute(0, 2, 1, 3).to(dst.dtype)

    for b0 in range(0, B, bs):
        b1 = min(B, b0 + bs)
        hide = ~_seen(case, st["q_len"], st["kv_len"], b0, b1)
        for h0 in range(0, Hk, hs):
            h1 = min(Hk, h0 + hs)
            q, k, v = rows(st["q"], b0, b1, h0, h1, Nq), rows(st["k"], b0, b1, h0, h1, Nk), rows(st["v"], b0, b1, h0, h1, Nk)
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
            s5 = s.view(b1 - b0, h1 - h0, G, Nq, Nk)
            s5.masked_fill_(hide.view(b1 - b0, 1, 1, Nq, Nk), float("-inf"))
            m = s.amax(-1, keepdim=True)
            m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
            s.sub_(m).exp_()
            tot = s.sum(-1, keepdim=True)
            p = s.div_(torch.where(tot == 0, torch.ones_like(tot), tot))
            o = torch.matmul(p, v)
            back(o, b0, b1, h0, h1, Nq, out)
            if case["train"]:
                do = rows(st["do"], b0, b1, h0, h1, Nq)
                dp = torch.matmul(do, v.transpose(1, 2).contiguous())
                dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
                back(torch.matmul(dp, k) * scale, b0, b1, h0, h1, Nq, dq)
                back(torch.matmul(dp.transpose(1, 2).contiguous(), q) * scale, b0, b1, h0, h1, Nk, dk)
                back(torch.matmul(p.transpose(1, 2).contiguous(), do), b0, b1, h0, h1, Nk, dv)
    return (out, dq, dk, dv) if case["train"] else out


def _plain_norm(st):
    case = st["case"]
    N, P, C, G = case["samples"], case["positions"], case["channels"], case["groups"]
    x = st["x"].float().view(N, P, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
    gamma, beta = st["gamma"].view(1, 1, G, C // G), st["beta"].view(1, 1, G, C // G)
    xh = (x - mean) * rstd
    z = xh * gamma + beta
    act = case["act"]
    if act == "relu":
        y, d = torch.where(z > 0, z, torch.zeros_like(z)), None
    elif act == "leaky":
        y, d = torch.where(z > 0, z, LEAKY * z), None
    elif act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        y, d = z * s, s * (1.0 + z * (1.0 - s))
    else:
        y, d = z, None
    y = y.view(N, P, C).to(st["x"].dtype)
    if not case["train"]:
        return y
    dz = st["dy"].float().view(N, P, G, C // G)
    if d is not None:
        dz = dz * d
    dgamma, dbeta = (dz * xh).sum((0, 1)).view(C), dz.sum((0, 1)).view(C)
    t = dz * gamma
    dx = (t - t.mean((1, 3), keepdim=True) - xh * (t * xh).mean((1, 3), keepdim=True)) * rstd
    return y, dx.view(N, P, C).to(st["x"].dtype), dgamma, dbeta


def _mul32(a, m):
    """(high, low) words of the 64-bit product of 32-bit words a (int64) and m (int), without leaving 63 bits."""
    lo = a * (m & 0xFFFF)
    hi = a * (m >> 16) + (lo >> 16)
    return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def _plain_pieces(n, seed, offset):
    """n 16-bit pieces: Philox4x32-10 (Salmon et al., 2011)."""
    i = torch.arange((n + 7) // 8, device=DEVICE, dtype=torch.int64)
    c = [i & 0xFFFFFFFF, i >> 32, torch.full_like(i, offset & 0xFFFFFFFF), torch.full_like(i, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul32(c[0], 0xD2511F53)
        h1, l1 = _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([w for v in c for w in (v & 0xFFFF, v >> 16)], 1).view(-1)[:n]


def _plain_dropout(st):
    case = st["case"]
    x = st["x"]
    t = int(math.floor(case["p"] * 65536 + 0.5))
    keep = (_plain_pieces(x.numel(), st["seed"], st["offset"]) >= t).view(x.shape)
    f = 65536.0 / (65536 - t) if t < 65536 else 0.0
    zero = torch.zeros((), device=x.device)
    xs = torch.where(keep, x.float() * f, zero)
    g = torch.where(keep, st["dy"].float() * f, zero)
    if case["act"] is not None:
        low = LEAKY if case["act"] == "leaky" else 0.0
        g = torch.where(xs > 0, g, low * g)
        xs = torch.where(xs > 0, xs, low * xs)
    return xs.to(x.dtype), g.to(x.dtype)


# -------------------------------------------------------------------------------------------------- the framework's
def _own(st):
    from trace_amd import autograd as tag, ops
    case = st["case"]
    if case["op"] == "attention":
        kw = dict(causal=case["causal"], q_len=st["q_len"], kv_len=st["kv_len"])
        if not case["train"]:
            return ops.attention(st["q"], st["k"], st["v"], **kw)
        q, k, v = (st[n].detach().requires_grad_(True) for n in "qkv")
        out = tag.attention(q, k, v, **kw)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), st["do"])
    if case["op"] == "group_norm":
        if not case["train"]:
            return ops.group_norm_act(st["x"], case["groups"], st["gamma"], st["beta"], EPS, case["act"])
        x, gamma, beta = (st[n].detach().requires_grad_(True) for n in ("x", "gamma", "beta"))
        y = tag.group_norm_act(x, case["groups"], gamma, beta, EPS, case["act"])
        return (y.detach(),) + torch.autograd.grad(y, (x, gamma, beta), st["dy"])
    x = st["x"].detach().requires_grad_(True)
    y = tag.dropout_act(x, case["p"], st["seed"], st["offset"], case["act"])
    return (y.detach(),) + torch.autograd.grad(y, (x,), st["dy"])


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "group_norm": _plain_norm, "dropout": _plain_dropout}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- in 64 bits, apart
def _exact_attention(st):
    case = st["case"]
    B, Nq, Nk, H, Hk, D = (case[n] for n in ("batch", "q_rows", "k_rows", "heads", "kv_heads", "head_dim"))
    q_len, kv_len = _lens(case)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE)
    grads = [torch.zeros(st[n].shape, dtype=torch.float64, device=DEVICE) for n in "qkv"] if case["train"] else None
    for b in range(B):
        lq, lk = q_len[b] if q_len else Nq, kv_len[b] if kv_len else Nk
        first = max(0, lq - lk) if case["causal"] else 0       # queries before it see no key
        if lk == 0 or first >= lq:
            continue
        for h in range(H):
            q = st["q"][b, first:lq, h].double().requires_grad_(case["train"])
            k = st["k"][b, :lk, h // (H // Hk)].double().requires_grad_(case["train"])
            v = st["v"][b, :lk, h // (H // Hk)].double().requires_grad_(case["train"])
            s = q @ k.t() / math.sqrt(D)
            if case["causal"]:
                far = torch.ones_like(s, dtype=torch.bool).triu(lk - lq + first + 1)
                s = s.masked_fill(far, float("-inf"))
            o = torch.softmax(s, -1) @ v
            out[b, first:lq, h] = o.detach()
            if case["train"]:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), st["do"][b, first:lq, h].double())
                grads[0][b, first:lq, h] = gq
                grads[1][b, :lk, h // (H // Hk)] += gk
                grads[2][b, :lk, h // (H // Hk)] += gv
    return (out,) + tuple(grads) if case["train"] else out


def _exact_norm(st):
    case = st["case"]
    G = case["groups"]
    ys, dxs, dg, db = [], [], 0.0, 0.0
    for n in range(case["samples"]):
        x = st["x"][n].double().requires_grad_(case["train"])
        gamma, beta = (st[t].double().requires_grad_(case["train"]) for t in ("gamma", "beta"))
        parts = x.unflatten(-1, (G, -1)).movedim(1, 0)                        # (G, P, C / G)
        var, mean = torch.var_mean(parts.reshape(G, -1), dim=1, unbiased=False)
        h = (parts - mean.view(G, 1, 1)) / (var.view(G, 1, 1) + EPS).sqrt()
        z = h.movedim(0, 1).flatten(1) * gamma + beta
        y = {None: lambda t: t, "relu": torch.relu, "leaky": lambda t: torch.nn.functional.leaky_relu(t, LEAKY),
             "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z)
        ys.append(y.detach())
        if case["train"]:
            a, b, c = torch.autograd.grad(y, (x, gamma, beta), st["dy"][n].double())
            dxs.append(a)
            dg, db = dg + b, db + c
    y = torch.stack(ys)
    return (y, torch.stack(dxs), dg, db) if case["train"] else y


def _exact_dropout(st):
    import numpy as np
    case = st["case"]
    n = st["x"].numel()
    word = np.uint64(0xFFFFFFFF)
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    x = np.empty((4, i.size), np.uint64)
    x[0], x[1] = i & word, i >> np.uint64(32)
    x[2], x[3] = st["offset"] % (1 << 32), st["offset"] >> 32
    key = [st["seed"] % (1 << 32), st["seed"] >> 32]
    for r in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)       # exact: both factors have 32 bits
        k0 = np.uint64((key[0] + r * 0x9E3779B9) % (1 << 32))
        k1 = np.uint64((key[1] + r * 0xBB67AE85) % (1 << 32))
        x = np.stack([(b >> np.uint64(32)) ^ x[1] ^ k0, b & word, (a >> np.uint64(32)) ^ x[3] ^ k1, a & word])
    pieces = np.stack([x & np.uint64(0xFFFF), x >> np.uint64(16)], 1).reshape(8, -1).T.reshape(-1)[:n]
    drop = int(case["p"] * 65536 + 0.5)
    keep = torch.from_numpy(pieces >= np.uint64(drop)).to(DEVICE).view(st["x"].shape)
    f = 65536.0 / max(65536 - drop, 1)
    low = {None: 1.0, "relu": 0.0, "leaky": LEAKY}[case["act"]]
    res = []
    for t in (st["x"], st["dy"]):
        r = t.double() * f
        r = torch.where(st["x"] > 0, r, low * r)
        res.append(torch.where(keep, r, torch.zeros_like(r)))
    return tuple(res)


def exact(case, seed):
    if case["op"] == "attention" and case["batch"] * case["heads"] > 4000:
        return None             # one small product after another: minutes
    st = prepare(case, seed)
    return {"attention": _exact_attention, "group_norm": _exact_norm, "dropout": _exact_dropout}[case["op"]](st)
