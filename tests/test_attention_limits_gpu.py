"""A long cache of many sequences and heads: what bounds a call are the rows of its own grids, not query heads times key rows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U, F = torch.finfo(torch.bfloat16).eps / 2, 2.0 ** -24


def test_many_sequences_over_long_caches():
    """128 sequences x 64 heads over 8 key heads of 262144 rows (all of them one row block in memory, broadcast), a token each: rows
    of different sequences and heads against the definition in 64 bits.  Bound as in test_attention_gpu.py: the result's rounding,
    that of the probabilities, and what 32 bits lose in scores, exponentials and sums."""
    from trace_amd import ops
    B, H, Hk, Nk, D = 128, 64, 8, 262144, 128
    assert B * H * Nk >= 1 << 31
    g = torch.Generator().manual_seed(8)
    q = torch.randn((B, 1, H, D), generator=g).bfloat16()
    k, v = (torch.randn((1, Nk, 1, D), generator=g).bfloat16() for _ in range(2))
    kd, vd = (t.to(DEV).expand(B, Nk, Hk, D) for t in (k, v))
    out, lse = ops.attention(q.to(DEV), kd, vd, return_lse=True)
    assert torch.isfinite(out).all()
    kk, vv = k[0, :, 0].double(), v[0, :, 0].double()
    for b, h in ((0, 0), (0, 63), (1, 8), (64, 31), (127, 0), (127, 63)):
        qq = q[b, 0, h].double()
        s = kk @ qq * D ** -0.5
        l = torch.logsumexp(s, 0)
        P = torch.exp(s - l)
        o, A = P @ vv, P @ vv.abs()
        p_rel = 2 * float(((D + 2) * F * D ** -0.5 * (kk.abs() @ qq.abs())).max()) + 2 ** -20 + float(l.abs() + s.abs().max()) * 2 ** -22 + Nk * F
        bound = U * o.abs() + (U + p_rel + Nk * F) * A * (1 + U)
        assert bool(((out[b, 0, h].double().cpu() - o).abs() <= bound).all()), (b, h)
        assert abs(float(lse[b, h, 0]) - float(l)) <= p_rel + float(l.abs()) * 2 ** -22 + 1e-6, (b, h)


def test_rows_are_counted_apart():
    """the same for a call with a backward pass: few query heads' rows, many key rows"""
    from trace_amd import ops
    B, H, Hk, Nk, D = 1 << 14, 64, 1, 2100, 8
    assert B * H * Nk >= 1 << 31
    q = torch.ones((1, 1, 1, D), dtype=torch.bfloat16, device=DEV).expand(B, 1, H, D)
    k = torch.zeros((B, Nk, Hk, D), dtype=torch.bfloat16, device=DEV)
    v = torch.ones((1, Nk, 1, D), dtype=torch.bfloat16, device=DEV).expand(B, Nk, Hk, D)
    res = ops.attention(q, k, v, for_backward=True)
    assert bool((res[0] == 1).all()) and float((res[1] - math.log(Nk)).abs().max()) < 1e-5
    dq, dk, dv = ops.attention_backward(res[0], q, k, v, *res)
    # P = 1 / Nk, dS = P (8 - delta), delta = 8 but for a rounding or two in 32 bits of out + rest; dv = 64 heads / Nk: one rounding
    # of P and one of the result
    assert not dq.any() and float(dk.float().abs().max()) <= H * D ** -0.5 / Nk * 8 * 4 * F
    assert float((dv.float() * (Nk / 64.0) - 1).abs().max()) <= 2 * U + U * U + 1e-5


def test_rows_past_30_bits():
    """1.5 x 2^30 keys, all of them one row in memory: the mean of equal values, the logarithm of their number and, under a causal
    mask, the same (the last query sees every key)"""
    from trace_amd import ops
    Nk, D = 3 << 29, 8
    q = torch.full((1, 1, 1, D), 0.5, dtype=torch.bfloat16, device=DEV)
    k = torch.full((1, 1, 1, D), 0.25, dtype=torch.bfloat16, device=DEV).expand(1, Nk, 1, D)
    v = torch.arange(D, device=DEV).to(torch.bfloat16).view(1, 1, 1, D).expand(1, Nk, 1, D)
    for causal in (False, True):
        out, lse = ops.attention(q, k, v, causal=causal, return_lse=True)
        assert torch.equal(out, v[:, :1])
        want = D * 0.125 * D ** -0.5 + math.log(Nk)
        assert abs(float(lse) - want) <= 8 * 2.0 ** -23 * want
    few = torch.tensor([Nk - 7], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.attention(q, k, v, kv_len=few), v[:, :1])
