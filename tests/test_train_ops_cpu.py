"""The numpy generator the GPU tests compare against, pinned by the published known answers of Philox4x32-10, and the refusals
of the operators' C entry points (all of them before anything is launched)."""
import ctypes

import numpy as np
import pytest

from philox_ref import philox


@pytest.mark.parametrize("ctr,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_known_answers(ctr, key, want):
    got = philox(np.array(ctr, np.uint64).reshape(4, 1), key)
    assert tuple(int(v) for v in got[:, 0]) == want


def test_dropout_entry_refuses():
    from trace_amd import _lib as L
    l = L.lib()
    ok = 1 << 20
    for args in ((None, 8, 100, 0, 0, None, 0, ok), (ok, 8, 100, 0, 0, None, 0, None), (ok, -1, 100, 0, 0, None, 0, ok),
                 (ok, 8, -1, 0, 0, None, 0, ok), (ok, 8, 65537, 0, 0, None, 0, ok), (ok, 8, 100, 0, 0, None, 256, ok),
                 (ok, 8, 100, 0, 0, None, 9, ok), (ok + 2, 8, 100, 0, 0, None, 0, ok), (ok, 8, 100, 0, 0, ok + 4, 0, ok)):
        assert l.trace_dropout_act_bf16(*args, None) != 0 and l.trace_last_error()
        assert l.trace_dropout_act_f32(*args, None) != 0
    assert l.trace_dropout_act_bf16(None, 0, 100, 0, 0, None, 0, None, None) == 0
    for args in ((ok, None, 8, 100, 0, 0, None, 0, ok), (None, ok, 8, 100, 0, 0, None, 8, ok)):
        assert l.trace_dropout_act_bwd_bf16(*args, None) != 0


def test_group_norm_entry_refuses():
    from trace_amd import _lib as L
    l = L.lib()
    ok, ws = 1 << 20, 1 << 30
    good = dict(x=ok, N=2, P=10, C=16, G=4, gamma=None, beta=None, eps=1e-5, act=0, y=ok, stats=ok, ws=ok, n=ws)
    for bad in (dict(x=None), dict(y=None), dict(stats=None), dict(G=3), dict(G=0), dict(C=0), dict(N=-1), dict(P=-1), dict(P=1 << 30),
                dict(N=65536), dict(C=8200, G=1), dict(act=9), dict(act=16), dict(eps=-1.0), dict(x=ok + 8), dict(y=ok + 2),
                dict(P=100000, C=64, G=8, n=0), dict(P=100000, C=64, G=8, ws=None)):
        a = dict(good, **bad)
        assert l.trace_group_norm_act_bf16(*a.values(), None) != 0, bad
        assert l.trace_last_error()
    assert l.trace_group_norm_workspace_bytes(2, 10, 16, 3, 0) == 0
    assert l.trace_group_norm_workspace_bytes(8, 25088, 256, 32, 0) > 0


def test_attention_entry_refuses():
    from trace_amd import _lib as L
    l = L.lib()
    ok = 1 << 20

    def desc(**kw):
        d = L.AttentionDesc()
        a = dict(batch=2, q_rows=5, k_rows=7, heads=4, kv_heads=2, head_dim=64, causal=0, scale=0.125)
        a.update(kw)
        st = a.pop("strides", (8, 8, 8))
        for n, v in a.items():
            setattr(d, n, v)
        for n in ("stride_q", "stride_k", "stride_v", "stride_do"):
            setattr(d, n, (ctypes.c_longlong * 3)(*st))
        return d
    for kw in (dict(batch=-1), dict(q_rows=-1), dict(k_rows=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(head_dim=0), dict(head_dim=4),
               dict(head_dim=68), dict(head_dim=520), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(strides=(8, 4, 8)), dict(batch=1 << 15, heads=1 << 10, kv_heads=1, q_rows=1 << 10)):
        d = desc(**kw)
        assert l.trace_attention_fwd_bf16(d, ok, ok, ok, ok, ok, None, ok, 1 << 40, None) != 0, kw
        assert l.trace_attention_bwd_bf16(d, *[ok] * 10, ok, 1 << 40, None) != 0, kw
        assert l.trace_attention_fwd_workspace_bytes(d) == 0
    d = desc()
    for i in (0, 1, 2, 3):
        for v in (None, ok + 8):
            a = [ok] * 6
            a[i] = v
            assert l.trace_attention_fwd_bf16(d, *a, ok, 1 << 30, None) != 0
    assert l.trace_attention_fwd_bf16(d, ok, ok, ok, ok, ok, ok + 8, ok, 1 << 30, None) != 0
    for i in range(10):
        a = [ok] * 10
        a[i] = None
        assert l.trace_attention_bwd_bf16(d, *a, ok, 1 << 30, None) != 0
    assert l.trace_attention_bwd_bf16(d, *[ok] * 10, ok, 16, None) != 0            # workspace too small
    assert l.trace_attention_bwd_bf16(d, *[ok] * 10, None, 1 << 30, None) != 0
    long_keys = desc(q_rows=1, k_rows=100000)
    assert l.trace_attention_fwd_workspace_bytes(long_keys) > 0
    assert l.trace_attention_fwd_bf16(long_keys, ok, ok, ok, ok, ok, None, ok, 0, None) != 0
    assert l.trace_attention_fwd_bf16(desc(batch=0), *[None] * 7, 0, None) == 0
