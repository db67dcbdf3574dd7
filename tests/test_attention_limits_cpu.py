"""How large a call of the attention entry points may be: refused before anything is launched, and not refused for what is no limit."""
import ctypes

import pytest


def desc(**kw):
    from trace_amd import _lib as L
    d = L.AttentionDesc()
    for n, v in dict(dict(batch=1, q_rows=5, k_rows=7, heads=1, kv_heads=1, head_dim=8, causal=0, scale=0.125), **kw).items():
        setattr(d, n, v)
    for n in ("stride_q", "stride_k", "stride_v", "stride_do"):
        setattr(d, n, (ctypes.c_longlong * 3)(0, 0, 0))      # broadcast rows: such calls need no memory for their operands
    return d


@pytest.mark.parametrize("kw", [dict(k_rows=(1 << 31) - 10), dict(q_rows=(1 << 31) - 10), dict(q_rows=(1 << 31) - 200),
                                dict(k_rows=(1 << 31) - 511), dict(q_rows=(1 << 31) - 511)])
def test_rows_whose_tiles_pass_32_bits_are_refused(kw):
    """the last tile of 2^31 - 10 rows ends behind 2^31: row numbers would wrap to negative ones, in front of the operand"""
    from trace_amd import _lib as L
    l, ok = L.lib(), 1 << 20
    d = desc(**kw)
    assert l.trace_attention_fwd_workspace_bytes(d) == 0 and l.trace_attention_bwd_workspace_bytes(d) == 0
    assert b"too many rows" in l.trace_last_error()
    # no pointers but the call is refused for its rows, in front of anything else
    assert l.trace_attention_fwd_bf16(d, *[None] * 7, 0, None) != 0 and b"too many rows" in l.trace_last_error()
    assert l.trace_attention_bwd_bf16(d, *[None] * 11, 0, None) != 0 and b"too many rows" in l.trace_last_error()


@pytest.mark.parametrize("kw", [dict(batch=1 << 10, heads=1 << 10, q_rows=(1 << 11) - 2), dict(batch=1 << 10, heads=1 << 10, kv_heads=1 << 10, k_rows=1 << 11),
                                dict(batch=1 << 20, heads=1 << 12, kv_heads=4)])
def test_grids_past_32_bits_are_refused(kw):
    from trace_amd import _lib as L
    d = desc(**kw)
    assert L.lib().trace_attention_fwd_bf16(d, *[None] * 7, 0, None) != 0 and b"too many rows" in L.lib().trace_last_error()
    assert L.lib().trace_attention_bwd_bf16(d, *[None] * 11, 0, None) != 0 and b"too many rows" in L.lib().trace_last_error()


@pytest.mark.parametrize("kw", [dict(batch=128, heads=64, kv_heads=8, q_rows=1, k_rows=262144, head_dim=128), dict(heads=8, kv_heads=1, k_rows=(1 << 31) - 512),
                                dict(q_rows=(1 << 31) - 512, k_rows=1),
                                dict(batch=1 << 12, heads=1 << 9, q_rows=1, k_rows=1 << 16)])
def test_query_heads_times_key_rows_is_no_limit(kw):
    """the call passes the check of its sizes: the next thing that is wrong with it, null pointers, is what it is refused for"""
    from trace_amd import _lib as L
    d = desc(**kw)
    assert L.lib().trace_attention_bwd_workspace_bytes(d) > 0
    assert L.lib().trace_attention_fwd_bf16(d, *[None] * 7, 0, None) != 0 and b"null pointer" in L.lib().trace_last_error()
    assert L.lib().trace_attention_bwd_bf16(d, *[None] * 11, 0, None) != 0 and b"null pointer" in L.lib().trace_last_error()
