"""Backward of the conv / GEMM family through the same HIP kernels (`loss.backward()` of
tools/train_net_step_rel.py:625 reaches the I3D stages the config leaves trainable, lib/i3d/resnet3d.py:746-767, and
the Linear layers of the relation head).

A convolution's two gradients are convolutions / GEMMs again, so no new device code is needed:

  data gradient    dx = conv3d(zero-stuffed dy, W flipped and transposed, stride 1, padding d (k - 1) - p)
                   - the implicit-GEMM kernel of the forward pass on another operand;
  weight gradient  dW[co][tap][ci] = sum_pos dy[pos][co] x[pos s + tap d - p][ci]: per tap one NT GEMM of dy^T (Cout, M)
                   with the tap's shifted input view transposed (Cin, M), f32 result (K = M positions, split-K inside);
  bias gradient    column sums of dy.

Operands are bf16 as in the forward pass (dy is rounded to bf16), accumulation f32, weight gradients come back in f32
for the f32 master weights.  The strided views / zero stuffing / transposes around the kernels are torch indexing and
`ops.transpose` - plumbing, not the product's arithmetic.  BatchNorm is handled by the caller (ConvModule.run_train):
folded into the weights in eval mode, torch's batch_norm over the raw conv output in training mode.

Softmax attention, group norm + activation and dropout + activation have kernels of their own for both directions
(csrc/attention.hip, norm_ops.hip, dropout_ops.hip); their wrappers stand at the end.

Capturing a backward pass into a graph: let go of every result of an eager pass over the same leaves first (or take fresh
leaves).  torch keeps a leaf's gradient node, with the stream it was made on, as long as any such result lives, and a capture that
reaches another stream through it ends in an error that torch does not recover from.
"""
import functools

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import ops


def _triple_out(i, k, s, p, d):
    return (i + 2 * p - d * (k - 1) - 1) // s + 1


def conv3d_dgrad(gy, w_bf, x_shape, ksize, stride, padding, dilation):
    """gy (N,To,Ho,Wo,Cout) bf16, w_bf (Cout, taps*Cin) bf16 tap-major -> dx (N,Ti,Hi,Wi,Cin) bf16."""
    N, Ti, Hi, Wi, Cin = x_shape
    kt, kh, kw = ksize
    Cout = w_bf.shape[0]
    pads = []
    for k, p, d in zip(ksize, padding, dilation):
        q = d * (k - 1) - p
        if q < 0:
            raise RuntimeError("conv3d backward: padding %d exceeds dilation*(k-1) = %d" % (p, d * (k - 1)))
        pads.append(q)
    # zero-stuff dy back onto the stride-1 grid and append the rows the strided forward never reached
    sizes = []
    for i, k, s, p, d, o in zip((Ti, Hi, Wi), ksize, stride, padding, dilation, gy.shape[1:4]):
        sizes.append(i + 2 * p - d * (k - 1))      # length of the stride-1 output grid
    if tuple(stride) != (1, 1, 1) or tuple(sizes) != tuple(gy.shape[1:4]):
        up = torch.zeros((N, sizes[0], sizes[1], sizes[2], Cout), dtype=gy.dtype, device=gy.device)
        up[:, ::stride[0], ::stride[1], ::stride[2]][:, :gy.shape[1], :gy.shape[2], :gy.shape[3]] = gy
        gy = up
    wt = w_bf.view(Cout, kt, kh, kw, Cin).flip(1, 2, 3).permute(4, 1, 2, 3, 0).reshape(Cin, kt * kh * kw * Cout).contiguous()
    gx = ops.conv3d(gy.contiguous(), wt, None, ksize, (1, 1, 1), tuple(pads), dilation)
    if tuple(gx.shape) != tuple(x_shape):
        raise RuntimeError("conv3d backward: data gradient shape %s != input shape %s" % (tuple(gx.shape), tuple(x_shape)))
    return gx


def conv3d_wgrad(gy, x, ksize, stride, padding, dilation):
    """gy (N,To,Ho,Wo,Cout) bf16, x (N,Ti,Hi,Wi,Cin) bf16 -> dW (Cout, taps*Cin) f32, tap-major like the weights."""
    N, To, Ho, Wo, Cout = gy.shape
    Cin = x.shape[-1]
    kt, kh, kw = ksize
    M = N * To * Ho * Wo
    gyT = ops.transpose(gy.reshape(M, Cout), pad_to=8)                                   # (Cout, Mp), zero tail
    if tuple(padding) != (0, 0, 0):
        x = F.pad(x, (0, 0, padding[2], padding[2], padding[1], padding[1], padding[0], padding[0]))
    taps = []
    for a in range(kt):
        for b in range(kh):
            for c in range(kw):
                t0, h0, w0 = a * dilation[0], b * dilation[1], c * dilation[2]
                xs = x[:, t0:t0 + (To - 1) * stride[0] + 1:stride[0], h0:h0 + (Ho - 1) * stride[1] + 1:stride[1],
                       w0:w0 + (Wo - 1) * stride[2] + 1:stride[2], :]
                xsT = ops.transpose(xs.reshape(M, Cin), pad_to=8)                        # (Cin, Mp)
                taps.append(ops.gemm_nt(gyT, xsT, out_f32=True))                         # (Cout, Cin)
    return torch.stack(taps, 1).reshape(Cout, kt * kh * kw * Cin)


class _Conv3d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, ksize, stride, padding, dilation, relu):
        wb = w.detach().to(torch.bfloat16).contiguous()
        y = ops.conv3d(x.detach(), wb, None if bias is None else bias.detach(), ksize, stride, padding, dilation, relu=relu)
        ctx.save_for_backward(x.detach(), wb, y if relu else None)
        ctx.cfg = (tuple(ksize), tuple(stride), tuple(padding), tuple(dilation), relu, w.dtype)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, wb, y = ctx.saved_tensors
        ksize, stride, padding, dilation, relu, wdt = ctx.cfg
        gy = gy.to(torch.bfloat16)
        if relu:
            gy = gy * (y > 0)
        gy = gy.contiguous()
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = conv3d_dgrad(gy, wb, x.shape, ksize, stride, padding, dilation)
        if ctx.needs_input_grad[1]:
            gw = conv3d_wgrad(gy, x, ksize, stride, padding, dilation).to(wdt)
        if ctx.needs_input_grad[2]:
            gb = gy.float().sum((0, 1, 2, 3))
        return gx, gw, gb, None, None, None, None, None


def conv3d(x, w, bias, ksize, stride=(1, 1, 1), padding=(0, 0, 0), dilation=(1, 1, 1), relu=False):
    """Differentiable ops.conv3d: x (N,T,H,W,Cin) bf16, w (Cout, taps*Cin) f32 (or bf16) master weights, tap-major,
    bias (Cout) f32 or None."""
    return _Conv3d.apply(x, w, bias, tuple(ksize), tuple(stride), tuple(padding), tuple(dilation), bool(relu))


class _GemmNT(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, relu):
        wb = w.detach().to(torch.bfloat16).contiguous()
        xb = x.detach().to(torch.bfloat16).contiguous()
        y = ops.gemm_nt(xb, wb, bias=None if bias is None else bias.detach(), relu=relu)
        ctx.save_for_backward(xb, wb, y if relu else None)
        ctx.cfg = (relu, w.dtype, x.dtype)
        return y

    @staticmethod
    def backward(ctx, gy):
        xb, wb, y = ctx.saved_tensors
        relu, wdt, xdt = ctx.cfg
        if gy.shape[0] == 0:      # no rows: sums over nothing
            grads = (xb.to(xdt), wb.new_zeros(wb.shape, dtype=wdt), wb.new_zeros(wb.shape[:1], dtype=torch.float32))
            return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,)
        gy = gy.to(torch.bfloat16)
        if relu:
            gy = gy * (y > 0)
        gy = gy.contiguous()
        M, N = gy.shape
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            wT = ops.transpose(wb, pad_to=8)                                     # (K, Np)
            g = gy if wT.shape[1] == N else F.pad(gy, (0, wT.shape[1] - N))
            gx = ops.gemm_nt(g.contiguous(), wT).to(xdt)                         # (M, K)
        if ctx.needs_input_grad[1]:
            gw = ops.gemm_nt(ops.transpose(gy, pad_to=8), ops.transpose(xb, pad_to=8), out_f32=True).to(wdt)   # (N, K)
        if ctx.needs_input_grad[2]:
            gb = gy.float().sum(0)
        return gx, gw, gb, None


def gemm_nt(x, w, bias=None, relu=False):
    """Differentiable act(x @ w^T + bias): x (M,K) bf16, w (N,K) f32 (or bf16) master weights, K % 8 == 0."""
    return _GemmNT.apply(x, w, bias, bool(relu))


def _once(backward):
    """once_differentiable, which only a backward pass that is itself recorded (create_graph) has to pay for: its no_grad block
    costs as much host time as two launches."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _as(t, dtype):
    return t if t.dtype == dtype else t.to(dtype)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_len, kv_len):
        out, lse, rest = ops.attention(q, k, v, scale, causal, q_len, kv_len, for_backward=True)
        ctx.save_for_backward(q, k, v, out, lse, rest, q_len, kv_len)
        ctx.cfg = (scale, causal)
        return out

    @staticmethod
    @_once
    def backward(ctx, gout):
        q, k, v, out, lse, rest, q_len, kv_len = ctx.saved_tensors
        grads = ops.attention_backward(_as(gout, torch.bfloat16), q, k, v, out, lse, rest, *ctx.cfg, q_len, kv_len)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 4


def attention(q, k, v, scale=None, causal=False, q_len=None, kv_len=None):
    """Differentiable ops.attention (same arguments); gradients reach q, k and v.  Kept for the backward pass: the operands,
    the output, what its rounding lost (another bf16 tensor like it) and one f32 per row - the probabilities are recomputed.
    Without a gradient to come it is ops.attention itself, whose output may differ in its last bit from the one that a gradient
    belongs to (the first pass of a checkpointed block, validation): both are within their rounding of the exact one."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return ops.attention(q, k, v, scale, causal, q_len, kv_len)
    return _Attention.apply(q, k, v, scale, bool(causal), q_len, kv_len)


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, gamma, beta, eps, act):
        y, stats = ops.group_norm_act(x, groups, gamma, beta, eps, act, return_stats=True)
        ctx.save_for_backward(x, stats, gamma, beta)
        ctx.cfg = (groups, act)
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, stats, gamma, beta = ctx.saved_tensors
        groups, act = ctx.cfg
        need = ctx.needs_input_grad
        dx, dg, db = ops.group_norm_act_backward(_as(gy, x.dtype), x, stats, groups, gamma, beta, act, param_grads=need[2] or need[3])
        return (dx if need[0] else None, None, _as(dg, gamma.dtype) if need[2] else None, _as(db, beta.dtype) if need[3] else None,
                None, None)


def group_norm_act(x, groups, gamma=None, beta=None, eps=1e-5, act=None):
    """Differentiable ops.group_norm_act (same arguments); gradients reach x, gamma and beta.  Kept for the backward pass: x and
    two f32 per (sample, group)."""
    return _GroupNormAct.apply(x, int(groups), gamma, beta, float(eps), act)


class _DropoutAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, act, step):
        y = ops.dropout_act(x, p, seed, offset, act, step)
        ctx.save_for_backward(x if act not in (None, "none") else None, step)
        ctx.cfg = (p, seed, offset, act, x.dtype)
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, step = ctx.saved_tensors
        p, seed, offset, act, dt = ctx.cfg
        return (ops.dropout_act_backward(_as(gy, dt), x, p, seed, offset, act, step),) + (None,) * 5


def dropout_act(x, p, seed, offset=0, act=None, step=None, training=True):
    """Differentiable ops.dropout_act (same arguments); without `training` nothing is dropped (p = 0).  Kept for the backward
    pass: x where an activation follows, no mask.  `step` must not be advanced before the backward pass has been issued (autograd
    reports it)."""
    return _DropoutAct.apply(x, float(p) if training else 0.0, int(seed), int(offset), act, step)
