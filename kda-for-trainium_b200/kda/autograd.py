"""Autograd bindings: the library's forward and backward kernels as one
differentiable op for training code.

    y = kda.autograd.rmsnorm_matmul(x, w, g, 1e-6)   # bf16 x, w; fp32 g (or None)
    y.backward(dy)                                   # x.grad, w.grad, g.grad from the kernels
    y = kda.autograd.swiglu(x, w_up, w_down, w_gate)  # bf16; all four gradients from the kernels
    o = kda.autograd.gqa_full(q, k, v, causal=True, rope_theta=1e4)  # bf16; dq, dk, dv from the kernels
    q, k = kda.autograd.qk_norm_rope(q, k, gq, gk, table)            # dq, dk, dgq, dgk from the kernels
    o = kda.autograd.gqa_window(q, k, v, 1024, sinks=4)              # bf16; dq, dk, dv from the kernels
"""

from __future__ import annotations

import torch

from . import ops


class _RMSNormMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, g, eps):
        ctx.save_for_backward(x, w, g)
        ctx.eps = float(eps)
        return ops.rmsnorm_matmul(x, w, g, eps)

    @staticmethod
    def backward(ctx, dy):
        x, w, g = ctx.saved_tensors
        dx, dw, dg = ops.rmsnorm_matmul_backward(dy.to(torch.bfloat16).contiguous(), x, w, g, ctx.eps)
        return dx, dw, dg, None


def rmsnorm_matmul(x, w, g=None, eps=0.0):
    """Differentiable ``kda.rmsnorm_matmul``: gradients for x, w and g come
    from ``kda.rmsnorm_matmul_backward``."""
    return _RMSNormMatmul.apply(x, w, g, eps)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_up, w_down, w_gate):
        # the forward keeps g = x w_gate and u = x w_up, so the backward does
        # not recompute them
        out, g, u = ops.swiglu_gu(x, w_up, w_down, w_gate)
        ctx.save_for_backward(x, w_up, w_down, w_gate, g, u)
        return out

    @staticmethod
    def backward(ctx, dout):
        x, w_up, w_down, w_gate, g, u = ctx.saved_tensors
        return ops.swiglu_backward(dout.to(torch.bfloat16).contiguous(), x, w_up, w_down, w_gate, g=g, u=u)


def swiglu(x, w_up, w_down, w_gate):
    """Differentiable ``kda.swiglu`` (bf16): the forward (``kda.swiglu_gu``) keeps
    g and u, the gradients come from ``kda.swiglu_backward`` on them."""
    return _SwiGLU.apply(x, w_up, w_down, w_gate)


class _GQA(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, rope_theta):
        # the forward keeps its output and row log2-sum-exp, so the backward
        # does not run it again
        out, lse = ops.gqa_full_lse(q, k, v, causal=causal, rope_theta=rope_theta)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.causal, ctx.rope_theta = bool(causal), rope_theta
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = ops.gqa_full_backward(dout.to(torch.bfloat16).contiguous(), q, k, v, causal=ctx.causal,
                                           rope_theta=ctx.rope_theta, fwd_out=out, lse=lse)
        return dq, dk, dv, None, None


def gqa_full(q, k, v, causal=False, rope_theta=None):
    """Differentiable ``kda.gqa_full`` (bf16; output in the reference order
    (B, QH, S, D)): the forward keeps its row log2-sum-exp, the gradients come
    from ``kda.gqa_full_backward`` on the saved forward."""
    return _GQA.apply(q, k, v, causal, rope_theta)


class _FirstOnly(torch.autograd.Function):
    """The first n of ``tensors``, a backward's gradients, unchanged; the others are
    what they were computed from.  Differentiating them again raises."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tensors[:n]

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("kda.autograd: second derivatives of this operator are not implemented")


def _first_only(grads, *computed_from):
    """With create_graph=True the gradients become part of a graph; the kernels are
    not, so a term that goes through them would be left out without a word."""
    return _FirstOnly.apply(len(grads), *grads, *computed_from) if torch.is_grad_enabled() else grads


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, gq, gk, table, positions, eps):
        ctx.save_for_backward(q, k, gq, gk, table, positions)
        ctx.eps = float(eps)
        return ops.qk_norm_rope(q, k, gq, gk, table, positions=positions, eps=eps)

    @staticmethod
    def backward(ctx, dq, dk):
        q, k, gq, gk, table, positions = ctx.saved_tensors
        grads = ops.qk_norm_rope_backward(dq.to(q.dtype).contiguous(), dk.to(q.dtype).contiguous(), q, k, gq, gk,
                                          table, positions=positions, eps=ctx.eps)
        return (*_first_only(grads, dq, dk, q, k, gq, gk), None, None, None)


def qk_norm_rope(q, k, gq, gk, table, *, positions=None, eps=1e-6):
    """Differentiable ``kda.qk_norm_rope``: gradients for q, k, gq and gk come
    from ``kda.qk_norm_rope_backward``; second derivatives raise."""
    return _QKNormRope.apply(q, k, gq, gk, table, positions, eps)


class _GQAWindow(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks):
        out, lse = ops.gqa_window_lse(q, k, v, window, sinks)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.window, ctx.sinks = int(window), int(sinks)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        grads = ops.gqa_window_backward(dout.to(torch.bfloat16).contiguous(), q, k, v, out, lse, ctx.window, ctx.sinks)
        return (*_first_only(grads, dout, q, k, v), None, None)


def gqa_window(q, k, v, window, sinks=0):
    """Differentiable ``kda.gqa_window`` (bf16): the forward keeps its row
    log2-sum-exp, the gradients come from ``kda.gqa_window_backward``; second
    derivatives raise."""
    return _GQAWindow.apply(q, k, v, window, sinks)
