"""The linear layer ``y = act(x w^T + bias) + residual`` and its backward pass over libqrb200
(include/qrb200_nn.h): tensor-core products with everything else in their epilogue.

float32 (with float32 accuracy), bfloat16 and float16; sums are fp32 and each result is rounded
once.  All work is enqueued on torch's current stream of x's device; inputs are not modified, and a
backward pass that had kept what ``out`` names raises, as after torch's own in-place operations; wrong
arguments raise TypeError or ValueError before anything is enqueued; results repeat.
"""
from __future__ import annotations

import torch

from .delta import _refuse_capture, _wants_grad
from .ops import _fast


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        y, pre = _fast().linear_forward(x, w, bias, activation, residual, activation != "none", None)
        ctx.save_for_backward(x, w, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("linear", "linear_backward")
        x, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _fast().linear_backward(dy, x, w, ctx.activation, pre, need[0], need[1], need[2])
        return dx, dw, db, dy if need[3] else None, None


def linear(x, w, bias=None, *, activation="none", residual=None, return_pre=False, out=None):
    """``act(x w^T + bias) + residual`` for x (..., k), w (n, k), bias (n,) and residual (..., n), all of one
    type; ``activation`` is "none", "relu", "silu" or "gelu" (the exact, erf form).

    ``return_pre`` also returns ``x w^T + bias`` rounded to the type, which ``linear_backward`` needs for an
    activation.  ``out`` takes the result; it may be ``residual`` itself, and overlap no input otherwise.  Any
    strides: rows that are not dense are copied, and rows that are not 16-byte aligned are laid out in scratch
    memory first.
    Differentiable with respect to x, w, bias and residual, once; forward-mode tangents are refused
    (NotImplementedError).
    """
    if _wants_grad(x, w, bias, residual, out):
        if out is not None or return_pre:
            raise ValueError("out and return_pre are not supported where out or an input requires gradients")
        _refuse_capture("linear", "linear_backward")
        return _Linear.apply(x, w, bias, residual, activation)
    y, pre = _fast().linear_forward(x, w, bias, activation, residual, return_pre, out)
    return (y, pre) if return_pre else y


def linear_backward(dy, x, w, *, activation="none", pre=None, with_bias=False, with_dx=True, with_dw=True):
    """``(dx, dw, dbias)`` of ``linear`` for the gradient dy of its result; those not asked for are None.

    ``pre`` is what ``linear(..., return_pre=True)`` returned (needed with an activation only).  The gradient
    of the residual is dy itself.  With 16-bit types dp = dy act'(pre) is rounded to the type before its two
    products, which is as much again as rounding dx and dw (in bf16 2.3e-3 of error in place of 1.7e-3); dbias
    is summed before that, in fp32.  Records no gradients of its own.  Can be captured into a CUDA graph.
    """
    return _fast().linear_backward(dy, x, w, activation, pre, with_dx, with_dw, with_bias)
