"""The gated delta rule over libqrb200 (include/qrb200_nn.h).

Per head a state ``S`` (dk x dv) passes through scaled Householder-like transforms, one a token::

    S~_t = exp(g_t) S_{t-1}
    u_t  = beta_t (v_t - S~_t^T k_t)
    S_t  = S~_t + k_t u_t^T
    o_t  = scale S_t^T q_t

``gated_delta_rule`` runs whole sequences in the chunked compact-WY form blocked QR uses for its
reflectors, ``gated_delta_rule_backward`` is its gradient, and ``gated_delta_step`` advances one
token per row for generation.  float32, bfloat16 and float16; states, ``g`` and ``beta`` are
float32.  All work is enqueued on torch's current stream of the inputs' device; wrong arguments raise
TypeError or ValueError before anything is enqueued.  Inputs are not modified, but for the states that
``gated_delta_step`` advances in place and what ``out`` names; a backward pass that had kept a tensor
written so raises, as after torch's own in-place operations.
"""
from __future__ import annotations

import torch

from .ops import _fast

_CAPTURE = ("{} cannot record gradients while a CUDA graph is captured: under torch.no_grad(), capture the "
            "forward call and {} instead")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def _refuse_capture(name: str, backward: str) -> None:
    # Autograd joins the streams its accumulators were made on, which a capture does not survive.
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(_CAPTURE.format(name, backward))


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, scale, seq_offsets):
        ctx.save_for_backward(q, k, v, g, beta, initial_state, seq_offsets)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _fast().delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dfinal_state):
        _refuse_capture("gated_delta_rule", "gated_delta_rule_backward")
        q, k, v, g, beta, initial_state, seq_offsets = ctx.saved_tensors
        if do is None:
            if dfinal_state is None:
                return (None,) * 8
            do = torch.zeros_like(v)
        grads = gated_delta_rule_backward(do, q, k, v, g, beta, scale=ctx.scale, initial_state=initial_state,
                                          seq_offsets=seq_offsets, dfinal_state=dfinal_state)
        return (*grads, None, None)


def gated_delta_rule(q, k, v, g, beta, *, scale=None, initial_state=None, seq_offsets=None, out=None):
    """``(o, final_state)`` of the gated delta rule.

    ``q``, ``k``: (batch, time, heads_k, dk) with dk <= 128; ``v``: (batch, time, heads, dv) with dv <= 256
    and heads a multiple of heads_k (value head h reads q/k head ``h // (heads // heads_k)``); ``g`` (the
    decay's logarithm; -inf empties the state, and what is positive must not add up to 88 or more) and
    ``beta``: (batch, time, heads) float32.  Any strides; tensors whose last dimension is not dense are
    copied.  ``scale`` defaults to dk ** -0.5,
    ``initial_state`` (sequences, heads, dk, dv) float32 to zeros.

    ``seq_offsets`` (sequences + 1, int32 or int64, on the device) packs sequences of different lengths,
    empty ones too, along the time of a batch of one; it starts at 0 and does not decrease.  Rows behind
    the last sequence are not read; their o is 0, or with ``out=(o, final_state)`` left as it was.
    ``out`` takes the results: final_state may be ``initial_state`` itself, but neither may overlap it otherwise,
    nor ``seq_offsets`` or one another.

    Differentiable with respect to q, k, v, g, beta and initial_state (autograd calls
    ``gated_delta_rule_backward``), once; forward-mode tangents are refused (NotImplementedError).  A value that
    is not finite may spoil its sequence from the start of its 64-token chunk on.
    """
    if out is not None and _wants_grad(q, k, v, g, beta, initial_state, *out):
        raise ValueError("out is not supported where it or an input requires gradients")
    if _wants_grad(q, k, v, g, beta, initial_state):
        _refuse_capture("gated_delta_rule", "gated_delta_rule_backward")
        return _GatedDeltaRule.apply(q, k, v, g, beta, initial_state, scale, seq_offsets)
    o, s = (None, None) if out is None else out
    return _fast().delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, o, s)


def gated_delta_rule_backward(do, q, k, v, g, beta, *, scale=None, initial_state=None, seq_offsets=None,
                              dfinal_state=None):
    """``(dq, dk, dv, dg, dbeta, dinitial_state)`` from the gradients of o and (None: zero) final_state.

    The other arguments are those of ``gated_delta_rule``; dinitial_state is None without an initial state.
    The forward recurrence is run again, so nothing has to be kept between the passes.  q/k heads that
    several value heads share get the sum of their gradients, added in head order: results repeat.  dg is the
    difference of sums of o do and v dv over up to 64 tokens and is good to about 1e-6 of those: where a gate is
    nearly closed, its true value (which goes to 0) may be smaller.  A value that is not finite may spoil every
    gradient of its sequence.  Records no gradients of its own.  Can be captured into a CUDA graph.
    """
    return _fast().delta_backward(do, q, k, v, g, beta, scale, initial_state, seq_offsets, dfinal_state)


def gated_delta_step(q, k, v, g, beta, state, *, scale=None, slots=None, state_out=None, out=None):
    """``o`` of one token per row: (batch, heads_k, dk) q and k, (batch, heads, dv) v, (batch, heads) g and
    beta, and a pool ``state`` (slots, heads, dk, dv) float32 whose slots may be strided.

    Row i advances state ``slots[i]`` (int32 on the device; default i) in place, or from ``state`` into the
    same slot of ``state_out``, which may be another pool (other slots of it are left as they are) but must
    not overlap ``state`` otherwise.  ``out`` takes o.  Neither may overlap an input, but out may be ``v``.
    A negative slot marks a padding row: its o is 0.  A slot outside the pool, or one that an earlier row holds,
    is refused: that row's o is NaN and it changes no state.
    """
    return _fast().delta_step(q, k, v, g, beta, state, scale, slots, state_out, out)
