"""Causal convolution of each channel with a few taps, ahead of a recurrence.

    z_t = bias + sum_j weight_j x_{t - taps + 1 + j},   y = z, or silu(z)

* ``causal_conv(x, weight, ...)`` -- a whole prompt (or the next piece of one),
  differentiable in all its inputs;
* ``causal_conv_step(x, weight, state, ...)`` -- one token of every sequence, the
  last tokens kept in ``state``;
* ``ref_causal_conv(x, weight, ...)`` -- the definition in plain PyTorch, for
  comparisons only; no CUDA path calls it.

The reference has no convolution; its module wrapper (benchmarks/
based_attention_benchmark.py:24-69) has the projections that it stands behind.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops_recurrent as ops
from ..ops import check_tangents


def ref_causal_conv(x, weight, bias=None, activation=None, initial_state=None, lengths=None):
    """(output, final state) in the inputs' dtype."""
    b, t, c = x.shape
    taps = weight.shape[1]
    before = x.new_zeros(b, taps - 1, c) if initial_state is None else initial_state
    whole = torch.cat([before, x], 1)
    y = sum(weight[:, j] * whole[:, j:j + t] for j in range(taps))
    y = y if bias is None else y + bias
    y = y if activation is None else torch.nn.functional.silu(y)
    ends = torch.full((b,), t, device=x.device) if lengths is None else lengths.clamp(0, t).long()
    inside = torch.arange(t, device=x.device) < ends[:, None]
    at = ends[:, None] + torch.arange(taps - 1, device=x.device)
    final = whole.gather(1, at[..., None].expand(-1, -1, c))
    return torch.where(inside[..., None], y, torch.zeros_like(y)), final


def _gradients(ctx, d_out, d_state=None):
    x, weight, bias, initial_state, lengths = ctx.saved_tensors
    if d_out is None and d_state is None:
        return (None,) * 7
    if d_out is None:
        d_out = torch.zeros_like(x)
    need = ctx.needs_input_grad
    dx, d_weight, d_bias, d_init = ops.causal_conv_backward(
        x, weight, bias, ctx.activation, initial_state, lengths, d_out, d_state,
        want_d_weight=need[1] or need[2], want_d_initial=need[4])
    return (dx if need[0] else None, d_weight if need[1] else None,
            d_bias if need[2] else None, None, d_init, None, None)


_gradients_once = once_differentiable(_gradients)


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, initial_state, lengths, return_state):
        out, final = ops.causal_conv(x, weight, bias, activation, initial_state, lengths,
                                     return_state)
        ctx.save_for_backward(x, weight, bias, initial_state, lengths)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return (out, final) if return_state else out

    @staticmethod
    def backward(ctx, *grads):
        # (gradients of gradients are refused; the check costs 4 us elsewhere)
        if torch.is_grad_enabled():
            return _gradients_once(ctx, *grads)
        return _gradients(ctx, *grads)


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, return_state=False,
                lengths=None):
    """Causal convolution of each channel on the sm_100a kernels.

    x: (b, t, channels), float32 or bfloat16, any strides with a dense last
    dimension; ``weight``: (channels, taps), 2 to 4 taps, the last one for the
    token itself; ``bias``: (channels,); both fp32 or in x.dtype, and alike.
    ``activation``: None or "silu".  ``initial_state``: (b, taps - 1, channels)
    in x.dtype, the tokens before the first, oldest first (zeros without it).
    ``lengths``: as for ``gated_recurrence``.

    Returns (b, t, channels) in x.dtype, contiguous, or with ``return_state``
    also the last taps - 1 tokens.  Sums in fp32.  Differentiable once, backward,
    in x, weight, bias and ``initial_state`` (forward mode is refused); the
    gradients of weight and bias are summed in a fixed order."""
    check_tangents(x, weight, bias, initial_state)
    if torch.is_grad_enabled() and any(
            isinstance(v, torch.Tensor) and v.requires_grad
            for v in (x, weight, bias, initial_state)):
        return _CausalConv.apply(x, weight, bias, activation, initial_state, lengths,
                                 bool(return_state))
    out, final = ops.causal_conv(x, weight, bias, activation, initial_state, lengths, return_state)
    return (out, final) if return_state else out


def causal_conv_step(x, weight, state, bias=None, activation=None):
    """One token of every sequence on the sm_100a kernel.

    x: (b, channels); ``state`` ((b, taps - 1, channels) in x.dtype, as
    ``causal_conv`` returns it) loses its oldest token and gains x, in place.
    Returns (b, channels) in x.dtype; no gradient."""
    check_tangents(x, weight, state, bias)
    return ops.causal_conv_step(x, weight, state, bias, activation)
