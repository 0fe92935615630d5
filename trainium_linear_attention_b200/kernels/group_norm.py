"""Group norm of each token's channels with an activation or an activated gate,
for the outputs of heads (the reference's module wrapper, benchmarks/
based_attention_benchmark.py:24-69, has them without a norm).

    z = (x - mean) / sqrt(var + eps) * weight + bias     over each group of a token
    y = act(z), or with a gate  z * act(gate)

The statistics are a token's own: a causal model's tokens may not see one another.

* ``group_norm(x, groups, ...)`` -- differentiable in all its tensors;
* ``ref_group_norm(x, groups, ...)`` -- the formula in plain PyTorch, for
  comparisons only; no CUDA path calls it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops_recurrent as ops
from ..ops import check_tangents


def ref_group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, eps=1e-5):
    """The formula in the inputs' dtype."""
    g = x.unflatten(-1, (groups, -1))
    g = g - g.mean(-1, keepdim=True)
    z = (g / torch.sqrt(g.square().mean(-1, keepdim=True) + eps)).flatten(-2)
    z = z if weight is None else z * weight
    z = z if bias is None else z + bias
    act = (lambda v: v) if activation is None else torch.nn.functional.silu
    return act(z) if gate is None else z * act(gate)


def _gradients(ctx, d_out):
    x, weight, bias, gate, stats = ctx.saved_tensors
    if d_out is None:
        return (None,) * 7
    need = ctx.needs_input_grad
    dx, d_gate, d_weight, d_bias = ops.group_norm_backward(
        x, ctx.groups, weight, bias, gate, ctx.activation, stats, d_out,
        want_d_affine=need[2] or need[3])
    return (dx if need[0] else None, None, d_weight if need[2] else None,
            d_bias if need[3] else None, d_gate if need[4] else None, None, None)


_gradients_once = once_differentiable(_gradients)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, gate, activation, eps):
        out, stats = ops.group_norm(x, groups, weight, bias, gate, activation, eps,
                                    want_stats=True)
        ctx.save_for_backward(x, weight, bias, gate, stats)
        ctx.groups, ctx.activation = groups, activation
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, *grads):
        # (gradients of gradients are refused; the check costs 4 us elsewhere)
        if torch.is_grad_enabled():
            return _gradients_once(ctx, *grads)
        return _gradients(ctx, *grads)


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, eps=1e-5):
    """Group norm of the channels of x (..., channels) on the sm_100a kernel.

    x, gate: float32 or bfloat16, alike, any strides with a dense last dimension
    (up to two leading dimensions are read in place).  ``groups`` divides the
    channels into neighbours of up to 8192; ``weight`` and ``bias``: (channels,),
    fp32 or in x.dtype, or None for ones and zeros.  ``activation``: None or
    "silu", applied to the gate where there is one, else to the normed value.
    Statistics in fp32, the variance from squared differences.  Returns y
    (contiguous, in x.dtype).  Differentiable once, backward (forward mode is
    refused); the gradients of weight and bias are summed in a fixed order."""
    check_tangents(x, weight, bias, gate)
    if torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias, gate)):
        return _GroupNorm.apply(x, groups, weight, bias, gate, activation, float(eps))
    return ops.group_norm(x, groups, weight, bias, gate, activation, float(eps))[0]
