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

import operator

import torch

from .._torch_binding import module, silu
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


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, eps=1e-5):
    """Group norm of the channels of x (..., channels) on the sm_100a kernel.

    x, gate: float32 or bfloat16, alike, any strides with a dense last dimension
    (up to two leading dimensions are read in place).  ``groups`` divides the
    channels into neighbours of up to 8192; ``weight`` and ``bias``: (channels,),
    fp32 or in x.dtype, or None for ones and zeros.  ``activation``: None or
    "silu", applied to the gate where there is one, else to the normed value.
    Statistics in fp32, the variance from squared differences, the activation's
    sigmoid to 2^-20 (0 below 2^-126).  Returns y
    (contiguous, in x.dtype).  Differentiable once, backward (forward mode is
    refused); the gradients of weight and bias are summed in a fixed order."""
    check_tangents(x, weight, bias, gate)
    return module().group_norm(x, operator.index(groups), weight, bias, gate, silu(activation),
                               float(eps))
