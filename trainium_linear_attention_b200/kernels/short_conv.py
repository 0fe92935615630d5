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

from .._torch_binding import module, silu
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
    also the last taps - 1 tokens.  Sums in fp32, the activation's sigmoid to 2^-20
    (0 below 2^-126).  Differentiable once, backward,
    in x, weight, bias and ``initial_state`` (forward mode is refused); the
    gradients of weight and bias are summed in a fixed order."""
    check_tangents(x, weight, bias, initial_state)
    return module().causal_conv(x, weight, bias, silu(activation), initial_state, lengths,
                                bool(return_state))


def causal_conv_step(x, weight, state, bias=None, activation=None):
    """One token of every sequence on the sm_100a kernel.

    x: (b, channels); ``state`` ((b, taps - 1, channels) in x.dtype, as
    ``causal_conv`` returns it) loses its oldest token and gains x, in place.
    Returns (b, channels) in x.dtype; no gradient."""
    check_tangents(x, weight, state, bias)
    return module().causal_conv_step(x, weight, state, bias, silu(activation))
