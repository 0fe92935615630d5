"""Gated linear recurrence of each channel: prompts, training, single tokens.

    h_t = a_t h_{t-1} + beta_t u_t x_t,   u = sigmoid(input_gate), or 1 without one
    with log_decay:  a = exp(log_decay * sigmoid(gate)),  beta = sqrt(1 - a^2)
    without:         a = sigmoid(gate),                   beta = 1 - a

Beside the linear attentions, whose state is a matrix for each head (the
reference's chunked kernel, kernels/nki_attention_chunked.py:20-113), this is the
mixer whose state is one number for each channel and whose decay goes by the
token:

* ``gated_recurrence(x, gate, ...)`` -- a whole prompt (or the next piece of
  one), differentiable in all its inputs;
* ``gated_recurrence_step(x, gate, state, ...)`` -- one token of every sequence,
  the state updated in place;
* ``ref_gated_recurrence(x, gate, ...)`` -- the definition in plain PyTorch, for
  comparisons only; no CUDA path calls it.
"""

from __future__ import annotations

import torch

from .._torch_binding import module
from ..ops import check_tangents


def ref_gated_recurrence(x, gate, log_decay=None, input_gate=None, initial_state=None,
                         lengths=None):
    """The definition, token by token, in the inputs' dtype: (output, final state)."""
    b, t, c = x.shape
    a = torch.sigmoid(gate)
    if log_decay is None:
        beta = torch.sigmoid(-gate)
    else:
        log_a = log_decay.to(x.dtype) * a
        a, beta = log_a.exp(), torch.sqrt(-torch.expm1(2 * log_a))
    add = beta * x if input_gate is None else beta * torch.sigmoid(input_gate) * x
    h = x.new_zeros(b, c) if initial_state is None else initial_state.to(x.dtype)
    outs = [x.new_zeros(b, 0, c)]
    for i, (ai, bi) in enumerate(zip(a.unbind(1), add.unbind(1))):
        new = ai * h + bi
        if lengths is None:
            h = new
            outs.append(h[:, None])
        else:
            inside = (i < lengths)[:, None]
            h = torch.where(inside, new, h)
            outs.append(torch.where(inside, new, torch.zeros_like(new))[:, None])
    return torch.cat(outs, 1), h


def gated_recurrence(x, gate, log_decay=None, input_gate=None, initial_state=None,
                     return_state=False, lengths=None):
    """The recurrence over a whole prompt on the sm_100a kernels.

    x, gate, input_gate: (b, t, channels), float32 or bfloat16, any strides
    with a dense last dimension (slices of one projection are read in place);
    the gates are taken ahead of their sigmoid.  ``log_decay``: fp32
    (channels,), finite and <= 0, the logarithm of the decay of a whole open
    gate.  ``initial_state``: fp32 (b, channels), the state before the first
    token.  ``lengths``: int32 or int64 (b,) on the same device, the tokens of each
    sequence of a right-padded batch (taken into [0, t]): what lies behind them
    is not read, its outputs and gradients are zero, and the final state is the
    one after the sequence's last token.

    Returns (b, t, channels) in x.dtype, contiguous, or with ``return_state``
    also the fp32 state after the last token.  Differentiable once, backward,
    in x, the gates, ``log_decay`` and ``initial_state`` (forward mode is
    refused); the gradient of ``log_decay`` is summed in a fixed order, and is
    not defined where it is 0.  The state is carried in fp32 as h + (a - 1) h +
    b with a - 1 to a relative 2^-22: a slow decay is as exact as the state's own
    rounding, half a step a token.  In fp32 too reciprocals and the root are within
    an ulp, not correctly rounded; a sigmoid below 2^-126 is 0, and where 1 - a^2 is
    below 2^-100 (gates under about -70) a token's part is off by up to 4e-19 of
    u x."""
    check_tangents(x, gate, log_decay, input_gate, initial_state)
    return module().gated_recurrence(x, gate, log_decay, input_gate, initial_state, lengths,
                                     bool(return_state))


def gated_recurrence_step(x, gate, state, log_decay=None, input_gate=None):
    """One token of every sequence on the sm_100a kernel.

    x, gate, input_gate: (b, channels); ``state`` (fp32 (b, channels), as
    ``gated_recurrence`` returns it) is updated in place.  Returns (b, channels)
    in x.dtype; no gradient."""
    check_tangents(x, gate, log_decay, input_gate, state)
    return module().gated_recurrence_step(x, gate, state, log_decay, input_gate)
