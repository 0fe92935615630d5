"""Linear attention with a decay for each head: prompts, training, single tokens.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t

the recurrence of the reference's chunked kernel (kernels/
nki_attention_chunked.py:20-113) with identity features and a forgetting
factor, in the three forms a model needs:

* ``decay_linear_attention(q, k, v, log_decay, ...)`` -- a whole prompt (or the
  next piece of one), differentiable in q, k, v and the initial state;
* ``decay_linear_attention_step(q, k, v, log_decay, state, ...)`` -- one token
  of every sequence, the state updated in place;
* ``ref_decay_attn(q, k, v, log_decay, ...)`` -- the definition in plain
  PyTorch, for comparisons only; no CUDA path calls it.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import ops


def ref_decay_attn(q, k, v, log_decay, scale=None, initial_state=None):
    """The dense definition in the inputs' dtype: (output, final state).
    Materialises the (t, t) weights."""
    t, d = q.shape[-2:]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    g = log_decay.to(q.dtype).view(-1, 1, 1)
    i = torch.arange(t, device=q.device, dtype=q.dtype)
    lag = i[:, None] - i[None, :]
    weight = torch.where(lag > 0, torch.exp(g * lag.clamp(min=1)), (lag == 0).to(q.dtype))
    out = (q @ k.transpose(-2, -1) * weight) @ v
    left = t - 1 - i
    into = torch.where(left > 0, torch.exp(g * left.clamp(min=1)), torch.ones_like(g * left))
    state = (k * into.transpose(-2, -1)).transpose(-2, -1) @ v
    if initial_state is not None:
        out = out + torch.exp(g * (i[:, None] + 1)) * (q @ initial_state)
        state = state + (torch.exp(g * t) if t else 1.0) * initial_state
    return out * scale, state


def _gradients(ctx, d_out, d_state=None):
    q, k, v, log_decay, initial_state = ctx.saved_tensors
    if d_out is None and d_state is None:
        return (None,) * 7
    if d_out is None:
        d_out = torch.zeros_like(v)
    need = ctx.needs_input_grad
    dq, dk, dv, d0 = ops.decay_attention_backward(
        q, k, v, log_decay, d_out, scale=ctx.scale, initial_state=initial_state,
        d_state=d_state, want_d_initial=need[4])
    return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
            None, d0, None, None)


_gradients_once = once_differentiable(_gradients)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, scale, return_state):
        got = ops.decay_attention(q, k, v, log_decay, scale=scale, initial_state=initial_state,
                                  return_state=return_state)
        ctx.save_for_backward(q, k, v, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return got

    @staticmethod
    def backward(ctx, *grads):
        # (gradients of gradients are refused; the check costs 4 us elsewhere)
        if torch.is_grad_enabled():
            return _gradients_once(ctx, *grads)
        return _gradients(ctx, *grads)


def decay_linear_attention(q, k, v, log_decay, scale=None, initial_state=None,
                           return_state=False):
    """Causal linear attention with a decay for each head on the sm_100a kernels.

    q, k: (b, h, t, d_qk); v: (b, h, t, d_v), float32 or bfloat16, widths up to
    128, b * h up to 65535, any strides with a dense last dimension (a
    projection's transposed heads are read in place, and the output is laid
    out as v).  ``log_decay``:
    float32 (h,), <= 0, a constant (one that requires a gradient is refused
    where gradients are recorded).  ``scale`` defaults to 1/sqrt(d_qk).
    ``initial_state``: fp32 (b, h, d_qk, d_v), the state before the first
    token.  Returns (b, h, t, d_v) in q.dtype, or with ``return_state`` also
    the fp32 state after the last token.  Differentiable once, backward, in q, k,
    v and ``initial_state``; forward mode is refused.

    Sequences of different lengths in one batch: pad them on the left with zero
    k (a zero token adds nothing to the zero state, and ends where the others
    do), or leave out what the right padding returns; a value that is not
    finite reaches the outputs of its own tile of 128 tokens, so padding should
    be finite.  bf16 runs on tensor cores: the weights of a tile's values and
    the state's read-out are rounded to bf16, the state is carried in fp32.  A
    final state that is returned, and the gradient of ``initial_state``, are
    exact to fp32; where neither is asked for the state is fed with products of
    two bf16 terms (2^-14.8 at most, 2^-17.8 in the mean square), so an output's
    last bit may go by ``return_state``."""
    ops.check_tangents(q, k, v, log_decay, initial_state)
    if torch.is_grad_enabled() and any(
            isinstance(x, torch.Tensor) and x.requires_grad for x in (q, k, v, initial_state)):
        ops._check_constant(log_decay)  # (gradients are off inside the function)
        return _DecayAttention.apply(q, k, v, log_decay, initial_state, scale, bool(return_state))
    return ops.decay_attention(q, k, v, log_decay, scale=scale, initial_state=initial_state,
                               return_state=return_state)


def decay_linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One token of every sequence on the sm_100a kernel.

    q, k: (b, h, d_qk); v: (b, h, d_v).  ``state`` (fp32 (b, h, d_qk, d_v), as
    ``decay_linear_attention`` returns it) is updated in place.  Returns
    (b, h, d_v) in q.dtype; no gradient."""
    ops.check_tangents(q, k, v, log_decay, state)
    return ops.decay_attention_step(q, k, v, log_decay, state, scale=scale)
