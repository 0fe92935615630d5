"""Block of a gated linear recurrence, beside those of the linear attentions
(``based_module``), with the constructor arguments and forward of those (the
reference's module wrappers, benchmarks/based_attention_benchmark.py:24-69, and
the norms around them).

The projections are ``nn.Linear`` layers without bias (cuBLAS GEMMs); all that
lies between them runs on the library's sm_100a kernels, which fail loudly when
the CUDA library is missing.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from .based_module import _pre_norm
from .gated_recurrence import gated_recurrence, gated_recurrence_step
from .group_norm import group_norm
from .short_conv import causal_conv, causal_conv_step


class GatedRecurrence(nn.Module):
    """norm (with the residual stream) -> input and output-gate projection ->
    short convolution -> recurrence and input gates -> gated linear recurrence ->
    norm of each head's channels times the activated output gate -> output
    projection.  ``dim`` channels in ``heads`` groups of the norm.

    ``log_decay = -softplus(decay)``, ``decay`` (dim,) trained; it starts where
    half-open gates keep 0.9 to 0.999 of the state for each token.

    ``forward(x, residual=None, state=None, return_state=False, lengths=None)`` ->
    (output, residual stream[, state]) for a prompt, or the next piece of one with
    ``state``; ``lengths`` (b,): the tokens of each sequence of a right-padded
    batch, for the state that is returned.  ``step(x, state, residual=None)`` ->
    (output, residual stream) for one token per sequence (x: (b, dim)), ``state``
    updated in place.  ``state``: the last taps - 1 inputs of the convolution
    (b, taps - 1, dim) and the recurrence's fp32 (b, dim); ``empty_state(b)`` is that
    of a new sequence (called under the autocast, if any, that the block is called under:
    the convolution's inputs have the projections' type).
    """

    def __init__(self, dim: int, heads: int = 8, eps: float = 1e-6, taps: int = 4):
        super().__init__()
        if dim % heads:
            raise ValueError(f"{heads} heads do not divide {dim} channels")
        if taps not in (2, 3, 4):
            raise ValueError(f"taps must be 2, 3 or 4, got {taps}")
        self.num_heads, self.eps, self.taps = heads, eps, taps
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.in_proj = nn.Linear(dim, 2 * dim, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(dim, taps).uniform_(-1, 1) * taps ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(dim))
        self.gate_proj = nn.Linear(dim, 2 * dim, bias=False)
        keep = 0.9 + 0.099 * torch.arange(dim) / max(dim - 1, 1)
        self.decay = nn.Parameter(torch.log(torch.expm1(-2.0 * torch.log(keep))))
        self.head_norm_weight = nn.Parameter(torch.ones(dim))
        self.head_norm_bias = nn.Parameter(torch.zeros(dim))
        self.o_proj = nn.Linear(dim, dim, bias=False)

    def _log_decay(self) -> torch.Tensor:
        return -nn.functional.softplus(self.decay.float())

    def _finish(self, h: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        return self.o_proj(group_norm(h, self.num_heads, self.head_norm_weight,
                                      self.head_norm_bias, gate=gate, activation="silu",
                                      eps=self.eps))

    def empty_state(self, batch: int):
        w = self.conv_weight
        dtype = (torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda")
                 else self.in_proj.weight.dtype)
        return (w.new_zeros(batch, self.taps - 1, w.shape[0], dtype=dtype),
                torch.zeros(batch, w.shape[0], device=w.device))

    def forward(self, hidden_states: torch.Tensor, residual: torch.Tensor | None = None,
                state=None, return_state: bool = False, lengths: torch.Tensor | None = None):
        x, stream = _pre_norm(hidden_states, residual, self.norm_weight, self.eps)
        x, out_gate = self.in_proj(x).chunk(2, -1)
        before, h0 = (None, None) if state is None else state
        x, tail = causal_conv(x, self.conv_weight, self.conv_bias, "silu", before,
                              return_state=True, lengths=lengths)
        gate, input_gate = self.gate_proj(x).chunk(2, -1)
        h, end = gated_recurrence(x, gate, self._log_decay(), input_gate, h0, return_state=True,
                                  lengths=lengths)
        out = self._finish(h, out_gate)
        return (out, stream, (tail, end)) if return_state else (out, stream)

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, state, residual: torch.Tensor | None = None):
        x, stream = _pre_norm(hidden_states, residual, self.norm_weight, self.eps)
        x, out_gate = self.in_proj(x).chunk(2, -1)
        tail, h = state
        x = causal_conv_step(x, self.conv_weight, tail, self.conv_bias, "silu")
        gate, input_gate = self.gate_proj(x).chunk(2, -1)
        y = gated_recurrence_step(x, gate, h, self._log_decay(), input_gate)
        return self._finish(y, out_gate), stream
