"""BASED attention modules: q, k, v, o projections around one attention call.

Same classes, constructor arguments and forward as the reference's module
wrappers (benchmarks/based_attention_benchmark.py:24-69):

* ``TrainiumBasedLinearAttention(dim, heads=8, eps=1e-6)`` -- the reference
  path: ``ref_based_attn`` in plain PyTorch between the projections (for
  comparisons; it materialises the (t, t) score matrix).
* ``TrainiumBasedLinearAttentionNKI(dim, heads=8, eps=1e-6, window_size=None)``
  -- the kernel path: ``solution_nki`` (the parallel BASED kernel) as in the
  reference; ``attention="auto"`` uses ``solution`` instead (parallel or
  chunked by the measured crossover), ``window_size`` adds the
  sliding-window term (the full BASED layer, ``based_layer``), and
  ``pre_norm`` puts the root-mean-square norm with the residual stream ahead
  of the projections (``rms_norm``).
* ``DecayLinearAttention(dim, heads=8, ...)`` -- the same projections around
  linear attention with a decay for each head (``decay_linear_attention``) and
  a norm of each head's output, trainable, with ``step`` for single tokens.

The projections are ``nn.Linear`` layers without bias (cuBLAS GEMMs); the
attention runs on the library's sm_100a kernels, which fail loudly when the
CUDA library is missing.  Head layout as the reference: ``(b, t, dim)`` ->
``(b, heads, t, dim // heads)`` and back.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from .based_layer import based_layer
from .decay_attention import decay_linear_attention, decay_linear_attention_step
from .pytorch_attention import ref_based_attn, solution, solution_nki
from .rms_norm import rms_norm


class _Projections(nn.Module):
    def __init__(self, dim: int, heads: int, eps: float):
        super().__init__()
        assert dim % heads == 0
        self.num_heads = heads
        self.head_dim = dim // heads
        self.eps = eps
        self.q_proj = nn.Linear(dim, dim, bias=False)
        self.k_proj = nn.Linear(dim, dim, bias=False)
        self.v_proj = nn.Linear(dim, dim, bias=False)
        self.o_proj = nn.Linear(dim, dim, bias=False)

    def _heads(self, proj: nn.Linear, x: torch.Tensor) -> torch.Tensor:
        b, t, _ = x.size()
        return proj(x).view(b, t, self.num_heads, self.head_dim).transpose(1, 2)

    def _attend(self, q, k, v):
        raise NotImplementedError

    def forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
        b, t, _ = hidden_states.size()
        q = self._heads(self.q_proj, hidden_states)
        k = self._heads(self.k_proj, hidden_states)
        v = self._heads(self.v_proj, hidden_states)
        y = self._attend(q, k, v)
        y = y.transpose(1, 2).reshape(b, t, -1)
        return self.o_proj(y.to(hidden_states.dtype))


class TrainiumBasedLinearAttention(_Projections):
    """BASED attention module, reference path (``ref_based_attn``)."""

    def __init__(self, dim: int, heads: int = 8, eps: float = 1e-6):
        super().__init__(dim, heads, eps)

    def _attend(self, q, k, v):
        return ref_based_attn(q, k, v, eps=self.eps)


class TrainiumBasedLinearAttentionNKI(_Projections):
    """BASED attention module on the sm_100a kernels.

    ``attention``: "parallel" (``solution_nki``, the reference's call) or
    "auto" (``solution``).  ``window_size``: if set, the full BASED layer
    (linear attention + sliding-window softmax over the last ``window_size``
    keys) replaces the linear attention.  ``pre_norm``: the hidden states (plus
    ``residual``, if given) are normed ahead of the projections; the call then
    returns (output, residual stream), the second being the sum that the next
    block adds this block's output to.
    """

    def __init__(self, dim: int, heads: int = 8, eps: float = 1e-6,
                 window_size: int | None = None, attention: str = "parallel",
                 pre_norm: bool = False):
        super().__init__(dim, heads, eps)
        if attention not in ("parallel", "auto"):
            raise ValueError("attention must be 'parallel' or 'auto'")
        if window_size is not None and int(window_size) < 1:
            raise ValueError("window_size must be >= 1")
        self.window_size = window_size
        self.attention = attention
        self.norm_weight = nn.Parameter(torch.ones(dim)) if pre_norm else None

    def forward(self, hidden_states: torch.Tensor, residual: torch.Tensor | None = None):
        if self.norm_weight is None:
            if residual is not None:
                raise ValueError("residual needs pre_norm=True")
            return super().forward(hidden_states)
        normed, stream = _pre_norm(hidden_states, residual, self.norm_weight, self.eps)
        return super().forward(normed), stream

    def _attend(self, q, k, v):
        if self.window_size is not None:
            return based_layer(q, k, v, window_size=self.window_size, eps=self.eps)
        if self.attention == "auto":
            return solution(q, k, v, eps=self.eps)
        return solution_nki(q, k, v, eps=self.eps)


def _pre_norm(hidden_states, residual, weight, eps):
    """(norm of hidden_states + residual, the sum itself)."""
    if residual is None:
        return rms_norm(hidden_states, weight, eps=eps), hidden_states
    return rms_norm(hidden_states, weight, residual=residual, eps=eps)


class DecayLinearAttention(_Projections):
    """Block of linear attention with a decay for each head, on the sm_100a kernels.

    norm (with the residual stream) -> q, k, v projections -> decayed linear
    attention -> norm of each head's output -> output projection.  The heads
    are read as the projections leave them and the heads' norm writes
    (b, t, dim) rows: no transposed copies.  ``log_decay``: fp32 (heads,), by
    default the geometric slopes -2^(-8 i / heads), i = 1 .. heads; a buffer,
    not trained.  The projections and norms are; gradients run through the
    operators' own backward kernels.

    ``forward(x, residual=None, state=None, return_state=False)`` -> (output,
    residual stream[, state]) for a prompt, or the next piece of one with
    ``state``; ``step(x, state, residual=None)`` -> (output, residual stream)
    for one token per sequence (x: (b, dim)), ``state`` (fp32 (b, heads,
    head_dim, head_dim), zeros for a new sequence) updated in place.
    """

    def __init__(self, dim: int, heads: int = 8, eps: float = 1e-6, log_decay=None):
        super().__init__(dim, heads, eps)
        if self.head_dim > 128:
            raise ValueError(f"head dim {self.head_dim} > 128")
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.head_norm_weight = nn.Parameter(torch.ones(self.head_dim))
        if log_decay is None:
            log_decay = -torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads)
        log_decay = torch.as_tensor(log_decay, dtype=torch.float32).detach().clone()
        if tuple(log_decay.shape) != (heads,):
            raise ValueError(f"log_decay must be ({heads},), got {tuple(log_decay.shape)}")
        self.register_buffer("log_decay", log_decay)

    def _apply(self, fn, recurse=True):
        # the decay moves with the module but keeps its fp32 values when that is cast
        kept = self.log_decay
        super()._apply(fn, recurse)
        if kept.is_meta or self.log_decay.is_meta:
            self.log_decay = self.log_decay.float()
        else:
            self.log_decay = kept.to(self.log_decay.device)
        return self

    def _finish(self, y: torch.Tensor) -> torch.Tensor:
        """Heads' norm and output projection of y (..., heads, head_dim)."""
        y = rms_norm(y, self.head_norm_weight, eps=self.eps)
        return self.o_proj(y.flatten(-2))

    def forward(self, hidden_states: torch.Tensor, residual: torch.Tensor | None = None,
                state: torch.Tensor | None = None, return_state: bool = False):
        x, stream = _pre_norm(hidden_states, residual, self.norm_weight, self.eps)
        got = decay_linear_attention(
            self._heads(self.q_proj, x), self._heads(self.k_proj, x), self._heads(self.v_proj, x),
            self.log_decay, initial_state=state, return_state=return_state)
        y, end = got if return_state else (got, None)
        out = self._finish(y.transpose(1, 2))
        return (out, stream, end) if return_state else (out, stream)

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, state: torch.Tensor,
             residual: torch.Tensor | None = None):
        x, stream = _pre_norm(hidden_states, residual, self.norm_weight, self.eps)
        b = x.shape[0]
        q, k, v = (p(x).view(b, self.num_heads, self.head_dim)
                   for p in (self.q_proj, self.k_proj, self.v_proj))
        return self._finish(decay_linear_attention_step(q, k, v, self.log_decay, state)), stream
