"""Root-mean-square norm with the residual's addition, for the blocks around
the attention (the reference's module wrapper, benchmarks/
based_attention_benchmark.py:24-69, has the projections without a norm).

* ``rms_norm(x, weight=None, residual=None, eps=1e-6)`` -- y, or with a residual
  (y, x + residual), differentiable in x, weight and residual;
* ``rms_norm_fp8(x, weight=None, residual=None, eps=1e-6, group_size=None)`` --
  the same with y held in e4m3 and fp32 scales, ahead of an 8-bit product;
* ``ref_rms_norm(x, weight=None, residual=None, eps=1e-6)`` -- the formula in
  plain PyTorch, for comparisons only; no CUDA path calls it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops


def ref_rms_norm(x, weight=None, residual=None, eps=1e-6):
    """(y, x + residual) in the inputs' dtype."""
    s = x if residual is None else x + residual
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight), s


def _gradients(ctx, d_y, d_sum=None):
    s, weight, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    if d_y is None:  # only the sum was used
        d_w = torch.zeros_like(weight) if need[1] else None
        return d_sum if need[0] else None, d_w, d_sum if need[2] else None, None
    d_s, d_w = ops.rms_norm_backward(s, weight, rstd, d_y, d_sum, want_d_weight=need[1])
    return d_s if need[0] else None, d_w, d_s if need[2] else None, None


_gradients_once = once_differentiable(_gradients)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, rstd = ops.rms_norm(x, weight, residual, eps, want_rstd=True)
        ctx.save_for_backward(x if residual is None else total, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, *grads):
        # (gradients of gradients are refused; the check costs 4 us elsewhere)
        if torch.is_grad_enabled():
            return _gradients_once(ctx, *grads)
        return _gradients(ctx, *grads)


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """Root-mean-square norm of the rows of x (..., d) on the sm_100a kernel.

    x, residual: float32 or bfloat16, any strides with a dense last dimension
    (up to three leading dimensions are read in place); weight: (d,) fp32 or
    bf16, or None for ones; d <= 16384.  Statistics in fp32.  Returns y
    (contiguous, in x.dtype), or with ``residual`` the pair (y, x + residual),
    where y is normed from the unrounded sum.  Differentiable once, backward
    (forward mode is refused).  The same call gives the same bits; a row's last
    bit may go by the number of rows."""
    ops.check_tangents(x, weight, residual)
    if torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, residual)):
        return _RmsNorm.apply(x, weight, residual, float(eps))
    y, total, _ = ops.rms_norm(x, weight, residual, eps)
    return y if residual is None else (y, total)


def rms_norm_fp8(x, weight=None, residual=None, eps=1e-6, group_size=None):
    """``rms_norm`` with its output in e4m3 (inference: no gradient).

    Returns (y, scales), or with ``residual`` (y, scales, x + residual): y
    float8_e4m3fn like x, scales fp32 (..., d / group_size) with y * scale the
    normed value; one scale per row without ``group_size``, else per 16, 32,
    64, 128 or 256 neighbours.  A scale is max(amax, 2^-96) / 448."""
    ops.check_tangents(x, weight, residual)
    y, scales, total = ops.rms_norm_fp8(x, weight, residual, eps, group_size)
    return (y, scales) if residual is None else (y, scales, total)
