"""Torch-facing calls of the gated linear recurrence, the short convolution and
the group norm (no autograd), beside those of :mod:`.ops` and in their manner:
CUDA tensors in, the kernel enqueued on the current stream of their device, new
outputs returned, failures raised.  The checks of a call are made once for each
signature (shapes, strides, types, devices) and kept under it.
"""

from __future__ import annotations

import ctypes
import operator

import torch

from . import _native as N
from .ops import (_dtype_code, _get_device, _keep, _on_device, _proto, _ptr, _sig, _stream_ptr,
                  _Strides)

_LENGTHS = {torch.int32: 32, torch.int64: 64}


def _check_tensor(t, name, dims):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != len(dims):
        raise ValueError(f"{name} must be ({', '.join(dims)}), got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device}); "
                         "this library has no CPU implementation")
    return _dtype_code(t)


def _check_like(t, name, like):
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} on {like.device}")


def _check_exact(t, name, shape, dtype, device):
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} {shape} on {device}")


def _check_lengths(lengths, batch, device):
    if lengths is None:
        return 0
    if not isinstance(lengths, torch.Tensor):
        raise TypeError("lengths must be a torch.Tensor")
    if (lengths.dtype not in _LENGTHS or tuple(lengths.shape) != (batch,)
            or lengths.device != device):
        raise ValueError(f"lengths must be int32 or int64 ({batch},) on {device}")
    return _LENGTHS[lengths.dtype]


def _check_activation(activation):
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return int(activation is not None)


def _check_affine(weight, bias, names, shape, like):
    """The code of the type that both have; they may be fp32 beside bf16 inputs."""
    for t, name, s in ((weight, names[0], shape), (bias, names[1], shape[:1])):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if tuple(t.shape) != s or t.device != like.device:
            raise ValueError(f"{name} must be {s} on {like.device}")
        _dtype_code(t)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{names[0]} and {names[1]} differ in type: {weight.dtype}, {bias.dtype}")
    given = weight if weight is not None else bias
    return _dtype_code(like if given is None else given)


def _token_strides(t):
    """{batch, tokens} strides of (b, t, c) with a dense last dimension, else None."""
    if t is None:
        return None
    b, n, c = t.shape
    if t.numel() == 0:
        return _Strides(n * c, c)
    sb, st, sc = t.stride()
    if sc != 1 and c > 1:
        return None
    return _Strides(sb if b > 1 else n * c, st if n > 1 else c)


class _TokensPlan:
    """What the calls on (batch, tokens, channels) share."""

    def __init__(self, x, others, names, lengths):
        dims = ("batch", "tokens", "channels")
        code = _check_tensor(x, "x", dims)
        if x.shape[-1] < 1:
            raise ValueError(f"x must be (batch, tokens, channels), got shape {tuple(x.shape)}")
        for t, name in zip(others, names):
            _check_like(t, name, x)
        b, t, c = x.shape
        self.bits = _check_lengths(lengths, b, x.device)
        self.device, self.dtype, self.index = x.device, x.dtype, x.device.index
        self.sizes, self.code = (b, t, c), code
        tensors = (x, *others)
        self.strides = tuple(_token_strides(v) for v in tensors)
        self.copy = tuple(v is not None and s is None for v, s in zip(tensors, self.strides))
        self.any_copy = any(self.copy)
        self.out = _proto((b, t, c), x.dtype, x.device)

    def read(self, tensors):
        return [t.contiguous() if c else t for t, c in zip(tensors, self.copy)]


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _lookup(plans, key_of, make):
    try:
        key = key_of()
        plan = plans.get(key)
    except AttributeError:  # not tensors: the checks say which
        key = plan = None
    return plan if plan is not None else _keep(plans, key, make())


# ---- gated linear recurrence --------------------------------------------------------
class _RecurPlan(_TokensPlan):
    def __init__(self, x, gate, input_gate, log_decay, state, d_state, lengths, d_out):
        super().__init__(x, (gate, input_gate, d_out), ("gate", "input_gate", "d_out"), lengths)
        if gate is None:
            raise TypeError("gate must be a torch.Tensor")
        b, t, c = self.sizes
        _check_exact(log_decay, "log_decay", (c,), torch.float32, x.device)
        _check_exact(state, "initial_state", (b, c), torch.float32, x.device)
        _check_exact(d_state, "d_state", (b, c), torch.float32, x.device)
        self.state = _proto((b, c), torch.float32, x.device)
        self.d_log = _proto((c,), torch.float32, x.device)
        saved, ws = ctypes.c_size_t(0), ctypes.c_size_t(0)
        with _on_device(x.device):
            N.check(N.lib().la_recurrence_plan(b, t, c, ctypes.byref(saved), ctypes.byref(ws)),
                    "la_recurrence_plan")
        self.saved_shape = (saved.value // 4,)
        self.saved = _proto(self.saved_shape, torch.float32, x.device)
        self.ws_bytes = ws.value
        self.workspace = _proto((ws.value,), torch.uint8, x.device)


_recur_plans: dict = {}


def _recur_plan(x, gate, input_gate, log_decay, state, d_state, lengths, d_out):
    args = (x, gate, input_gate, log_decay, state, d_state, lengths, d_out)
    return _lookup(_recur_plans, lambda: tuple(map(_sig, args)), lambda: _RecurPlan(*args))


def gated_recurrence(x, gate, log_decay=None, input_gate=None, initial_state=None, lengths=None,
                     return_state: bool = False, want_saved: bool = False):
    """Forward pass: (out, final state or None, what the gradient needs or None)."""
    plan = _recur_plan(x, gate, input_gate, log_decay, initial_state, None, lengths, None)
    if plan.any_copy:
        x, gate, input_gate, _ = plan.read((x, gate, input_gate, None))
        return gated_recurrence(x, gate, log_decay, input_gate, initial_state, lengths,
                                return_state, want_saved)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return gated_recurrence(x, gate, log_decay, input_gate, initial_state, lengths,
                                    return_state, want_saved)
    log_decay, initial_state, lengths = _dense(log_decay), _dense(initial_state), _dense(lengths)
    out = torch.empty_like(plan.out)
    final = torch.empty_like(plan.state) if return_state else None
    saved = torch.empty_like(plan.saved) if want_saved else None
    xs, gs, us, _ = plan.strides
    st = N.lib().la_recurrence_fwd(
        x.data_ptr(), xs, gate.data_ptr(), gs, _ptr(input_gate), us, _ptr(log_decay),
        _ptr(initial_state), _ptr(lengths), plan.bits, out.data_ptr(), _ptr(final), _ptr(saved),
        *plan.sizes, plan.code, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_recurrence_fwd")
    return out, final, saved


def gated_recurrence_backward(x, gate, log_decay, input_gate, saved, lengths, d_out, d_state=None,
                              want_d_decay: bool = False, want_d_initial: bool = False):
    """Gradients (x, gate, input_gate or None, log_decay or None, initial state
    or None) of ``gated_recurrence`` on the same inputs."""
    plan = _recur_plan(x, gate, input_gate, log_decay, None, d_state, lengths, d_out)
    _check_exact(saved, "saved", plan.saved_shape, torch.float32, plan.device)
    if plan.any_copy:
        x, gate, input_gate, d_out = plan.read((x, gate, input_gate, d_out))
        return gated_recurrence_backward(x, gate, log_decay, input_gate, saved, lengths, d_out,
                                         d_state, want_d_decay, want_d_initial)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return gated_recurrence_backward(x, gate, log_decay, input_gate, saved, lengths,
                                             d_out, d_state, want_d_decay, want_d_initial)
    log_decay, d_state, lengths = _dense(log_decay), _dense(d_state), _dense(lengths)
    dx, d_gate = torch.empty_like(plan.out), torch.empty_like(plan.out)
    d_input = torch.empty_like(plan.out) if input_gate is not None else None
    d_log = workspace = None
    if want_d_decay and log_decay is not None:
        d_log, workspace = torch.empty_like(plan.d_log), torch.empty_like(plan.workspace)
    d_init = torch.empty_like(plan.state) if want_d_initial else None
    xs, gs, us, ds = plan.strides
    st = N.lib().la_recurrence_bwd(
        x.data_ptr(), xs, gate.data_ptr(), gs, _ptr(input_gate), us, _ptr(log_decay),
        saved.data_ptr(), _ptr(lengths), plan.bits, d_out.data_ptr(), ds, _ptr(d_state),
        dx.data_ptr(), d_gate.data_ptr(), _ptr(d_input), _ptr(d_log), _ptr(d_init), *plan.sizes,
        plan.code, _ptr(workspace), plan.ws_bytes, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_recurrence_bwd")
    return dx, d_gate, d_input, d_log, d_init


def _batch_stride(t):
    """The batch stride of (b, c) with a dense last dimension, else None."""
    if t is None:
        return 0
    b, c = t.shape
    if t.stride(1) != 1 and c > 1 and t.numel():
        return None
    return t.stride(0) if b > 1 else c


def _check_step_state(state, shape, dtype, device):
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    _check_exact(state, "state", shape, dtype, device)
    inner, dense = 1, True
    for n, s in zip(shape[:0:-1], state.stride()[:0:-1]):
        dense = dense and (s == inner or n == 1)
        inner *= n
    stride = state.stride(0) if shape[0] > 1 else inner
    if state.numel() and (not dense or stride < inner):
        raise ValueError(f"state needs dense {shape[1:]} entries that do not overlap")
    return max(stride, inner)


class _RecurStepPlan:
    def __init__(self, x, gate, log_decay, input_gate, state):
        self.code = _check_tensor(x, "x", ("batch", "channels"))
        b, c = x.shape
        if c < 1:
            raise ValueError(f"x must be (batch, channels), got shape {tuple(x.shape)}")
        if gate is None:
            raise TypeError("gate must be a torch.Tensor")
        _check_like(gate, "gate", x)
        _check_like(input_gate, "input_gate", x)
        _check_exact(log_decay, "log_decay", (c,), torch.float32, x.device)
        self.state_stride = _check_step_state(state, (b, c), torch.float32, x.device)
        self.device, self.index, self.sizes = x.device, x.device.index, (b, c)
        self.strides = tuple(map(_batch_stride, (x, gate, input_gate)))
        self.copy = None in self.strides
        self.out = _proto((b, c), x.dtype, x.device)


_recur_step_plans: dict = {}


def _check_in_place(state):
    if state.requires_grad:
        raise ValueError("state is updated in place: it may not require a gradient")


def _changed(state):
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)


def gated_recurrence_step(x, gate, state, log_decay=None, input_gate=None):
    """One token of every sequence: x, gates (b, c); ``state`` fp32 (b, c) is
    updated in place.  Returns (b, c)."""
    args = (x, gate, log_decay, input_gate, state)
    plan = _lookup(_recur_step_plans, lambda: tuple(map(_sig, args)),
                   lambda: _RecurStepPlan(*args))
    _check_in_place(state)
    if plan.copy:
        return gated_recurrence_step(x.contiguous(), gate.contiguous(), state, log_decay,
                                     None if input_gate is None else input_gate.contiguous())
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return gated_recurrence_step(x, gate, state, log_decay, input_gate)
    log_decay = _dense(log_decay)
    out = torch.empty_like(plan.out)
    xs, gs, us = plan.strides
    st = N.lib().la_recurrence_step(
        x.data_ptr(), xs, gate.data_ptr(), gs, _ptr(input_gate), us, _ptr(log_decay),
        state.data_ptr(), plan.state_stride, out.data_ptr(), *plan.sizes, plan.code,
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_recurrence_step")
    _changed(state)
    return out


# ---- short causal convolution -------------------------------------------------------
_TAPS = (2, 3, 4)


def _check_taps(weight, channels):
    if not isinstance(weight, torch.Tensor):
        raise TypeError("weight must be a torch.Tensor")
    if weight.dim() != 2 or weight.shape[0] != channels or weight.shape[1] not in _TAPS:
        raise ValueError(f"weight must be ({channels}, taps) with taps in {_TAPS}, "
                         f"got shape {tuple(weight.shape)}")
    return weight.shape[1]


class _ConvPlan(_TokensPlan):
    def __init__(self, x, weight, bias, state, d_state, lengths, d_out):
        super().__init__(x, (d_out,), ("d_out",), lengths)
        b, t, c = self.sizes
        taps = _check_taps(weight, c)
        self.wcode = _check_affine(weight, bias, ("weight", "bias"), (c, taps), x)
        shape = (b, taps - 1, c)
        _check_exact(state, "initial_state", shape, x.dtype, x.device)
        _check_exact(d_state, "d_state", shape, x.dtype, x.device)
        self.sizes += (taps,)
        self.state = _proto(shape, x.dtype, x.device)
        ws = ctypes.c_size_t(0)
        N.check(N.lib().la_short_conv_workspace_size(*self.sizes, ctypes.byref(ws)),
                "la_short_conv_workspace_size")
        self.ws_bytes = ws.value
        self.workspace = _proto((ws.value,), torch.uint8, x.device)


_conv_plans: dict = {}


def _conv_plan(*args):
    return _lookup(_conv_plans, lambda: tuple(map(_sig, args)), lambda: _ConvPlan(*args))


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, lengths=None,
                return_state: bool = False):
    """Forward pass: (out, final state or None)."""
    plan = _conv_plan(x, weight, bias, initial_state, None, lengths, None)
    silu = _check_activation(activation)
    if plan.any_copy:
        return causal_conv(x.contiguous(), weight, bias, activation, initial_state, lengths,
                           return_state)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return causal_conv(x, weight, bias, activation, initial_state, lengths, return_state)
    weight, bias, initial_state, lengths = map(_dense, (weight, bias, initial_state, lengths))
    out = torch.empty_like(plan.out)
    final = torch.empty_like(plan.state) if return_state else None
    st = N.lib().la_short_conv_fwd(
        x.data_ptr(), plan.strides[0], weight.data_ptr(), _ptr(bias), plan.wcode,
        _ptr(initial_state), _ptr(lengths), plan.bits, out.data_ptr(), _ptr(final), *plan.sizes,
        silu, plan.code, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_short_conv_fwd")
    return out, final


def causal_conv_backward(x, weight, bias, activation, initial_state, lengths, d_out, d_state=None,
                         want_d_weight: bool = True, want_d_initial: bool = False):
    """Gradients (x, weight or None, bias or None, initial state or None)."""
    plan = _conv_plan(x, weight, bias, initial_state, d_state, lengths, d_out)
    silu = _check_activation(activation)
    if plan.any_copy:
        x, d_out = plan.read((x, d_out))
        return causal_conv_backward(x, weight, bias, activation, initial_state, lengths, d_out,
                                    d_state, want_d_weight, want_d_initial)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return causal_conv_backward(x, weight, bias, activation, initial_state, lengths,
                                        d_out, d_state, want_d_weight, want_d_initial)
    weight, bias, initial_state, lengths, d_state = map(
        _dense, (weight, bias, initial_state, lengths, d_state))
    dx = torch.empty_like(plan.out)
    d_weight = d_bias = workspace = None
    if want_d_weight:
        d_weight = torch.empty_like(weight)
        d_bias = None if bias is None else torch.empty_like(bias)
        workspace = torch.empty_like(plan.workspace)
    d_init = torch.empty_like(plan.state) if want_d_initial else None
    st = N.lib().la_short_conv_bwd(
        x.data_ptr(), plan.strides[0], weight.data_ptr(), _ptr(bias), plan.wcode,
        _ptr(initial_state), _ptr(lengths), plan.bits, d_out.data_ptr(), plan.strides[1],
        _ptr(d_state), dx.data_ptr(), _ptr(d_weight), _ptr(d_bias), _ptr(d_init), *plan.sizes,
        silu, plan.code, _ptr(workspace), plan.ws_bytes, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_short_conv_bwd")
    return dx, d_weight, d_bias, d_init


class _ConvStepPlan:
    def __init__(self, x, weight, state, bias):
        self.code = _check_tensor(x, "x", ("batch", "channels"))
        b, c = x.shape
        if c < 1:
            raise ValueError(f"x must be (batch, channels), got shape {tuple(x.shape)}")
        taps = _check_taps(weight, c)
        self.wcode = _check_affine(weight, bias, ("weight", "bias"), (c, taps), x)
        self.state_stride = _check_step_state(state, (b, taps - 1, c), x.dtype, x.device)
        self.device, self.index, self.sizes = x.device, x.device.index, (b, c, taps)
        self.stride = _batch_stride(x)
        self.out = _proto((b, c), x.dtype, x.device)


_conv_step_plans: dict = {}


def causal_conv_step(x, weight, state, bias=None, activation=None):
    """One token of every sequence: x (b, c); ``state`` (b, taps - 1, c), in
    x's type, is updated in place.  Returns (b, c)."""
    args = (x, weight, state, bias)
    plan = _lookup(_conv_step_plans, lambda: tuple(map(_sig, args)), lambda: _ConvStepPlan(*args))
    silu = _check_activation(activation)
    _check_in_place(state)
    if plan.stride is None:
        return causal_conv_step(x.contiguous(), weight, state, bias, activation)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return causal_conv_step(x, weight, state, bias, activation)
    weight, bias = _dense(weight), _dense(bias)
    out = torch.empty_like(plan.out)
    st = N.lib().la_short_conv_step(
        x.data_ptr(), plan.stride, weight.data_ptr(), _ptr(bias), plan.wcode, state.data_ptr(),
        plan.state_stride, out.data_ptr(), *plan.sizes, silu, plan.code,
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_short_conv_step")
    _changed(state)
    return out


# ---- group norm -----------------------------------------------------------------------
class _GroupNormPlan:
    def __init__(self, x, groups, gate, weight, bias, d_out):
        if not isinstance(x, torch.Tensor):
            raise TypeError("x must be a torch.Tensor")
        if x.dim() < 1 or x.shape[-1] < 1:
            raise ValueError(f"x must be (..., channels), got shape {tuple(x.shape)}")
        if x.device.type != "cuda":
            raise ValueError(f"x must be a CUDA tensor (got {x.device}); "
                             "this library has no CPU implementation")
        self.code = _dtype_code(x)
        _check_like(gate, "gate", x)
        _check_like(d_out, "d_out", x)
        c = x.shape[-1]
        if groups < 1 or c % groups:
            raise ValueError(f"groups must divide the {c} channels, got {groups}")
        self.wcode = _check_affine(weight, bias, ("weight", "bias"), (c,), x)
        self.device, self.index = x.device, x.device.index
        self.shape, self.sizes = x.shape, (c, groups)
        lead = x.shape[:-1]
        rows = x.numel() // c
        tensors = (x, gate, d_out)
        if all(t is None or t.is_contiguous() for t in tensors):
            self.c_shape = _Strides(1, rows)
            self.strides = tuple(None if t is None else _Strides(0, c) for t in tensors)
            self.copy = None
        else:  # up to two leading dimensions are read in place
            copy = tuple(t is not None and (len(lead) > 2 or (t.stride(-1) != 1 and c > 1))
                         for t in tensors)
            self.copy = copy if any(copy) else None
            if self.copy is None:
                pad = (1,) * (2 - len(lead))
                self.c_shape = _Strides(*pad, *lead)
                self.strides = tuple(
                    None if t is None else _Strides(*((0,) * len(pad)), *t.stride()[:-1])
                    for t in tensors)
        self.out = _proto(tuple(x.shape), x.dtype, x.device)
        self.stats = _proto((*lead, groups, 2), torch.float32, x.device)
        ws = ctypes.c_size_t(0)
        with _on_device(x.device):
            N.check(N.lib().la_group_norm_bwd_workspace_size(rows, c, ctypes.byref(ws)),
                    "la_group_norm_bwd_workspace_size")
        self.ws_bytes = ws.value
        self.workspace = _proto((ws.value,), torch.uint8, x.device)

    def read(self, tensors):
        return [t.contiguous() if c else t for t, c in zip(tensors, self.copy)]


_group_plans: dict = {}


def _group_plan(x, groups, gate, weight, bias, d_out):
    return _lookup(_group_plans,
                   lambda: (_sig(x), groups, _sig(gate), _sig(weight), _sig(bias), _sig(d_out)),
                   lambda: _GroupNormPlan(x, groups, gate, weight, bias, d_out))


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, eps: float = 1e-5,
               want_stats: bool = False):
    """Forward pass: (out, fp32 (..., groups, 2) means and reciprocal deviations
    or None)."""
    groups = operator.index(groups)
    plan = _group_plan(x, groups, gate, weight, bias, None)
    silu = _check_activation(activation)
    if plan.copy is not None:
        x, gate, _ = plan.read((x, gate, None))
        return group_norm(x, groups, weight, bias, gate, activation, eps, want_stats)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return group_norm(x, groups, weight, bias, gate, activation, eps, want_stats)
    weight, bias = _dense(weight), _dense(bias)
    out = torch.empty_like(plan.out)
    stats = torch.empty_like(plan.stats) if want_stats else None
    st = N.lib().la_group_norm_fwd(
        x.data_ptr(), plan.strides[0], _ptr(gate), plan.strides[1], _ptr(weight), _ptr(bias),
        plan.wcode, out.data_ptr(), _ptr(stats), plan.c_shape, *plan.sizes, silu, plan.code, eps,
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_group_norm_fwd")
    return out, stats


def group_norm_backward(x, groups, weight, bias, gate, activation, stats, d_out,
                        want_d_affine: bool = True):
    """Gradients (x, gate or None, weight or None, bias or None)."""
    plan = _group_plan(x, groups, gate, weight, bias, d_out)
    silu = _check_activation(activation)
    if plan.copy is not None:
        x, gate, d_out = plan.read((x, gate, d_out))
        return group_norm_backward(x, groups, weight, bias, gate, activation, stats, d_out,
                                   want_d_affine)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return group_norm_backward(x, groups, weight, bias, gate, activation, stats, d_out,
                                       want_d_affine)
    _check_exact(stats, "stats", tuple(plan.stats.shape), torch.float32, plan.device)
    weight, bias, stats = _dense(weight), _dense(bias), _dense(stats)
    dx = torch.empty_like(plan.out)
    d_gate = None if gate is None else torch.empty_like(plan.out)
    d_weight = d_bias = workspace = None
    if want_d_affine:
        d_weight = None if weight is None else torch.empty_like(weight)
        d_bias = None if bias is None else torch.empty_like(bias)
        if not (weight is None and bias is None):
            workspace = torch.empty_like(plan.workspace)
    st = N.lib().la_group_norm_bwd(
        x.data_ptr(), plan.strides[0], _ptr(gate), plan.strides[1], _ptr(weight), _ptr(bias),
        plan.wcode, stats.data_ptr(), d_out.data_ptr(), plan.strides[2], dx.data_ptr(),
        _ptr(d_gate), _ptr(d_weight), _ptr(d_bias), plan.c_shape, *plan.sizes, silu, plan.code,
        _ptr(workspace), plan.ws_bytes, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_group_norm_bwd")
    return dx, d_gate, d_weight, d_bias
