"""Torch-facing calls into the native library (device memory + streams only).

Every function takes ``(b, h, t, d)`` CUDA tensors, enqueues the kernel on
``torch.cuda.current_stream()`` and returns a freshly allocated output in
``q.dtype``.  Inputs are never modified.  Failures raise; nothing falls back
to another implementation.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _native as N

_DTYPES = {torch.float32: N.LA_DTYPE_FLOAT32, torch.bfloat16: N.LA_DTYPE_BFLOAT16}


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32 or bfloat16") from None


def _check_qkv(q, k, v, same_dv: bool = False):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dim() != 4:
            raise ValueError(f"{name} must be (batch, heads, seq_len, dim), got shape {tuple(t.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v dtypes differ: {q.dtype}, {k.dtype}, {v.dtype}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.device.type != "cuda":
            raise ValueError(f"{name} must be a CUDA tensor (got {t.device}); "
                             "this library has no CPU implementation")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k, v are on different devices")
    if q.shape != k.shape:
        raise ValueError(f"q and k shapes differ: {tuple(q.shape)} vs {tuple(k.shape)}")
    if v.shape[:3] != q.shape[:3]:
        raise ValueError(f"v shape {tuple(v.shape)} does not match q {tuple(q.shape)}")
    if same_dv and v.shape[-1] != q.shape[-1]:
        raise ValueError("v must have the same head dim as q for this op")
    return _dtype_code(q)


# Host cost matters: a call's launch latency is exposed whenever the GPU is
# idle, so the per-call Python work below avoids object churn (raw stream
# handle, plain ints for pointers, no device switch when already current,
# plan results cached per shape).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device) -> int:
    """The raw cudaStream_t of the current stream of `device`."""
    index = torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _on_device(device):
    """Make `device` current for the call (a no-op when it already is)."""
    index = torch.device(device).index
    if index is None or index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(index)


def based_parallel(q, k, v, eps: float = 1e-6) -> torch.Tensor:
    """Parallel (quadratic) BASED attention, normalised, causal."""
    code = _check_qkv(q, k, v)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    b, h, t, d = q.shape
    dv = v.shape[-1]
    out = torch.empty((b, h, t, dv), dtype=q.dtype, device=q.device)
    with _on_device(q.device):
        st = N.lib().la_based_parallel_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(out), b, h, t, d, dv,
                                           code, float(eps), _stream_ptr(q.device))
    N.check(st, "la_based_parallel_fwd")
    return out


def feature_dim(d_qk: int) -> int:
    return 1 + d_qk + d_qk * (d_qk + 1) // 2


def chunked_plan(batch_heads: int, seq_len: int, d_qk: int, d_v: int, dtype: torch.dtype,
                 segments: int = 0):
    """(segments, workspace_bytes) the library will use for this shape on the
    current device."""
    return _chunked_plan(int(batch_heads), int(seq_len), int(d_qk), int(d_v), _DTYPES[dtype],
                         int(segments), torch.cuda.current_device())


@functools.lru_cache(maxsize=1024)
def _chunked_plan(batch_heads, seq_len, d_qk, d_v, code, segments, device_index):
    g = ctypes.c_int(0)
    ws = ctypes.c_size_t(0)
    st = N.lib().la_based_chunked_plan(batch_heads, seq_len, d_qk, d_v, code, segments,
                                       ctypes.byref(g), ctypes.byref(ws))
    N.check(st, "la_based_chunked_plan")
    return g.value, ws.value


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def based_chunked(q, k, v, chunk_size: int = 64, eps: float = 1e-6, normalize: bool = True,
                  init_state: torch.Tensor | None = None, return_state: bool = False,
                  segments: int = 0, workspace: torch.Tensor | None = None,
                  reuse_segments: bool = False, feature_map: str = "taylor"):
    """Chunked recurrent linear attention (BASED Taylor features by default).

    ``init_state`` / the returned final state are fp32 ``(b*h, F, d_v + 1)``
    in the key-side feature basis documented in ``include/la_attention.h``.
    ``feature_map="identity"`` uses phi(x) = x (F = d_qk, numerator only).
    """
    code = _check_qkv(q, k, v)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    b, h, t, d = q.shape
    dv = v.shape[-1]
    if chunk_size < 1:
        raise ValueError("chunk_size must be >= 1")
    if feature_map not in ("taylor", "identity"):
        raise ValueError(f"feature_map must be 'taylor' or 'identity', got {feature_map!r}")
    identity = feature_map == "identity"
    if identity and normalize:
        raise ValueError("the identity feature map is numerator-only (normalize=False)")
    F = d if identity else feature_dim(d)
    if init_state is not None:
        if (init_state.dtype != torch.float32 or init_state.device != q.device
                or tuple(init_state.shape) != (b * h, F, dv + 1)):
            raise ValueError(f"init_state must be float32 {(b * h, F, dv + 1)} on {q.device}")
        init_state = init_state.contiguous()
    out = torch.empty((b, h, t, dv), dtype=q.dtype, device=q.device)
    final = torch.empty((b * h, F, dv + 1), dtype=torch.float32, device=q.device) if return_state else None
    with _on_device(q.device):
        _, ws_bytes = chunked_plan(b * h, t, d, dv, q.dtype, segments)
        if workspace is None:
            workspace = _workspace(ws_bytes, q.device)
        elif workspace.numel() * workspace.element_size() < ws_bytes:
            raise ValueError(f"workspace too small: need {ws_bytes} bytes")
        flags = ((N.LA_CHUNKED_NORMALIZE if normalize else 0)
                 | (N.LA_CHUNKED_REUSE_SEGMENTS if reuse_segments else 0)
                 | (N.LA_CHUNKED_IDENTITY if identity else 0))
        st = N.lib().la_based_chunked_fwd(
            _ptr(q), _ptr(k), _ptr(v), _ptr(out), b, h, t, d, dv, code, int(chunk_size),
            float(eps), flags, _ptr(init_state), _ptr(final), _ptr(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size(),
            int(segments), _stream_ptr(q.device))
    N.check(st, "la_based_chunked_fwd")
    if return_state:
        return out, final
    return out


def based_chunked_state(k, v, segments: int = 0, workspace: torch.Tensor | None = None):
    """Total state sum_j phi_k(k_j) [v_j, 1]^T per head, fp32 ``(b*h, F, d_v+1)``."""
    code = _check_qkv(k, k, v)
    k, v = k.contiguous(), v.contiguous()
    b, h, t, d = k.shape
    dv = v.shape[-1]
    state = torch.empty((b * h, feature_dim(d), dv + 1), dtype=torch.float32, device=k.device)
    with _on_device(k.device):
        _, ws_bytes = chunked_plan(b * h, t, d, dv, k.dtype, segments)
        if workspace is None:
            workspace = _workspace(ws_bytes, k.device)
        st = N.lib().la_based_chunked_state(
            _ptr(k), _ptr(v), _ptr(state), b, h, t, d, dv, code, _ptr(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size(),
            int(segments), _stream_ptr(k.device))
    N.check(st, "la_based_chunked_state")
    return state


def sliding_window(q, k, v, window_size: int = 64) -> torch.Tensor:
    """Causal sliding-window softmax attention over [i - W + 1, i]."""
    code = _check_qkv(q, k, v, same_dv=True)
    if int(window_size) < 1:
        raise ValueError("window_size must be >= 1")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    b, h, t, d = q.shape
    out = torch.empty_like(q)
    with _on_device(q.device):
        st = N.lib().la_sliding_window_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(out), b, h, t, d, code,
                                           int(window_size), _stream_ptr(q.device))
    N.check(st, "la_sliding_window_fwd")
    return out


def based_layer(q, k, v, window_size: int = 64, eps: float = 1e-6, segments: int = 0,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The full BASED layer: chunked BASED attention plus sliding-window
    softmax attention over the same q, k, v (window <= 129): two tensor-core
    kernels for bf16, d_qk = 16, d_v = 64 (the second adds its term to the
    first's output), one pass on CUDA cores otherwise."""
    code = _check_qkv(q, k, v)
    if int(window_size) < 1:
        raise ValueError("window_size must be >= 1")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    b, h, t, d = q.shape
    dv = v.shape[-1]
    out = torch.empty((b, h, t, dv), dtype=q.dtype, device=q.device)
    with _on_device(q.device):
        g, ws_bytes = chunked_plan(b * h, t, d, dv, q.dtype, segments)
        if workspace is None:
            workspace = _workspace(ws_bytes, q.device)
        st = N.lib().la_based_layer_fwd(
            _ptr(q), _ptr(k), _ptr(v), _ptr(out), b, h, t, d, dv, code, int(window_size),
            float(eps), _ptr(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size(),
            int(segments), _stream_ptr(q.device))
    N.check(st, "la_based_layer_fwd")
    return out


def check_tangents(*tensors) -> None:
    """Forward-mode derivatives are refused: a dual tensor requires no gradient, and
    a kernel given its address would drop the tangent."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (-1 outside of a dual level)
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("this operator has no forward-mode derivative")


# ---- plans ---------------------------------------------------------------------
# The checks of a call, its strides as the C entry points take them and its
# workspace depend on shapes, strides, types and devices alone.  They are worked
# out at the first call of a signature and kept under it, so that a decoding
# step or a small norm does not spend more time here than on the GPU.  Nothing
# is kept by a tensor's address or contents.
_Int64x3 = ctypes.c_int64 * 3
_MAX_PLANS = 4096
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class _Strides(int):
    """The address of three int64, with the array that holds them: what ctypes
    converts fastest."""

    def __new__(cls, *values):
        array = _Int64x3(*values)
        self = super().__new__(cls, ctypes.addressof(array))
        self.array = array
        return self


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _keep(plans: dict, key, plan):
    if len(plans) >= _MAX_PLANS:
        plans.clear()
    plans[key] = plan
    return plan


_one_element: dict = {}


def _proto(shape, dtype, device):
    """One element (never read) seen as ``shape``: ``torch.empty_like`` of it makes
    that contiguous tensor in a third of the time of ``torch.empty`` with its
    shape, type and device (1 against 3 us)."""
    if 0 in shape:
        return torch.empty(shape, dtype=dtype, device=device)
    key = (dtype, device)
    one = _one_element.get(key)
    if one is None:
        one = _one_element[key] = torch.empty((), dtype=dtype, device=device)
    return one.expand(shape)


# ---- linear attention with a decay for each head ---------------------------------
def _heads_strides(t: torch.Tensor):
    """Strides of ``t`` (b, h, t, d) as the kernels read it in place -- a dense
    last dimension, and for bf16 rows of whole 16-byte packs where the width
    allows them -- or None where they rule that out (or overlap)."""
    b, h, n, d = t.shape
    if t.numel() == 0:  # contiguous whatever its strides are: a copy would not change them
        return _Strides(h * n * d, n * d, d)
    sb, sh, st, sd = t.stride()
    ok = ((sd == 1 or d == 1) and (sb > 0 or b == 1) and (sh > 0 or h == 1)
          and (st >= d or n == 1))
    if ok and d % 8 == 0 and t.dtype == torch.bfloat16:
        ok = (sb % 8 == 0 or b == 1) and (sh % 8 == 0 or h == 1) and (st % 8 == 0 or n == 1)
    if not ok:
        return None
    # a dimension of one entry has no stride of its own
    return _Strides(sb if b > 1 else h * n * d, sh if h > 1 else n * d, st if n > 1 else d)


def _tokens_first(t: torch.Tensor) -> bool:
    """Whether ``t`` (b, h, t, d) lies as (b, t, h, d): a transposed projection."""
    return t.shape[1] > 1 and t.shape[2] > 1 and t.stride(1) < t.stride(2)


def _empty_heads(b, h, n, d, proto, tokens_first, like=None):
    if like is not None:  # dense, and laid out as wanted
        return torch.empty_like(like)
    out = torch.empty_like(proto)
    return out.transpose(1, 2) if tokens_first else out


def _check_log_decay(log_decay, heads, device):
    if not isinstance(log_decay, torch.Tensor):
        raise TypeError("log_decay must be a torch.Tensor")
    if (log_decay.dtype != torch.float32 or log_decay.device != device
            or tuple(log_decay.shape) != (heads,)):
        raise ValueError(f"log_decay must be float32 ({heads},) on {device}")
    _check_constant(log_decay)


def _check_constant(log_decay):
    if (isinstance(log_decay, torch.Tensor) and log_decay.requires_grad
            and torch.is_grad_enabled()):
        raise ValueError("log_decay is a constant of the operator: it has no gradient")


def _check_state(state, shape, device, name):
    if not isinstance(state, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if state.dtype != torch.float32 or state.device != device or tuple(state.shape) != shape:
        raise ValueError(f"{name} must be float32 {shape} on {device}")


class _DecayPlan:
    """One signature of the decayed linear attention: sizes, strides, workspace."""

    __slots__ = ("index", "device", "dtype", "sizes", "scale", "pack", "copy", "strides",
                 "outs", "dense", "out_strides", "state_shape", "state", "ws_bytes", "workspace",
                 "pad")

    def __init__(self, q, k, v, log_decay, states, grad, segments):
        code = _check_qkv(q, k, v)
        b, h, t, d = q.shape
        dv = v.shape[-1]
        _check_log_decay(log_decay, h, q.device)
        for name, s in states:
            if s is not None:
                _check_state(s, (b, h, d, dv), q.device, name)
        if grad is not None and (not isinstance(grad, torch.Tensor) or grad.shape != v.shape
                                 or grad.dtype != v.dtype or grad.device != v.device):
            raise ValueError(f"d_out must be {v.dtype} {tuple(v.shape)} on {v.device}")
        self.device, self.dtype = q.device, q.dtype
        self.index = q.device.index
        self.sizes = (b, h, t, d, dv, code)
        self.scale = 1.0 / math.sqrt(max(d, 1))  # (the library refuses d = 0)
        self.state_shape = (b, h, d, dv)
        read = (q, k, v) if grad is None else (q, k, v, grad)
        # bf16 rows of whole 16-byte packs have to start at 16 bytes
        self.pack = tuple(q.dtype == torch.bfloat16 and x.shape[-1] % 8 == 0 for x in read)
        # Widths that no 16-byte pack divides are widened with zeros for the
        # tensor-core kernel.  The CUDA-core kernel takes them as they are, at 10 us
        # per tile of 64 tokens and SM, and has walked a few of those before the
        # copies are launched: forward / gradients of 4 heads of 55 x 40 / 57 in 23 /
        # 24 us against 83 / 135 widened, of 32 heads of 500 x 60 in 52 / 93 against
        # 87 / 137, of 64 heads of 1000 x 60 in 138 / 321 against 85 / 150, of one head
        # of 32768 x 60 in 155 / 205 against 89 / 140.
        walks = (b * h * -(-dv // 64) * (1 if d <= 64 else 2) if grad is None
                 else b * h * (2 * -(-d // 64) + -(-dv // 64)))
        few = t <= 4096 and walks * -(-t // 64) <= 6 * torch.cuda.get_device_properties(
            q.device).multi_processor_count
        self.pad = ((-d % 8, -dv % 8) if q.dtype == torch.bfloat16 and (d % 8 or dv % 8)
                    and not few else None)
        self.strides = tuple(_heads_strides(x) for x in read)
        self.copy = any(s is None for s in self.strides)
        written = (v,) if grad is None else (q, k, v)
        self.outs = tuple(
            (b, h, t, x.shape[-1],
             _proto((b, t, h, x.shape[-1]) if _tokens_first(x) else (b, h, t, x.shape[-1]),
                    x.dtype, x.device), _tokens_first(x))
            for x in written)
        self.dense = tuple((x.transpose(1, 2) if o[-1] else x).is_contiguous()
                           for x, o in zip(written, self.outs))
        self.out_strides = tuple(
            _Strides(h * t * w, w if first else t * w, h * w if first else w)
            for _, _, _, w, _, first in self.outs)
        n, ws = ctypes.c_int(0), ctypes.c_size_t(0)
        with _on_device(q.device):
            st = N.lib().la_decay_plan(*self.sizes, int(grad is not None), segments,
                                       ctypes.byref(n), ctypes.byref(ws))
        N.check(st, "la_decay_plan")
        self.ws_bytes = ws.value
        self.workspace = _proto((ws.value,), torch.uint8, q.device) if ws.value else None
        self.state = _proto(self.state_shape, torch.float32, q.device)


_decay_plans: dict = {}


def _decay_plan(q, k, v, log_decay, initial_state, d_state, grad, segments) -> _DecayPlan:
    try:
        key = (_sig(q), _sig(k), _sig(v), _sig(log_decay), _sig(initial_state), _sig(d_state),
               _sig(grad), segments)
        plan = _decay_plans.get(key)
        if plan is not None and not (log_decay.requires_grad and torch.is_grad_enabled()):
            return plan
    except AttributeError:  # not tensors: the checks say which
        key = None
    return _keep(_decay_plans, key, _DecayPlan(
        q, k, v, log_decay, (("initial_state", initial_state), ("d_state", d_state)), grad,
        segments))


def _in_place(x: torch.Tensor, strides, pack: bool) -> torch.Tensor:
    """``x``, or a copy of it where its layout or address cannot be read in place."""
    if strides is not None and not (pack and x.data_ptr() & 15):
        return x
    x = x.contiguous()
    return x.clone() if pack and x.data_ptr() & 15 else x  # (a view at an odd offset)


def _readable(plan, tensors):
    """The inputs as the kernels can read them, or None if they already are."""
    if not plan.copy:
        odd = 0
        for p, x in zip(plan.pack, tensors):
            if p:
                odd |= x.data_ptr()
        if not odd & 15:
            return None
    return [_in_place(x, s, p) for x, s, p in zip(tensors, plan.strides, plan.pack)]


def _widen(x, by, rows_by=0):
    """``x`` with ``by`` more zero columns (and ``rows_by`` more rows)."""
    return None if x is None else torch.nn.functional.pad(x, (0, by, 0, rows_by))


def _narrowed(outs, tensors):
    """The leading columns of ``tensors`` laid out as the plan's outputs."""
    got = []
    for o, x in zip(outs, tensors):
        y = _empty_heads(*o)
        got.append(y.copy_(x[..., :o[3]]))
    return got


def decay_attention(q, k, v, log_decay, scale=None, initial_state=None, return_state: bool = False,
                    segments: int = 0):
    """Forward pass of the decayed linear attention (no autograd): the output,
    or (output, final state fp32 (b, h, d_qk, d_v))."""
    plan = _decay_plan(q, k, v, log_decay, initial_state, None, None, segments)
    if plan.pad is not None:
        a, b = plan.pad
        got = decay_attention(_widen(q, a), _widen(k, a), _widen(v, b), log_decay,
                              plan.scale if scale is None else scale,
                              _widen(initial_state, b, a), return_state, segments)
        out, = _narrowed(plan.outs, (got[0] if return_state else got,))
        _, _, d, dv = plan.state_shape
        return (out, got[1][:, :, :d, :dv].contiguous()) if return_state else out
    again = _readable(plan, (q, k, v))
    if again is not None:
        out = decay_attention(*again, log_decay, scale, initial_state, return_state, segments)
        if _tokens_first(v) == _tokens_first(again[2]):
            return out
        y = _empty_heads(*plan.outs[0])
        y.copy_(out[0] if return_state else out)
        return (y, out[1]) if return_state else y
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return decay_attention(q, k, v, log_decay, scale, initial_state, return_state,
                                   segments)
    out = _empty_heads(*plan.outs[0], v if plan.dense[0] else None)
    final = torch.empty_like(plan.state) if return_state else None
    if not log_decay.is_contiguous():
        log_decay = log_decay.contiguous()
    if initial_state is not None and not initial_state.is_contiguous():
        initial_state = initial_state.contiguous()
    workspace = None if plan.workspace is None else torch.empty_like(plan.workspace)
    qs, ks, vs = plan.strides
    st = N.lib().la_decay_chunked_fwd(
        q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), plan.out_strides[0],
        log_decay.data_ptr(), *plan.sizes, plan.scale if scale is None else float(scale),
        _ptr(initial_state), _ptr(final), _ptr(workspace), plan.ws_bytes, segments,
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_decay_chunked_fwd")
    return (out, final) if return_state else out


def decay_attention_backward(q, k, v, log_decay, d_out, scale=None, initial_state=None,
                             d_state=None, want_d_initial: bool = False, segments: int = 0):
    """Gradients (dq, dk, dv, d_initial_state or None) of ``decay_attention``
    for the gradients of its output and (``d_state``) of its final state."""
    plan = _decay_plan(q, k, v, log_decay, initial_state, d_state, d_out, segments)
    if plan.pad is not None:
        a, b = plan.pad
        *grads, g0 = decay_attention_backward(
            _widen(q, a), _widen(k, a), _widen(v, b), log_decay, _widen(d_out, b),
            plan.scale if scale is None else scale, _widen(initial_state, b, a),
            _widen(d_state, b, a), want_d_initial, segments)
        _, _, d, dv = plan.state_shape
        return (*_narrowed(plan.outs, grads),
                None if g0 is None else g0[:, :, :d, :dv].contiguous())
    again = _readable(plan, (q, k, v, d_out))
    if again is not None:
        q, k, v, d_out = again
        return decay_attention_backward(q, k, v, log_decay, d_out, scale, initial_state, d_state,
                                        want_d_initial, segments)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return decay_attention_backward(q, k, v, log_decay, d_out, scale, initial_state,
                                            d_state, want_d_initial, segments)
    gq, gk, gv = (_empty_heads(*o, x if dense else None)
                  for o, x, dense in zip(plan.outs, (q, k, v), plan.dense))
    g0 = torch.empty_like(plan.state) if want_d_initial else None
    log_decay = log_decay.contiguous()
    initial_state = None if initial_state is None else initial_state.contiguous()
    d_state = None if d_state is None else d_state.contiguous()
    workspace = None if plan.workspace is None else torch.empty_like(plan.workspace)
    qs, ks, vs, ds = plan.strides
    gqs, gks, gvs = plan.out_strides
    st = N.lib().la_decay_chunked_bwd(
        q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, d_out.data_ptr(), ds, gq.data_ptr(),
        gqs, gk.data_ptr(), gks, gv.data_ptr(), gvs, log_decay.data_ptr(), *plan.sizes,
        plan.scale if scale is None else float(scale), _ptr(initial_state), _ptr(d_state),
        _ptr(g0), _ptr(workspace), plan.ws_bytes, segments, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_decay_chunked_bwd")
    return gq, gk, gv, g0


class _StepPlan:
    """One signature of the single-token form."""

    __slots__ = ("index", "device", "dtype", "sizes", "scale", "out", "strides", "copy")

    def __init__(self, q, k, v, log_decay, state):
        for name, x in (("q", q), ("k", k), ("v", v)):
            if not isinstance(x, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if x.dim() != 3:
                raise ValueError(f"{name} must be (batch, heads, dim), got shape {tuple(x.shape)}")
        code = _check_qkv(q.unsqueeze(2), k.unsqueeze(2), v.unsqueeze(2))
        b, h, d = q.shape
        dv = v.shape[-1]
        _check_log_decay(log_decay, h, q.device)
        _check_state(state, (b, h, d, dv), q.device, "state")
        sb, sh, sr, sc = state.stride()
        if ((sc != 1 and dv > 1) or (sr != dv and d > 1) or (sh < d * dv and h > 1)
                or (sb < d * dv and b > 1)):
            raise ValueError("state needs dense (d_qk, d_v) entries that do not overlap")
        if b > 1 and h > 1 and not (sb >= sh * (h - 1) + d * dv or sh >= sb * (b - 1) + d * dv):
            raise ValueError("the states of different sequences overlap")
        self.device, self.dtype, self.index = q.device, q.dtype, q.device.index
        self.sizes = (b, h, d, dv, code)
        self.scale = 1.0 / math.sqrt(max(d, 1))  # (the library refuses d = 0)
        self.out = _proto((b, h, dv), q.dtype, q.device)
        self.copy = any(x.stride(2) != 1 and x.shape[2] > 1 and x.numel() > 0 for x in (q, k, v))
        self.strides = tuple(_Strides(*x.stride()) for x in (q, k, v)) + (_Strides(sb, sh),)


_step_plans: dict = {}


def decay_attention_step(q, k, v, log_decay, state, scale=None) -> torch.Tensor:
    """One token of every sequence: q, k (b, h, d_qk), v (b, h, d_v); ``state``
    fp32 (b, h, d_qk, d_v) is updated in place.  Returns (b, h, d_v)."""
    try:
        key = (_sig(q), _sig(k), _sig(v), _sig(log_decay), _sig(state))
        plan = _step_plans.get(key)
    except AttributeError:  # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _keep(_step_plans, key, _StepPlan(q, k, v, log_decay, state))
    _check_constant(log_decay)
    if state.requires_grad:
        raise ValueError("state is updated in place: it may not require a gradient")
    if plan.copy:
        return decay_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), log_decay,
                                    state, scale)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return decay_attention_step(q, k, v, log_decay, state, scale)
    if not log_decay.is_contiguous():
        log_decay = log_decay.contiguous()
    out = torch.empty_like(plan.out)
    qs, ks, vs, ss = plan.strides
    st = N.lib().la_decay_step(
        q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), state.data_ptr(), ss,
        log_decay.data_ptr(), *plan.sizes, plan.scale if scale is None else float(scale),
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_decay_step")
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return out


# ---- root-mean-square norm ---------------------------------------------------------
_FP8_GROUPS = (16, 32, 64, 128, 256)


def _check_rows(x, name, like=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be (..., d), got shape {tuple(x.shape)}")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (got {x.device}); "
                         "this library has no CPU implementation")
    if like is not None and (x.shape != like.shape or x.dtype != like.dtype
                             or x.device != like.device):
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} on {like.device}")
    return _dtype_code(x)


class _NormPlan:
    """One signature of the norm: ``rows`` are the (..., d) tensors it reads,
    the first of them under ``name``, the others of the same shape and type."""

    __slots__ = ("index", "device", "dtype", "shape", "lead", "d", "codes", "strides", "c_shape",
                 "copy", "aligned", "weight_copy", "as_is", "dense", "group", "rstd", "scales",
                 "workspace", "ws_bytes")

    def __init__(self, rows, names, weight, group_size):
        x = rows[0]
        code = _check_rows(x, names[0])
        for t, name in zip(rows[1:], names[1:]):
            if t is not None:
                _check_rows(t, name, x)
        wcode = code
        d = x.shape[-1]
        if weight is not None:
            if not isinstance(weight, torch.Tensor):
                raise TypeError("weight must be a torch.Tensor")
            wcode = _dtype_code(weight)
            if tuple(weight.shape) != (d,) or weight.device != x.device:
                raise ValueError(f"weight must be ({d},) on {x.device}")
        self.group = d if group_size is None else group_size
        if group_size is not None and (group_size not in _FP8_GROUPS or d % group_size):
            raise ValueError(f"group_size must be None or one of {_FP8_GROUPS} dividing {d}, "
                             f"got {group_size}")
        self.device, self.dtype, self.index = x.device, x.dtype, x.device.index
        self.shape, self.lead, self.d, self.codes = x.shape, x.shape[:-1], d, (code, wcode)
        self.rstd = _proto(self.lead, torch.float32, x.device)
        self.scales = _proto((*self.lead, d // self.group), torch.float32, x.device)
        self.weight_copy = weight is not None and not weight.is_contiguous()
        lead = x.shape[:-1]
        if all(t is None or t.is_contiguous() for t in rows):
            self.c_shape = _Strides(1, 1, x.numel() // d)
            self.strides = (_Strides(0, 0, d),) * len(rows)
            self.copy = (False,) * len(rows)
        else:  # up to three leading dimensions are read in place
            pad = (1,) * (3 - len(lead))
            self.copy = tuple(t is not None and (len(lead) > 3 or (t.stride(-1) != 1 and d > 1))
                              for t in rows)
            if not any(self.copy):
                self.c_shape = _Strides(*(pad + tuple(lead)))
                self.strides = tuple(
                    None if t is None else _Strides(*((0,) * len(pad) + t.stride()[:-1]))
                    for t in rows)
        # scales of groups need rows of whole 16-byte packs
        self.aligned = self.group != d
        if self.aligned and not any(self.copy):
            pack = 16 // x.element_size()
            self.copy = tuple(t is not None and any(n % pack for n in s.array)
                              for t, s in zip(rows, self.strides))
        self.as_is = not any(self.copy) and not self.weight_copy
        self.dense = x.is_contiguous()
        n = ctypes.c_size_t(0)
        with _on_device(x.device):
            N.check(N.lib().la_rms_norm_bwd_workspace_size(x.numel() // d, d, ctypes.byref(n)),
                    "la_rms_norm_bwd_workspace_size")
        self.ws_bytes = n.value
        self.workspace = _proto((n.value,), torch.uint8, x.device) if n.value else None


_norm_plans: dict = {}


def _norm_plan(rows, names, weight, group_size=None) -> _NormPlan:
    try:
        key = (*map(_sig, rows), names, _sig(weight), group_size)
        plan = _norm_plans.get(key)
    except AttributeError:  # not tensors: the checks say which
        key = plan = None
    if plan is None:
        plan = _keep(_norm_plans, key, _NormPlan(rows, names, weight, group_size))
    return plan


def _norm_inputs(plan, rows, weight):
    """The rows and the weight as the kernels can read them, or None if they
    already are."""
    if plan.as_is and not plan.aligned:
        return None
    tensors = (*rows, weight)
    copies = [*plan.copy, plan.weight_copy]
    if plan.aligned:
        copies = [c or (t is not None and t.data_ptr() & 15 != 0)
                  for c, t in zip(copies, tensors)]
    if not any(copies):
        return None
    return [t.clone(memory_format=torch.contiguous_format) if c else t
            for c, t in zip(copies, tensors)]


def _empty_rows(plan, like, dtype=None):
    """An empty contiguous tensor of the rows' shape; ``like`` has that shape."""
    if plan.dense:
        return torch.empty_like(like, dtype=dtype)
    return torch.empty(plan.shape, dtype=dtype or plan.dtype, device=plan.device)


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, want_rstd: bool = False):
    """Forward pass of the norm (no autograd): (y, x + residual or None, fp32
    reciprocal root mean squares per row or None)."""
    plan = _norm_plan((x, residual), ("x", "residual"), weight)
    again = _norm_inputs(plan, (x, residual), weight)
    if again is not None:
        return rms_norm(again[0], again[2], again[1], eps, want_rstd)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return rms_norm(x, weight, residual, eps, want_rstd)
    y = _empty_rows(plan, x)
    total = torch.empty_like(y) if residual is not None else None
    rstd = torch.empty_like(plan.rstd) if want_rstd else None
    st = N.lib().la_rms_norm_fwd(
        x.data_ptr(), plan.strides[0], _ptr(residual), plan.strides[1], _ptr(weight), y.data_ptr(),
        _ptr(total), _ptr(rstd), plan.c_shape, plan.d, *plan.codes, eps, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_rms_norm_fwd")
    return y, total, rstd


def rms_norm_fp8(x, weight=None, residual=None, eps: float = 1e-6, group_size: int | None = None):
    """The norm with its output held in e4m3: (y, scales, x + residual or None),
    scales fp32 (..., d / group_size), one per row without a group size."""
    plan = _norm_plan((x, residual), ("x", "residual"), weight, group_size)
    again = _norm_inputs(plan, (x, residual), weight)
    if again is not None:
        return rms_norm_fp8(again[0], again[2], again[1], eps, group_size)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return rms_norm_fp8(x, weight, residual, eps, group_size)
    y = _empty_rows(plan, x, torch.float8_e4m3fn)
    scales = torch.empty_like(plan.scales)
    total = _empty_rows(plan, x) if residual is not None else None
    st = N.lib().la_rms_norm_fp8(
        x.data_ptr(), plan.strides[0], _ptr(residual), plan.strides[1], _ptr(weight), y.data_ptr(),
        scales.data_ptr(), _ptr(total), plan.c_shape, plan.d, plan.group, *plan.codes, eps,
        _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_rms_norm_fp8")
    return y, scales, total


def rms_norm_backward(s, weight, rstd, d_y, d_sum=None, want_d_weight: bool = True):
    """Gradients (of x and of the residual alike, of the weight or None) of
    ``rms_norm`` from its saved rows ``s`` (x + residual) and ``rstd``."""
    plan = _norm_plan((s, d_y, d_sum), ("s", "d_y", "d_sum"), weight)
    again = _norm_inputs(plan, (s, d_y, d_sum), weight)
    if again is not None:
        return rms_norm_backward(again[0], again[3], rstd, again[1], again[2], want_d_weight)
    if plan.index != _get_device():
        with torch.cuda.device(plan.index):
            return rms_norm_backward(s, weight, rstd, d_y, d_sum, want_d_weight)
    if rstd.shape != plan.lead or rstd.dtype != torch.float32 or rstd.device != plan.device:
        raise ValueError(f"rstd must be float32 {tuple(plan.lead)} on {plan.device}")
    rstd = rstd.contiguous()
    d_s = _empty_rows(plan, s)
    d_w = workspace = None
    if want_d_weight and weight is not None:
        d_w = torch.empty_like(weight)
        if plan.workspace is not None:
            workspace = torch.empty_like(plan.workspace)
    st = N.lib().la_rms_norm_bwd(
        s.data_ptr(), plan.strides[0], _ptr(weight), d_y.data_ptr(), plan.strides[1], _ptr(d_sum),
        plan.strides[2], rstd.data_ptr(), d_s.data_ptr(), _ptr(d_w), plan.c_shape, plan.d,
        *plan.codes, _ptr(workspace), plan.ws_bytes, _stream_ptr(plan.device))
    if st != N.LA_OK:
        N.check(st, "la_rms_norm_bwd")
    return d_s, d_w


_copy_streams: dict = {}


def _side_streams(device):
    """Two streams per device (host->device, device->host), created once."""
    key = torch.device(device).index
    if key not in _copy_streams:
        _copy_streams[key] = (torch.cuda.Stream(device), torch.cuda.Stream(device))
    return _copy_streams[key]


def based_chunked_host(q, k, v, chunk_size: int = 64, eps: float = 1e-6, normalize: bool = True,
                       head_groups: int = 8, device=None, out: torch.Tensor | None = None):
    """Chunked BASED attention on host-resident ``(b, h, t, d)`` tensors.

    The heads are processed in ``head_groups`` groups so that the host-to-
    device copy of one group, the kernels of the previous group and the
    device-to-host copy of the group before run at the same time (PCIe is
    full duplex): the copies run on two side streams of ``device`` and are
    joined back into its current stream before the call returns.  Inputs
    should be pinned (``pin_memory()``) for the copies to overlap.  The
    result is written into ``out`` (a pinned host tensor is allocated if it
    is None) and is complete once the current stream has reached this point
    (e.g. after ``torch.cuda.current_stream().synchronize()``).
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.device.type != "cpu":
            raise ValueError(f"{name} must be a host tensor for based_chunked_host")
    if q.shape != k.shape or v.shape[:3] != q.shape[:3]:
        raise ValueError("q, k, v shapes do not match")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    b, h, t, d = q.shape
    dv = v.shape[-1]
    bh = b * h
    if out is None:
        out = torch.empty((b, h, t, dv), dtype=q.dtype).pin_memory()
    elif out.shape != (b, h, t, dv) or out.dtype != q.dtype or out.device.type != "cpu":
        raise ValueError(f"out must be a host {q.dtype} tensor of shape {(b, h, t, dv)}")
    qf, kf, vf = (x.reshape(bh, t, x.shape[-1]) for x in (q, k, v))
    of = out.view(bh, t, dv)
    groups = max(1, min(int(head_groups), bh))
    step = -(-bh // groups)
    with _on_device(device):
        compute = torch.cuda.current_stream(device)
        h2d, d2h = _side_streams(device)
        qd = torch.empty((bh, t, d), dtype=q.dtype, device=device)
        kd = torch.empty_like(qd)
        vd = torch.empty((bh, t, dv), dtype=v.dtype, device=device)
        start = torch.cuda.Event()
        start.record(compute)  # the buffers are free once the compute stream is here
        h2d.wait_event(start)
        d2h.wait_event(start)
        for lo in range(0, bh, step):
            hi = min(bh, lo + step)
            with torch.cuda.stream(h2d):
                for dst, src in ((qd, qf), (kd, kf), (vd, vf)):
                    dst[lo:hi].copy_(src[lo:hi], non_blocking=True)
                ready = torch.cuda.Event()
                ready.record(h2d)
            compute.wait_event(ready)
            y = based_chunked(qd[lo:hi].unsqueeze(0), kd[lo:hi].unsqueeze(0),
                              vd[lo:hi].unsqueeze(0), chunk_size=chunk_size, eps=eps,
                              normalize=normalize)
            done = torch.cuda.Event()
            done.record(compute)
            d2h.wait_event(done)
            with torch.cuda.stream(d2h):
                of[lo:hi].copy_(y[0], non_blocking=True)
            y.record_stream(d2h)  # its memory is not reused before this copy ends
        finished = torch.cuda.Event()
        finished.record(d2h)
        compute.wait_event(finished)
        h2d_done = torch.cuda.Event()
        h2d_done.record(h2d)
        compute.wait_event(h2d_done)
    return out
