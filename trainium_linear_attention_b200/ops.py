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


# ---- linear attention with a decay for each head ---------------------------------
_Strides = ctypes.c_int64 * 3


def _heads_view(t: torch.Tensor):
    """``t`` (b, h, t, d) as the kernels read it -- a dense last dimension and,
    for bf16, 16-byte rows where the width allows them -- and its strides.  A
    copy is made only where the strides rule that out (or overlap)."""
    b, h, n, d = t.shape
    sb, sh, st, sd = t.stride()
    ok = ((sd == 1 or d == 1) and (sb > 0 or b == 1) and (sh > 0 or h == 1)
          and (st >= d or n == 1))
    if ok and d % 8 == 0 and t.dtype == torch.bfloat16:
        ok = (t.data_ptr() % 16 == 0 and (sb % 8 == 0 or b == 1) and (sh % 8 == 0 or h == 1)
              and (st % 8 == 0 or n == 1))
    if not ok:
        t = t.contiguous()
        if t.data_ptr() % 16:  # a contiguous view at an odd offset
            t = t.clone()
        sb, sh, st, _ = t.stride()
    # a dimension of one entry has no stride of its own
    return t, _Strides(sb if b > 1 else h * n * d, sh if h > 1 else n * d, st if n > 1 else d)


def _heads_like(t: torch.Tensor, d: int) -> torch.Tensor:
    """An empty (b, h, t, d) tensor laid out as ``t``: tokens before heads where
    ``t`` is a transposed projection, else contiguous."""
    b, h, n, _ = t.shape
    if h > 1 and n > 1 and t.stride(1) < t.stride(2):
        return torch.empty((b, n, h, d), dtype=t.dtype, device=t.device).transpose(1, 2)
    return torch.empty((b, h, n, d), dtype=t.dtype, device=t.device)


def _check_decay(q, k, v, log_decay):
    code = _check_qkv(q, k, v)
    _check_log_decay(log_decay, q.shape[1], q.device)
    return code


def _check_log_decay(log_decay, heads, device):
    if not isinstance(log_decay, torch.Tensor):
        raise TypeError("log_decay must be a torch.Tensor")
    if (log_decay.dtype != torch.float32 or log_decay.device != device
            or tuple(log_decay.shape) != (heads,)):
        raise ValueError(f"log_decay must be float32 ({heads},) on {device}")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of the operator: it has no gradient")


def _check_state(state, shape, device, name):
    if not isinstance(state, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if state.dtype != torch.float32 or state.device != device or tuple(state.shape) != shape:
        raise ValueError(f"{name} must be float32 {shape} on {device}")


def _default_scale(scale, d_qk: int) -> float:
    return 1.0 / math.sqrt(d_qk) if scale is None else float(scale)


@functools.lru_cache(maxsize=1024)
def _decay_plan(batch, heads, seq_len, d_qk, d_v, code, backward, segments, device_index):
    g = ctypes.c_int(0)
    ws = ctypes.c_size_t(0)
    st = N.lib().la_decay_plan(batch, heads, seq_len, d_qk, d_v, code, int(backward), segments,
                               ctypes.byref(g), ctypes.byref(ws))
    N.check(st, "la_decay_plan")
    return g.value, ws.value


def decay_attention(q, k, v, log_decay, scale=None, initial_state=None, return_state: bool = False,
                    segments: int = 0):
    """Forward pass of the decayed linear attention (no autograd): the output,
    or (output, final state fp32 (b, h, d_qk, d_v))."""
    code = _check_decay(q, k, v, log_decay)
    b, h, t, d = q.shape
    dv = v.shape[-1]
    if initial_state is not None:
        _check_state(initial_state, (b, h, d, dv), q.device, "initial_state")
        initial_state = initial_state.contiguous()
    out = _heads_like(v, dv)
    final = torch.empty((b, h, d, dv), dtype=torch.float32, device=q.device) if return_state else None
    log_decay = log_decay.contiguous()
    (q, qs), (k, ks), (v, vs), (_, os_) = (_heads_view(x) for x in (q, k, v, out))
    with _on_device(q.device):
        _, ws_bytes = _decay_plan(b, h, t, d, dv, code, False, int(segments),
                                  torch.cuda.current_device())
        workspace = _workspace(ws_bytes, q.device)
        st = N.lib().la_decay_chunked_fwd(
            _ptr(q), qs, _ptr(k), ks, _ptr(v), vs, _ptr(out), os_, _ptr(log_decay), b, h, t, d, dv,
            code, _default_scale(scale, d), _ptr(initial_state), _ptr(final), _ptr(workspace),
            ws_bytes, int(segments), _stream_ptr(q.device))
    N.check(st, "la_decay_chunked_fwd")
    return (out, final) if return_state else out


def decay_attention_backward(q, k, v, log_decay, d_out, scale=None, initial_state=None,
                             d_state=None, want_d_initial: bool = False, segments: int = 0):
    """Gradients (dq, dk, dv, d_initial_state or None) of ``decay_attention``
    for the gradients of its output and (``d_state``) of its final state."""
    code = _check_decay(q, k, v, log_decay)
    b, h, t, d = q.shape
    dv = v.shape[-1]
    if not isinstance(d_out, torch.Tensor) or d_out.shape != v.shape or d_out.dtype != v.dtype:
        raise ValueError(f"d_out must be {v.dtype} {tuple(v.shape)}")
    for name, s in (("initial_state", initial_state), ("d_state", d_state)):
        if s is not None:
            _check_state(s, (b, h, d, dv), q.device, name)
    initial_state = None if initial_state is None else initial_state.contiguous()
    d_state = None if d_state is None else d_state.contiguous()
    gq, gk, gv = _heads_like(q, d), _heads_like(k, d), _heads_like(v, dv)
    g0 = (torch.empty((b, h, d, dv), dtype=torch.float32, device=q.device) if want_d_initial
          else None)
    log_decay = log_decay.contiguous()
    (q, qs), (k, ks), (v, vs), (d_out, ds) = (_heads_view(x) for x in (q, k, v, d_out))
    (_, gqs), (_, gks), (_, gvs) = (_heads_view(x) for x in (gq, gk, gv))
    with _on_device(q.device):
        _, ws_bytes = _decay_plan(b, h, t, d, dv, code, True, int(segments),
                                  torch.cuda.current_device())
        workspace = _workspace(ws_bytes, q.device)
        st = N.lib().la_decay_chunked_bwd(
            _ptr(q), qs, _ptr(k), ks, _ptr(v), vs, _ptr(d_out), ds, _ptr(gq), gqs, _ptr(gk), gks,
            _ptr(gv), gvs, _ptr(log_decay), b, h, t, d, dv, code, _default_scale(scale, d),
            _ptr(initial_state), _ptr(d_state), _ptr(g0), _ptr(workspace), ws_bytes,
            int(segments), _stream_ptr(q.device))
    N.check(st, "la_decay_chunked_bwd")
    return gq, gk, gv, g0


def decay_attention_step(q, k, v, log_decay, state, scale=None) -> torch.Tensor:
    """One token of every sequence: q, k (b, h, d_qk), v (b, h, d_v); ``state``
    fp32 (b, h, d_qk, d_v) is updated in place.  Returns (b, h, d_v)."""
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
    if state.requires_grad:
        raise ValueError("state is updated in place: it may not require a gradient")
    sb, sh, sr, sc = state.stride()
    if ((sc != 1 and dv > 1) or (sr != dv and d > 1) or (sh < d * dv and h > 1)
            or (sb < d * dv and b > 1)):
        raise ValueError("state needs dense (d_qk, d_v) entries that do not overlap")
    if b > 1 and h > 1 and not (sb >= sh * (h - 1) + d * dv or sh >= sb * (b - 1) + d * dv):
        raise ValueError("the states of different sequences overlap")
    log_decay = log_decay.contiguous()
    q, k, v = (x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous() for x in (q, k, v))
    out = torch.empty((b, h, dv), dtype=q.dtype, device=q.device)
    with _on_device(q.device):
        st = N.lib().la_decay_step(
            _ptr(q), _Strides(*q.stride()), _ptr(k), _Strides(*k.stride()), _ptr(v),
            _Strides(*v.stride()), _ptr(out), _ptr(state), _Strides(sb, sh), _ptr(log_decay),
            b, h, d, dv, code, _default_scale(scale, d), _stream_ptr(q.device))
    N.check(st, "la_decay_step")
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


def _check_norm(x, weight, residual):
    code = _check_rows(x, "x")
    if residual is not None:
        _check_rows(residual, "residual", x)
    wcode = code
    if weight is not None:
        if not isinstance(weight, torch.Tensor):
            raise TypeError("weight must be a torch.Tensor")
        wcode = _dtype_code(weight)
        if tuple(weight.shape) != (x.shape[-1],) or weight.device != x.device:
            raise ValueError(f"weight must be ({x.shape[-1]},) on {x.device}")
    return code, wcode


def _row_views(*tensors):
    """The tensors (equal shapes, None allowed) as rows under three leading
    dimensions: ([tensor], [strides], shape).  Only rows that are not dense, or
    that more than three leading dimensions address, are copied."""
    first = next(t for t in tensors if t is not None)
    lead, d = first.shape[:-1], first.shape[-1]
    if all(t is None or t.is_contiguous() for t in tensors):
        shape = _Strides(1, 1, first.numel() // d)
        strides = _Strides(0, 0, d)
        return tensors, [strides] * len(tensors), shape
    if len(lead) > 3:
        return _row_views(*(None if t is None else t.contiguous() for t in tensors))
    pad = (1,) * (3 - len(lead))
    got, strides = [], []
    for t in tensors:
        if t is not None and t.stride(-1) != 1 and d > 1:
            t = t.contiguous()
        got.append(t)
        strides.append(None if t is None else _Strides(*((0,) * len(pad) + t.stride()[:-1])))
    return got, strides, _Strides(*(pad + tuple(lead)))


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, want_rstd: bool = False):
    """Forward pass of the norm (no autograd): (y, x + residual or None, fp32
    reciprocal root mean squares per row or None)."""
    code, wcode = _check_norm(x, weight, residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = torch.empty_like(y) if residual is not None else None
    rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if want_rstd
            else None)
    (x, residual), (xs, rs), shape = _row_views(x, residual)
    weight = None if weight is None else weight.contiguous()
    with _on_device(x.device):
        st = N.lib().la_rms_norm_fwd(
            _ptr(x), xs, _ptr(residual), rs, _ptr(weight), _ptr(y), _ptr(total), _ptr(rstd), shape,
            x.shape[-1], code, wcode, float(eps), _stream_ptr(x.device))
    N.check(st, "la_rms_norm_fwd")
    return y, total, rstd


def rms_norm_fp8(x, weight=None, residual=None, eps: float = 1e-6, group_size: int | None = None):
    """The norm with its output held in e4m3: (y, scales, x + residual or None),
    scales fp32 (..., d / group_size), one per row without a group size."""
    code, wcode = _check_norm(x, weight, residual)
    d = x.shape[-1]
    group = d if group_size is None else int(group_size)
    if group_size is not None and (group not in _FP8_GROUPS or d % group):
        raise ValueError(f"group_size must be None or one of {_FP8_GROUPS} dividing {d}, "
                         f"got {group_size}")
    y = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((*x.shape[:-1], d // group), dtype=torch.float32, device=x.device)
    total = (torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None
             else None)
    (x, residual), (xs, rs), shape = _row_views(x, residual)
    weight = None if weight is None else weight.contiguous()
    if group != d:  # whole 16-byte packs per group
        x, xs = _aligned_rows(x, xs, shape)
        residual, rs = _aligned_rows(residual, rs, shape)
        if weight is not None and weight.data_ptr() % 16:
            weight = weight.clone()
    with _on_device(x.device):
        st = N.lib().la_rms_norm_fp8(
            _ptr(x), xs, _ptr(residual), rs, _ptr(weight), _ptr(y), _ptr(scales), _ptr(total),
            shape, d, group, code, wcode, float(eps), _stream_ptr(x.device))
    N.check(st, "la_rms_norm_fp8")
    return y, scales, total


def _aligned_rows(t, strides, shape):
    """``t`` and its row strides, copied where its rows do not start at 16 bytes."""
    if t is None:
        return t, strides
    pack = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and all(s % pack == 0 for s in strides):
        return t, strides
    t = t.clone(memory_format=torch.contiguous_format)
    d = t.shape[-1]
    return t, _Strides(shape[1] * shape[2] * d, shape[2] * d, d)


def rms_norm_backward(s, weight, rstd, d_y, d_sum=None, want_d_weight: bool = True):
    """Gradients (of x and of the residual alike, of the weight or None) of
    ``rms_norm`` from its saved rows ``s`` (x + residual) and ``rstd``."""
    code, wcode = _check_norm(s, weight, None)
    _check_rows(d_y, "d_y", s)
    if d_sum is not None:
        _check_rows(d_sum, "d_sum", s)
    d = s.shape[-1]
    d_s = torch.empty(s.shape, dtype=s.dtype, device=s.device)
    d_w = torch.empty_like(weight, memory_format=torch.contiguous_format) if (
        want_d_weight and weight is not None) else None
    (s, d_y, d_sum), (ss, ys, us), shape = _row_views(s, d_y, d_sum)
    weight = None if weight is None else weight.contiguous()
    rstd = rstd.contiguous()
    with _on_device(s.device):
        ws_bytes = 0 if d_w is None else _norm_workspace(s.numel() // d, d,
                                                         torch.cuda.current_device())
        workspace = _workspace(ws_bytes, s.device)
        st = N.lib().la_rms_norm_bwd(
            _ptr(s), ss, _ptr(weight), _ptr(d_y), ys, _ptr(d_sum), us, _ptr(rstd), _ptr(d_s),
            _ptr(d_w), shape, d, code, wcode, _ptr(workspace), ws_bytes, _stream_ptr(s.device))
    N.check(st, "la_rms_norm_bwd")
    return d_s, d_w


@functools.lru_cache(maxsize=1024)
def _norm_workspace(rows, d, device_index):
    n = ctypes.c_size_t(0)
    N.check(N.lib().la_rms_norm_bwd_workspace_size(rows, d, ctypes.byref(n)),
            "la_rms_norm_bwd_workspace_size")
    return n.value


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
