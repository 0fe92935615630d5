"""The torch binding of the gated recurrence, the short convolution and the group norm:
how it calls the library, with other functions in the place of its entry points."""

import contextlib
import ctypes

import pytest
import torch

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N
from trainium_linear_attention_b200 import _torch_binding as B

gpu = pytest.mark.gpu


def address(function):
    return ctypes.cast(function, ctypes.c_void_p).value


@contextlib.contextmanager
def bound(replaced):
    """The binding with functions of no arguments (more are passed, and ignored) for entries."""
    entries = {n: address(getattr(N.lib(), n)) for n in B._ENTRIES}
    B.module().bind({**entries, **{n: address(f) for n, f in replaced.items()}}, N.LaError)
    try:
        yield
    finally:
        B.module().bind(entries, N.LaError)


def calls(grad=False):
    x = torch.ones(2, 3, 8, device="cuda").requires_grad_(grad)
    w = torch.ones(8, 4, device="cuda").requires_grad_(grad)
    state, tail = torch.zeros(2, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda")
    return {"la_recurrence_fwd": lambda: T.gated_recurrence(x, x),
            "la_short_conv_fwd": lambda: T.causal_conv(x, w),
            "la_group_norm_fwd": lambda: T.group_norm(x, 2),
            "la_recurrence_step": lambda: T.gated_recurrence_step(x[:, 0], x[:, 0], state),
            "la_short_conv_step": lambda: T.causal_conv_step(x[:, 0], w, tail)}


@gpu
def test_the_interpreter_is_free_during_a_call():
    """Its own question whether the calling thread has its lock, as the entry point: 0, which is
    a call that went well, without it, 1 with it, a status that raises."""
    for grad in (False, True):
        for name, call in calls(grad).items():
            with bound({name: ctypes.pythonapi.PyGILState_Check}):
                call()


@gpu
def test_statuses_raise_their_error():
    """A status other than ok is a LaError that has it, from calls and from backward passes
    (which run on the engine's thread)."""
    unsupported = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: N.LA_ERR_UNSUPPORTED)
    for name, call in calls().items():
        with bound({name: unsupported}), pytest.raises(N.LaError, match=name) as caught:
            call()
        assert caught.value.status == N.LA_ERR_UNSUPPORTED
    for name, call in calls(grad=True).items():
        if name.endswith("_fwd"):
            y, name = call(), name.replace("_fwd", "_bwd")
            with bound({name: unsupported}), pytest.raises(N.LaError, match=name) as caught:
                y.sum().backward()
            assert caught.value.status == N.LA_ERR_UNSUPPORTED
