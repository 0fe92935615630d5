"""The torch binding of the gated recurrence, the short convolution and the group norm:
how it calls the library, with other functions in the place of its entry points."""

import contextlib
import ctypes
import subprocess
import threading
from types import SimpleNamespace

import pytest
import torch

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N
from trainium_linear_attention_b200 import _torch_binding as B
from trainium_linear_attention_b200 import build as build_module

gpu = pytest.mark.gpu


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    """The file's name has the interpreter and the torch whose layouts it was built with."""
    assert B.path().exists()
    monkeypatch.setattr(B, "_module", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(RuntimeError, match="0.0.1.* is missing.*build"):
        T.group_norm(torch.zeros(2, 8), 2)


def test_what_a_binding_is_built_for(monkeypatch, tmp_path):
    """Another torch gets a file of its own; the same one, and an older file than the sources,
    are taken and built again."""
    ran = []

    def compiler(cmd, **_):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(B, "LIB_DIR", tmp_path)
    monkeypatch.setattr(subprocess, "run", compiler)
    build_module._build_binding(False)
    build_module._build_binding(False)
    assert len(ran) == 1 and B.path().exists()
    build_module._build_binding(True)
    assert len(ran) == 2
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build_module._build_binding(False)
    assert len(ran) == 3 and len(list(tmp_path.iterdir())) == 2


def test_the_library_is_linked_without_the_binding(monkeypatch, tmp_path):
    """A binding that fails to build is an error, but the C library is there by then."""
    (tmp_path / "a.cu").write_text("")
    monkeypatch.setattr(build_module, "CSRC", tmp_path)
    monkeypatch.setattr(build_module, "BUILD", tmp_path)
    monkeypatch.setattr(build_module, "LIB", tmp_path / "lib" / "library.so")
    monkeypatch.setattr(build_module, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(build_module, "_compile", lambda src, obj, verbose: obj.write_text(""))

    def link(cmd, **_):
        open(cmd[cmd.index("-o") + 1], "w").close()
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    def fails(force):
        raise RuntimeError("no headers")

    monkeypatch.setattr(subprocess, "run", link)
    monkeypatch.setattr(build_module, "_build_binding", fails)
    with pytest.raises(RuntimeError, match="no headers"):
        build_module.build()
    assert build_module.LIB.exists()


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


@gpu
def test_threads_on_streams_of_their_own():
    """Two threads' calls and backward passes at a time, of sizes that differ in the kernels'
    shared memory, give what they give one after the other."""
    def chain(c, seed):
        gen = torch.Generator().manual_seed(seed)
        x, gate = (torch.randn(3, 200, c, generator=gen).bfloat16().cuda().requires_grad_()
                   for _ in range(2))
        w = torch.randn(c, 4, generator=gen).cuda().requires_grad_()
        lam = -torch.rand(c, generator=gen).cuda().requires_grad_()

        def run():
            h = T.gated_recurrence(T.causal_conv(x, w, activation="silu"), gate, lam)
            y = T.group_norm(h, 1, gate=gate, activation="silu")
            return [y.detach(), *torch.autograd.grad(y, [x, gate, w, lam], torch.ones_like(y))]
        return run

    runs = [chain(c, i) for i, c in enumerate((63, 21, 64, 128))]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    found, failed = [[] for _ in runs], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    found[i].append(runs[i]())
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 (told to the test's thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(runs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for i, expected in enumerate(want):
        for got in found[i]:
            assert all(torch.equal(a, b) for a, b in zip(expected, got))
