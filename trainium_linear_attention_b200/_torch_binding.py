"""The torch side of the gated linear recurrence, the short convolution and the
group norm (``csrc/torch_binding.cpp``): checks, allocations and gradients in C++
around the entry points of the native library that :mod:`._native` has loaded.
Loading is lazy and fails loudly: there is no fallback implementation.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import sysconfig
import threading
from pathlib import Path

import torch

from . import _native as N

LIB_DIR = Path(__file__).resolve().parent / "lib"


def path() -> Path:
    """The extension for this interpreter and this torch, whose layouts are compiled into
    it: one built for others has another name and is not loaded."""
    return LIB_DIR / (f"_la_torch.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}"
                      f".abi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}.so")


_ENTRIES = tuple(n for n in N.EXPORTED_SYMBOLS
                 if n.startswith(("la_recurrence_", "la_short_conv_", "la_group_norm_")))

_lock = threading.Lock()
_module = None


def module():
    """The loaded extension, bound to the native library's entry points."""
    global _module
    if _module is None:
        with _lock:
            if _module is None:
                file = path()
                if not file.exists():
                    raise RuntimeError(f"{file} (the one for this Python and torch) is missing; "
                                       "build it with "
                                       "`python -m trainium_linear_attention_b200.build`")
                lib = N.lib()
                loader = importlib.machinery.ExtensionFileLoader("_la_torch", str(file))
                spec = importlib.util.spec_from_file_location("_la_torch", file, loader=loader)
                loaded = importlib.util.module_from_spec(spec)
                loader.exec_module(loaded)
                loaded.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
                             for n in _ENTRIES}, N.LaError)
                _module = loaded
    return _module


def silu(activation) -> bool:
    """Whether ``activation`` is "silu"; None is none, anything else an error."""
    if activation is None:
        return False
    if activation == "silu":
        return True
    raise ValueError(f"activation must be None or 'silu', got {activation!r}")
