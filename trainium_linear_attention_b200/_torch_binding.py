"""The torch side of the gated linear recurrence, the short convolution and the
group norm (``csrc/torch_binding.cpp``): checks, allocations and gradients in C++
around the entry points of the native library that :mod:`._native` has loaded.
Loading is lazy and fails loudly: there is no fallback implementation.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading
from pathlib import Path

from . import _native as N

PATH = Path(__file__).resolve().parent / "lib" / "_la_torch.so"

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
                if not PATH.exists():
                    raise RuntimeError(f"{PATH} is missing; build it with "
                                       "`python -m trainium_linear_attention_b200.build`")
                lib = N.lib()
                loader = importlib.machinery.ExtensionFileLoader("_la_torch", str(PATH))
                spec = importlib.util.spec_from_file_location("_la_torch", PATH, loader=loader)
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
