"""The serving operators' host side in C++ (csrc/torch_calls.cpp): a Python
module built next to ``libb200fa.so`` that checks tensors, allocates outputs
and calls the C ABI.  It is bound to the loaded library's entry points; there
is no fallback, a module that cannot be built or loaded raises."""

from __future__ import annotations

import ctypes as C
import importlib.util
import threading

import torch  # noqa: F401  (the module links against torch's libraries)

from . import build as _build
from . import lib

ENTRIES = ("b200fa_build_tables", "b200fa_rotary", "b200fa_append", "b200fa_paged_workspace_size", "b200fa_paged_fwd",
           "b200fa_last_error_string")

_lock = threading.Lock()
_module = None


def bind(module, so) -> None:
    """Points the module at the entry points of a loaded library."""
    module.bind({name: C.cast(getattr(so, name), C.c_void_p).value for name in ENTRIES}, lib.B200FAError)


def load():
    """The module, built first if its source changed."""
    global _module
    if _module is not None:
        return _module
    with _lock:
        if _module is None:
            path = _build.build_calls()
            spec = importlib.util.spec_from_file_location("fa_b200_calls", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            bind(module, lib.load())
            _module = module
    return _module
