"""Loads the extension module ``lib/_host.so`` (host side of the products over packed rows and of the
Adam step over many tensors) and hands it the C entries of the CUDA library.  Like the library it has
no fallback.  Unlike the library it is bound to the Python and the torch that it was built for."""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from pathlib import Path

import torch      # (also for the extension's symbols)

from . import _lib
from .build import HOST_LIB, HOST_STAMP, host_abi

_ENTRIES = ("mole_grouped_mm", "mole_grouped_mm_workspace_bytes", "mole_grouped_mm_wgrad",
            "mole_grouped_mm_wgrad_workspace_bytes", "mole_quantize_rows", "mole_grouped_mm_i8", "mole_adam_multi",
            "mole_last_error_string")


def _load(path: Path = HOST_LIB, stamp: Path = HOST_STAMP):
    how = "Build it with `python mole_b200/build.py` (needs nvcc and a C++ compiler)."
    if not path.exists():
        raise ImportError(f"{path} is missing.  {how}")
    if stamp.exists() and stamp.read_text() != host_abi():
        raise ImportError(f"{path} was built for {stamp.read_text()}; here is {host_abi()}.  {how}")
    loader = importlib.machinery.ExtensionFileLoader("_host", str(path))
    try:
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host", loader))
        loader.exec_module(module)
    except ImportError as e:
        raise ImportError(f"{path} does not load with {host_abi()} ({e}): it was built for another.  {how}") from e
    module.bind({name: C.cast(getattr(_lib.lib, name), C.c_void_p).value for name in _ENTRIES},
                _lib.check, torch.cuda.OutOfMemoryError)
    return module


host = _load()
