"""Loads the extension module ``lib/_host.so`` (host side of the products over packed rows and of the
Adam step over many tensors) and hands it the C entries of the CUDA library.  Like the library it has
no fallback."""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from pathlib import Path

import torch      # (also for the extension's symbols)

from . import _lib

_PATH = Path(__file__).resolve().parent / "lib" / "_host.so"
_ENTRIES = ("mole_grouped_mm", "mole_grouped_mm_workspace_bytes", "mole_grouped_mm_wgrad",
            "mole_grouped_mm_wgrad_workspace_bytes", "mole_quantize_rows", "mole_grouped_mm_i8", "mole_adam_multi",
            "mole_last_error_string")


def _load():
    if not _PATH.exists():
        raise ImportError(f"{_PATH} is missing.  Build it with `python mole_b200/build.py` (needs nvcc and a C++ compiler).")
    loader = importlib.machinery.ExtensionFileLoader("_host", str(_PATH))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host", loader))
    loader.exec_module(module)
    module.bind({name: C.cast(getattr(_lib.lib, name), C.c_void_p).value for name in _ENTRIES},
                _lib.check, torch.cuda.OutOfMemoryError)
    return module


host = _load()
