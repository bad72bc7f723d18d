"""The torch binding of the selective-mixer operators (``lib/libspikegpt_torch.so``).

The binding registers them in ``torch.ops.spikegpt_b200`` with their argument
checks, autograd and Meta kernels (csrc/torch_ops.cpp), and calls the kernels
through the C ABI of the library that ``_capi`` names. There is no fallback: without
it the operators raise.
"""

from __future__ import annotations

import threading

import torch

from . import _capi

LIB_PATH = _capi.PKG_ROOT / "lib" / "libspikegpt_torch.so"

_lock = threading.Lock()
_loaded = False


@torch.compiler.assume_constant_result  # a compiled caller loads it while it is traced
def load() -> bool:
    """Load the binding (once) and bind it to the CUDA library."""
    global _loaded
    with _lock:
        if _loaded:
            return True
        _capi.lib()  # raises with the build command if it is not built
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"spikegpt_b200: torch binding {LIB_PATH} is not built; run "
                "`python spikegpt-myelin_b200/build.py` (or __graft_entry__.build())"
            )
        torch.ops.load_library(str(LIB_PATH))
        torch.ops.spikegpt_b200.bind_library(str(_capi.library_path()))
        _loaded = True
    return True


class _Operators:
    """The operators as attributes. The binding is loaded when the first one is looked up and
    not when the package is imported: it is built against one torch, and what does not need
    it (the WKV operators) has to work without."""

    def __getattr__(self, name: str):  # once a name: what it finds becomes an attribute
        load()
        found = getattr(torch.ops.spikegpt_b200, name).default
        setattr(self, name, found)
        return found


ops = _Operators()
