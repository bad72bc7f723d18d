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


def load() -> None:
    """Load the binding (once) and bind it to the CUDA library."""
    global _loaded
    with _lock:
        if _loaded:
            return
        _capi.lib()  # raises with the build command if it is not built
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"spikegpt_b200: torch binding {LIB_PATH} is not built; run "
                "`python spikegpt-myelin_b200/build.py` (or __graft_entry__.build())"
            )
        torch.ops.load_library(str(LIB_PATH))
        torch.ops.spikegpt_b200.bind_library(str(_capi.library_path()))
        _loaded = True


def op(name: str):
    """The operator ``spikegpt_b200::<name>``."""
    load()
    return getattr(torch.ops.spikegpt_b200, name).default


def op_if_built(name: str):
    """The operator, or None while the libraries are not built (``op`` then tells why):
    modules look theirs up when they are imported, so that calls need no look-up."""
    return op(name) if LIB_PATH.exists() and _capi.library_path().exists() else None
