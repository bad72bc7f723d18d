"""Build recipe for libspikegpt_wkv.so (sm_100a) and its torch binding, in-tree.

    python spikegpt-myelin_b200/build.py          # builds lib/libspikegpt_{wkv,torch}.so

nvcc cross-compiles for sm_100a without a GPU; the binding (csrc/torch_ops.cpp) is
host code against torch's headers. The shared libraries are placed in
``spikegpt-myelin_b200/lib/`` so that they travel with the source tree; the
Python package loads them from there.
"""

from __future__ import annotations

import os
import subprocess
import sys
from importlib.metadata import version
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
LIB_DIR = PKG_ROOT / "lib"
LIB = LIB_DIR / "libspikegpt_wkv.so"
SOURCES = [CSRC / "wkv_capi.cu", CSRC / "mixer_capi.cu"]
TORCH_LIB = LIB_DIR / "libspikegpt_torch.so"
TORCH_SOURCE = CSRC / "torch_ops.cpp"
DEPS = SOURCES + sorted(CSRC.glob("*.cuh")) + [REPO_ROOT / "include" / "spikegpt_wkv.h"]

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
]


def nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(home) / "bin" / "nvcc"
    return str(cand) if cand.exists() else "nvcc"


def _newer(lib: Path, deps: list[Path]) -> bool:
    return lib.exists() and lib.stat().st_mtime >= max(p.stat().st_mtime for p in deps)


def _torch_stamp() -> Path:
    """The file that says which torch the binding was built against."""
    return TORCH_LIB.with_suffix(".torch")


def _binding_current() -> bool:
    """Built from this source, and against the torch that would load it: the binding uses
    torch's C++ interface, which another version may have changed."""
    stamp = _torch_stamp()
    return (
        _newer(TORCH_LIB, [TORCH_SOURCE, REPO_ROOT / "include" / "spikegpt_wkv.h"])
        and stamp.exists()
        and stamp.read_text() == version("torch")
    )


def _start_binding(force: bool) -> tuple[subprocess.Popen, Path] | None:
    """The compiler of the torch binding, started (it runs beside nvcc)."""
    if not force and _binding_current():
        return None
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    tmp = TORCH_LIB.with_name(TORCH_LIB.name + f".tmp{os.getpid()}")
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    # the system's g++, not $CXX: a compiler that links its own static libstdc++ into the
    # binding gives torch's exceptions and streams a second, uninitialised runtime
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(REPO_ROOT / "include"),
           *(a for p in [*include_paths(), str(cuda / "include")] for a in ("-isystem", p)), str(TORCH_SOURCE), "-o",
           str(tmp), *(f"-L{p}" for p in library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ldl"]
    return subprocess.Popen(cmd), tmp


def build(force: bool = False, verbose: bool = False) -> Path:
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    binding = _start_binding(force)
    try:
        lib = _build_kernels(force, verbose)
    finally:
        if binding is not None:
            status = binding[0].wait()
    if binding is not None:
        if status:
            raise subprocess.CalledProcessError(status, binding[0].args)
        binding[1].replace(TORCH_LIB)
        _torch_stamp().write_text(version("torch"))
    return lib


def _build_kernels(force: bool, verbose: bool) -> Path:
    if not force and LIB.exists():
        newest = max(p.stat().st_mtime for p in DEPS)
        if LIB.stat().st_mtime >= newest:
            return LIB
    tmp = LIB.with_name(LIB.name + f".tmp{os.getpid()}")
    cmd = [nvcc(), *NVCC_FLAGS, "-I", str(REPO_ROOT / "include"), "-I", str(CSRC)]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    objects = [LIB_DIR / f"{src.stem}.{os.getpid()}.o" for src in SOURCES]
    try:
        jobs = [subprocess.Popen([*cmd, "-c", str(src), "-o", str(obj)]) for src, obj in zip(SOURCES, objects)]
        status = [job.wait() for job in jobs]  # the sources compile side by side
        if any(status):
            raise subprocess.CalledProcessError(max(status, key=abs), cmd)
        subprocess.run([nvcc(), "-shared", *NVCC_FLAGS, *map(str, objects), "-o", str(tmp)], check=True)
    finally:
        for obj in objects:
            obj.unlink(missing_ok=True)
    tmp.replace(LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
