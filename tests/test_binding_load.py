"""CPU tests of when the torch binding of the mixer operators is loaded: at their first
call, so that a missing or damaged binding leaves the rest of the package working."""

from __future__ import annotations

import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parent.parent / "spikegpt-myelin_b200"


def _run(root: Path, code: str) -> subprocess.CompletedProcess:
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(root)!r})\n{code}"],
                          capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("binding", ["damaged", "missing"])
def test_a_bad_binding_stops_only_the_operators_that_need_it(tmp_path, binding):
    """The package from a copy whose binding is no library: it imports, the WKV operators and
    the C ABI are there, and the mixer operators say what is wrong."""
    shutil.copytree(PACKAGE / "spikegpt_b200", tmp_path / "spikegpt_b200", ignore=shutil.ignore_patterns("__pycache__"))
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "libspikegpt_wkv.so").symlink_to(PACKAGE / "lib" / "libspikegpt_wkv.so")
    if binding == "damaged":
        (tmp_path / "lib" / "libspikegpt_torch.so").write_bytes(b"not a library")
    done = _run(tmp_path, """
import torch, spikegpt_b200 as sg
from spikegpt_b200 import selective_model
assert sg._capi.PKG_ROOT != None and str(sg._capi.PKG_ROOT) in sg.__file__
assert sg._capi.lib().selective_scan_state_size(1, 8, 4, 4) == 64
k = torch.zeros(1, 3, 4)
try:
    sg.weighted_key_value_cuda(k, k, k[0, 0], k[0, 0])
    raise SystemExit("a CPU tensor was taken")
except (ValueError, NotImplementedError, RuntimeError) as e:
    assert "libspikegpt_torch" not in str(e)
sg.quantize_q4(torch.zeros(4, 64), 32)
for call in (lambda: sg.layer_norm(k), lambda: sg.causal_conv(k, torch.zeros(4, 4))):
    try:
        call()
        raise SystemExit("an operator ran without its binding")
    except (OSError, RuntimeError) as e:
        assert "libspikegpt_torch.so" in str(e), e
print("fine")
""")
    assert done.returncode == 0 and "fine" in done.stdout, done.stdout + done.stderr


def test_importing_the_package_loads_no_binding_and_compiling_a_caller_does():
    done = _run(PACKAGE, """
import torch, spikegpt_b200 as sg
from spikegpt_b200 import _native
assert "libspikegpt_torch" not in open("/proc/self/maps").read() and not _native._loaded
x, w = torch.zeros(2, 5, 8, device="meta", requires_grad=True), torch.zeros(8, 4, device="meta")
y = torch.compile(lambda v: sg.layer_norm(sg.causal_conv(v, w)), backend="eager", fullgraph=True)(x)
assert y.shape == x.shape and y.requires_grad and _native._loaded
print("fine")
""")
    assert done.returncode == 0 and "fine" in done.stdout, done.stdout + done.stderr


def test_another_torch_means_another_binding(tmp_path, monkeypatch):
    """The build takes the binding for current only if the torch it was built against is
    the one that is installed."""
    import importlib.util
    import os

    spec = importlib.util.spec_from_file_location("recipe", PACKAGE / "build.py")
    recipe = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(recipe)
    monkeypatch.setattr(recipe, "TORCH_LIB", tmp_path / "libspikegpt_torch.so")
    assert not recipe._binding_current()
    recipe.TORCH_LIB.write_bytes(b"")
    os.utime(recipe.TORCH_LIB, (2**32, 2**32))
    assert not recipe._binding_current()  # built before there was a stamp
    recipe._torch_stamp().write_text(recipe.version("torch"))
    assert recipe._binding_current() and recipe._start_binding(False) is None
    os.utime(recipe.TORCH_LIB, (0, 0))  # older than its source
    assert not recipe._binding_current()
    os.utime(recipe.TORCH_LIB, (2**32, 2**32))
    monkeypatch.setattr(recipe, "version", lambda name: "0.0.1")
    assert not recipe._binding_current()
