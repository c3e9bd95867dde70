"""The build's two parts: the library needs nvcc alone, the torch binding torch as well."""
import os
import subprocess
import sys

from conftest import ROOT
from potpori_b200 import build as b


def test_library_builds_without_torch():
    """Where torch is not installed, build() makes the library and leaves the binding as it is."""
    script = """
import sys
sys.modules["torch"] = None  # as if it were not installed
from potpori_b200 import build as b
done = []
b.build_library = lambda verbose=False: done.append("library")
assert b.build(force=True) == b.LIB and done == ["library"]
b.stale = lambda target=b.LIB, deps=b.DEPS: True
assert b.build() == b.LIB and done == ["library"] * 2
"""
    before = os.path.getmtime(b.BINDING)
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "torch is not installed" in r.stderr and os.path.getmtime(b.BINDING) == before


def test_binding_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    abi = b.binding_abi()
    assert abi.startswith("torch ")
    built = []
    monkeypatch.setattr(b, "stale", lambda target=b.LIB, deps=b.DEPS: False)
    monkeypatch.setattr(b, "build_binding", built.append)
    monkeypatch.setattr(b, "BINDING_BUILT_FOR", str(tmp_path / "built"))
    b.build()  # not known what it was built for
    (tmp_path / "built").write_text(abi)
    b.build()
    (tmp_path / "built").write_text(abi.replace("torch ", "torch 1."))
    b.build()
    assert built == [abi, abi]


def test_torch_without_package_metadata(monkeypatch):
    import importlib.metadata

    import torch

    def absent(name):
        raise importlib.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(importlib.metadata, "version", absent)
    assert b.binding_abi().startswith(f"torch {torch.__version__} ")
