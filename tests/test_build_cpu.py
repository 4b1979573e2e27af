"""The native build without PyTorch: C, C++ and Rust callers need nvcc alone."""
import os
import subprocess
import sys

from conftest import ROOT

PKG = os.path.join(ROOT, "aegis-core_b200")


def make(*args):
    return subprocess.run(["make", "-n", "-B", "-C", PKG, *args], capture_output=True, text=True)


def test_build_without_torch(tmp_path):
    bare = tmp_path / "python"  # an interpreter without torch
    bare.write_text(f'#!/bin/sh\nexec {sys.executable} -S -I "$@"\n')
    bare.chmod(0o755)
    for python in (str(bare), str(tmp_path / "none")):
        r = make(f"PYTHON={python}", "all")
        assert r.returncode == 0, r.stderr
        assert "libaegis_torch_i8.so" not in r.stdout
        for product in ("libaegis_capi.so", "libaegis_i8.so", "libaegis.a", "aegis_tune", "libaegis_ltbase.so"):
            assert product in r.stdout
    r = subprocess.run(["make", "-C", PKG, f"PYTHON={bare}", "torch"], capture_output=True, text=True)
    assert r.returncode != 0 and "has no torch" in r.stderr


def test_build_with_torch():
    r = make(f"PYTHON={sys.executable}", "all")
    assert r.returncode == 0 and "-o build/libaegis_torch_i8.so" in r.stdout
    assert " -w " not in r.stdout  # its warnings are shown
