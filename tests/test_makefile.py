"""What the package's Makefile builds, and from what (no GPU, nothing is
built)."""

import shutil
import subprocess
import sys

import pytest

from conftest import PKG

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def dry_run(*args):
    return subprocess.run(["make", "-n", "-C", PKG, *args], capture_output=True, text=True, check=True).stdout


def python(tmp_path, version):
    """An interpreter that answers every question with `version`."""
    p = tmp_path / f"python-{version}"
    p.write_text(f"#!/bin/sh\necho {version}\n")
    p.chmod(0o755)
    return f"PYTHON={p}"


def test_the_library_needs_no_torch():
    out = dry_run("-B", "PYTHON=/does/not/exist")
    assert "libiec_cuda.so" in out and "csrc/capi.cpp" in out
    assert "binding" not in out and "torch" not in out


def test_the_binding_is_built_for_its_torch(tmp_path):
    assert "ops_binding.cpp" in dry_run("-B", "binding", f"PYTHON={sys.executable}")
    out = dry_run("binding", python(tmp_path, "0.0-other"))  # not what it was built for
    assert "ops_binding.cpp" in out and "libiec_cuda" not in out
