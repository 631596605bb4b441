"""What the Makefile builds where there is no torch: the C-ABI, without the Python module."""
import os
import subprocess

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-ext_amd")


def _make(*args):
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_libraries_without_torch(tmp_path):
    python = tmp_path / "python3"
    python.write_text("#!/bin/sh\nexec /usr/bin/env python3 -S -E \"$@\"\n")  # no site-packages
    python.chmod(0o755)
    for interpreter in (str(python), str(tmp_path / "none")):
        out = _make(f"PYTHON={interpreter}")
        assert "libmi355x_dot.so" in out and "libTritonExtPassInfra.so" in out
        assert "_tx_calls.so" not in out


def test_libraries_and_module_with_torch():
    out = _make()
    assert "libmi355x_dot.so" in out and "_tx_calls.so" in out
