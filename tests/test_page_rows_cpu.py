"""Which rows of a page each load of a block takes, in every form, on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_of_every_form(tmp_path):
    exe = str(tmp_path / "page_rows_host")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "triton-ext_amd", "csrc"),
                    os.path.join(ROOT, "tests", "page_rows_host.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
