"""Which thread forms which sine of a token that is appended, for tokens of every number of threads, on the
host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_pair_is_formed_once(tmp_path):
    exe = str(tmp_path / "sine_share_host")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "triton-ext_amd", "csrc"),
                    os.path.join(ROOT, "tests", "sine_share_host.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
