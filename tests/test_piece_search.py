"""The search for a piece of the attention's work line, compiled for the host: units within
a kv head past 32 bits (1.5 million new tokens and more), and small random settings."""
import os
import subprocess

from gdn_18646_b200 import build


def test_piece_search_against_a_walk(tmp_path):
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "piece_search.cu")
    exe = str(tmp_path / "piece_search")
    r = subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "-O2", "-I" + build.INCLUDE, src, "-o", exe, "-cudart", "static"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr
