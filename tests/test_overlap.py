"""Whether two layouts of pages share memory (transformer_amd/csrc/overlap.h), against lists of their places, on the CPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_layouts_that_share_memory(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "overlap_model")
    subprocess.run([gxx, "-O2", "-std=c++17", "-o", exe, os.path.join(HERE, "overlap_model.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    words = r.stdout.split()
    counts = [int(words[i]) for i in (1, 2, 4, 5)]
    assert min(counts) > 1000
