"""The arithmetic that places a paged call's tokens, keys and pages, against the
definition (CPU; csrc/fl_paged_map.h compiled for the host with its sanitizers)."""

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_paged_map(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "paged_map_check")
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "paged_map_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe, "2000"], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
