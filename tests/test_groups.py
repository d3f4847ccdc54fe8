"""Groups of sequences that begin alike (karume_b200/csrc/kq_groups.h): boundaries that are in order never ask for more blocks of rows than the
launcher has, whatever the device arrays hold; those that are not are found out."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_groups_in_order_fit_their_grid(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path / "groups_check"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "karume_b200", "csrc"),
                    os.path.join(ROOT, "tests", "native", "groups_check.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout[-2000:]
    in_order, wild = (int(n) for n in done.stdout.split())
    assert in_order > 50000 and wild > 1000  # what the check is for does happen
