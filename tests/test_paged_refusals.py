"""Layouts of the paged-cache and norm entry points, checked on the CPU: each scenario of paged_refusals.py runs the library's
host code in a child process over a stand-in of the HIP runtime."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
DRIVER = os.path.join(HERE, "paged_refusals.py")


@pytest.mark.parametrize("name", ["pages_that_meet", "rows_that_meet_their_own", "norm_rows_that_meet_their_own"])
def test_layouts(name):
    assert os.path.exists(os.path.join(HERE, "cpp", "bin", "libfakehip.so")), "run __graft_entry__.build()"
    r = subprocess.run([sys.executable, DRIVER, name], capture_output=True, text=True, timeout=120)
    print(r.stdout[-3000:])
    assert r.returncode == 0, r.stderr[-3000:]
