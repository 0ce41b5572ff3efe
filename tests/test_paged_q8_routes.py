"""What the entry points over Q8_0 pages and reading pages back refuse and take, checked on the CPU: each scenario of
paged_q8_routes.py runs the library's host code in a child process over a stand-in of the HIP runtime."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
DRIVER = os.path.join(HERE, "paged_q8_routes.py")


@pytest.mark.parametrize("name", ["refusals", "accepted", "layouts", "limits", "views"])
def test_route(name):
    assert os.path.exists(os.path.join(HERE, "cpp", "bin", "libfakehip.so")), "run __graft_entry__.build()"
    r = subprocess.run([sys.executable, DRIVER, name], capture_output=True, text=True, timeout=120)
    print(r.stdout[-3000:])
    assert r.returncode == 0, r.stderr[-3000:]
