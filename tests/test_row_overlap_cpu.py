"""Which rows share memory, against a look at every pair of them. Runs on CPU."""
import os
import subprocess

import pytest

from msnhnet_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("rows") / "row_overlap_check")
    subprocess.run([build._host_cxx(), "-O1", "-std=c++17", "-Wall", "-o", exe, os.path.join(HERE, "row_overlap_check.cpp")], check=True)
    return exe


@pytest.mark.parametrize("seed", range(4))
def test_rows_that_share_memory_are_found(check, seed):
    r = subprocess.run([check, str(seed)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
