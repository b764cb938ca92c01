"""Runs tests/host_cpp/test_paged_sizes.cc: sizes that the paged objects of the C++ host mirror refuse."""
import os
import subprocess

import pytest

BINARY = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_cpp", "_build", "test_paged_sizes")


@pytest.mark.gpu
def test_cpp_paged_sizes():
    assert os.path.exists(BINARY), "build first: python __graft_entry__.py"
    run = subprocess.run([BINARY], capture_output=True, text=True, timeout=120)
    print(run.stdout[-2000:], run.stderr[-2000:])
    assert run.returncode == 0 and "all sizes refused" in run.stdout
