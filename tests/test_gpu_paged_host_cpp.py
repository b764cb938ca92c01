"""Runs tests/host_cpp/test_paged.cc: the paged cache of the C++ host mirror as a program uses it."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BINARY = os.path.join(HERE, "host_cpp", "_build", "test_paged")


@pytest.mark.gpu
def test_cpp_paged_steps():
    assert os.path.exists(BINARY), "build first: python __graft_entry__.py"
    run = subprocess.run([BINARY], capture_output=True, text=True, timeout=120)
    print(run.stdout[-2000:], run.stderr[-2000:])
    assert run.returncode == 0
    assert "all paged host tests passed" in run.stdout


def test_cpp_paged_test_is_built():
    assert os.path.exists(BINARY), "build first: python __graft_entry__.py"
