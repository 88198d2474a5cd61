"""The packed-prompt and shared-prefix members of the C++ host side on the GPU (tests/cpp/test_packed.cpp), built by
tests/cpp/Makefile (part of __graft_entry__.build())."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "test_packed")


@pytest.mark.gpu
def test_cpp_packed():
    assert os.path.exists(BIN), f"{BIN} is missing: build it with make -C tests/cpp"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, f"C++ tests failed:\n{r.stdout}\n{r.stderr}"
    assert r.stdout.count("PASS ") == 4
