"""The drop-in C++ header's 8-bit paged-cache calls from a plain C++ program,
built by tests/dropin/Makefile and run as its own process: it checks every step of
a small server, eager and captured, and prints one line per check."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "dropin", "paged_fp8_test")


def test_paged_fp8_header_program():
    assert os.path.exists(BIN), "tests/dropin/paged_fp8_test is missing: run __graft_entry__.build()"
    res = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(res.stdout, res.stderr, flush=True)
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-2000:]
    assert "ALL PASS" in res.stdout
    assert res.stdout.count("[PASS]") == 42
