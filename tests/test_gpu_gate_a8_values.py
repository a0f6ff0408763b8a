"""Runs the C++ gate over every value of the 8-bit rows, their products and log probabilities
(tests/cpp/gate_a8_values.cpp, built by __graft_entry__.build())."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

GATE = os.path.join(os.path.dirname(__file__), "cpp", "_build", "gate_a8_values")


def test_cpp_gate_a8_values():
    assert os.path.exists(GATE), "gate not built: run __graft_entry__.build()"
    r = subprocess.run([GATE], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "gate_a8_values: PASS" in r.stdout
