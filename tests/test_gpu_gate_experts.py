"""Runs the C++ gate over the layers of experts and the products with an epilogue
(tests/cpp/gate_experts.cpp, built by __graft_entry__.build())."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

GATE = os.path.join(os.path.dirname(__file__), "cpp", "_build", "gate_experts")


def test_cpp_gate_experts():
    assert os.path.exists(GATE), "gate not built: run __graft_entry__.build()"
    r = subprocess.run([GATE], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "gate_experts: PASS" in r.stdout
