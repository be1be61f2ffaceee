"""The C++ autograd graph (include/cortex_hip_graph.hpp) on the GPU where not all
tensors take a gradient: AdamW's parameters without one at every step, layers
without any (tests/cpp/layer_graph_more_test, built by __graft_entry__.build())."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "layer_graph_more_test")

pytestmark = pytest.mark.gpu


def test_cpp_layer_graph_more(hip):
    assert os.path.exists(BIN), "tests/cpp/layer_graph_more_test is not built (run __graft_entry__.build())"
    out = subprocess.run([BIN], capture_output=True, text=True, timeout=90)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "ALL OK" in out.stdout
