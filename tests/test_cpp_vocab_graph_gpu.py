"""The C++ autograd graph (include/cortex_hip_graph.hpp) on the GPU from tokens to
losses over a vocabulary: embedding, layer norm, log probabilities, distillation
(tests/cpp/vocab_graph_test, built by __graft_entry__.build())."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "vocab_graph_test")

pytestmark = pytest.mark.gpu


def test_cpp_vocab_graph(hip):
    assert os.path.exists(BIN), "tests/cpp/vocab_graph_test is not built (run __graft_entry__.build())"
    out = subprocess.run([BIN], capture_output=True, text=True, timeout=90)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "ALL OK" in out.stdout
