"""What the autograd graph's layers and AdamW ask the library for
(tests/cpp/layer_graph_host_test.cpp: the caching pool over host memory and
stand-ins for the kernels, built with AddressSanitizer/UBSan; no GPU)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layer_graph_calls():
    cpp = os.path.join(ROOT, "tests", "cpp")
    out = subprocess.run(["make", "-s", "-C", cpp], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    run = subprocess.run([os.path.join(cpp, "layer_graph_host_test")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "ALL OK" in run.stdout
