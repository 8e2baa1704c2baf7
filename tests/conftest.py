import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


# The CPU tests inspect the matrix-core path on small fixtures, below the
# size heuristics; the GPU tests set their own modes per module.
os.environ.setdefault("THVM_HIP_DENSE_FORCE", "1")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU")


def pytest_collection_modifyitems(items):
    # Its expected matrices take sqrt(max(1, rows / cols)) of [inputs][outputs]; the published factor is
    # sqrt(max(1, outputs / inputs)). test_gpu_block_training.py holds the same step with that one.
    for item in items:
        if item.nodeid.startswith("tests/test_gpu_residual_block.py::test_step"):
            item.add_marker(pytest.mark.xfail(strict=True, reason="expects the shape factor of the transposed matrix"))
