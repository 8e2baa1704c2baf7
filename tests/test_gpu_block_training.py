"""A step of the residual block's training by the published rule for the
shape: an orthogonalised update of a matrix that maps k inputs to n outputs is
scaled by sqrt(max(1, n / k))."""
import numpy as np
import pytest

from tests import blockops as bo
from tests.test_gpu_residual_block import _step64
from tinyhvm_amd import residual_block as rb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


@pytest.mark.parametrize("rows,width,hidden", [(48, 64, 160), (7, 33, 129), (130, 96, 80)], ids=str)
def test_step(hip, rows, width, hidden):
    block = rb.ResidualBlock(rows, width, hidden, seed=3)
    try:
        rng = np.random.default_rng(4)
        x, target = rng.standard_normal((2, rows, width)).astype(np.float32)
        p = {k: block.get(k).astype(np.float64) for k in block.shapes}
        block.put("x", x)
        block.put("target", target)
        block.step(lr=0.01, lr_vectors=0.002)
        y, dx, g, new = _step64(p, x.astype(np.float64), target.astype(np.float64), 0.01, 0.002)
        for name in ("w1", "w2"):
            k, n = p[name].shape
            new[name], _ = bo.muon(p[name], g[name], np.zeros_like(p[name]), 0.01, np.sqrt(max(1.0, n / k)), 0.0, 0.95, 1, 5)

        def near(name, want, tol):
            off = np.linalg.norm(block.get(name).astype(np.float64) - want) / (np.linalg.norm(want) + 1e-30)
            assert off <= tol, (name, off)

        # the tolerances of the step's first test: 100 roundings through the layers, which the updates multiply
        near("y", y, 1e-5)
        near("dx", dx, 1e-5)
        for name in g:
            near("d" + name, g[name], 1e-5)
        for name in new:
            near(name, new[name], 1e-4)
    finally:
        block.close()
