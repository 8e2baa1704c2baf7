"""The residual block's training (tinyhvm_amd/residual_block.py): a step's
values against the same step in 64 bits, and a run whose loss falls."""
import numpy as np
import pytest

from tests import blockops as bo
from tinyhvm_amd import residual_block as rb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


def _step64(p, x, target, lr, lr_vectors):
    """The block's first step from parameters p, by the definitions."""
    h, mean, rstd = bo.layer_norm(x, p["gamma"], p["beta"], 1e-5)
    z = h @ p["w1"] + p["b1"]
    a = bo.act("gelu", z)
    y = x + a @ p["w2"] + p["b2"]
    dy = 2 * (y - target) / y.size
    da = dy @ p["w2"].T
    dz = da * bo.slope("gelu", z)
    dx, dgamma, dbeta = bo.layer_norm_grad(dz @ p["w1"].T, x, mean, rstd, p["gamma"], dy)
    g = {"w1": h.T @ dz, "b1": dz.sum(0), "w2": a.T @ dy, "b2": dy.sum(0), "gamma": dgamma, "beta": dbeta}
    new = {}
    for k in p:
        if p[k].ndim == 2:
            new[k], _ = bo.muon(p[k], g[k], np.zeros_like(p[k]), lr, np.sqrt(max(1.0, p[k].shape[0] / p[k].shape[1])), 0.0, 0.95, 1, 5)
        else:      # adam's first step: the gradient's sign, but for epsilon
            new[k] = p[k] - lr_vectors * g[k] / (np.abs(g[k]) + 1e-8)
    return y, dx, g, new


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

        def near(got, want, tol):
            off = np.linalg.norm(got.astype(np.float64) - want) / (np.linalg.norm(want) + 1e-30)
            assert off <= tol, off

        # sums of up to 200 products in 32 bits through three layers: 1e-5 of the norm is over 100 of their roundings
        near(block.get("y"), y, 1e-5)
        near(block.get("dx"), dx, 1e-5)
        for k in g:
            near(block.get("d" + k), g[k], 1e-5)
        for k in new:
            # the matrices' update multiplies what is off by up to 3.5 ** 5; adam's divides by the gradient's size
            near(block.get(k), new[k], 1e-4)
    finally:
        block.close()


@pytest.mark.parametrize("graph", [False, True])
def test_training(hip, graph):
    losses = rb.main(["--rows", "200", "--width", "64", "--hidden", "128", "--steps", "40"] + (["--graph"] if graph else []))
    hip.thvm_hip_init()
    assert losses[-1] < 0.5 * losses[0], losses
