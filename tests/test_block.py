"""The residual block's definitions in 64 bits (tests/blockops.py), which the
GPU tests compare the kernels with: against torch's own, and the calls'
refusal without a device."""
import numpy as np
import pytest
import torch

from tests import blockops as bo


@pytest.mark.parametrize("name", bo.ACTS)
def test_activations(name):
    z = torch.linspace(-9, 9, 301, dtype=torch.float64, requires_grad=True)
    f = {"none": lambda v: v * 1.0, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": torch.nn.functional.silu}[name]
    y = f(z)
    g, = torch.autograd.grad(y.sum(), z)
    at = z.detach().numpy()
    assert np.allclose(bo.act(name, at), y.detach().numpy(), rtol=1e-12, atol=1e-14)
    assert np.allclose(bo.slope(name, at)[at != 0], g.numpy()[at != 0], rtol=1e-10, atol=1e-13)


def test_layer_norm():
    rng = np.random.default_rng(1)
    x, gamma, beta, dy = rng.standard_normal((7, 33)), rng.standard_normal(33), rng.standard_normal(33), rng.standard_normal((7, 33))
    t = [torch.from_numpy(v).requires_grad_() for v in (x, gamma, beta)]
    y = torch.nn.functional.layer_norm(t[0], (33,), t[1], t[2], 1e-5)
    got, mean, rstd = bo.layer_norm(x, gamma, beta, 1e-5)
    assert np.allclose(got, y.detach().numpy(), rtol=1e-12, atol=1e-12)
    for a, b in zip(bo.layer_norm_grad(dy, x, mean, rstd, gamma, None), torch.autograd.grad(y, t, torch.from_numpy(dy))):
        assert np.allclose(a, b.numpy(), rtol=1e-10, atol=1e-11)


@pytest.mark.parametrize("shape", [(20, 30), (30, 20), (16, 16)])
def test_orthogonalised_step(shape):
    """The step's polynomial acts on the singular values alone."""
    rng = np.random.default_rng(2)
    p, g = rng.standard_normal(shape), rng.standard_normal(shape)
    new, m = bo.muon(p, g, np.zeros(shape), 0.5, 2.0, 0.25, 0.9, 0, 5)
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / (np.linalg.norm(g) + 1e-7)
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    assert np.array_equal(m, g)
    assert np.allclose(new, (1 - 0.5 * 0.25) * p - 0.5 * 2.0 * (u * s) @ vt, rtol=1e-9, atol=1e-9)
    assert s[s > 0.6].size >= s.size - 1


def test_calls_without_a_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    L = bo.lib()
    one = bo.ids([1])
    assert L.thvm_hip_layer_norm(1, 0, 0, 2, 0, 0, 4, 4, 1e-5, 0) == -1
    assert L.thvm_hip_layer_norm_grad(1, 0, 0, 2, 3, 4, 5, 0, 0, 4, 4, 0) == -1
    assert L.thvm_hip_linear(1, 0, 2, 3, 0, 0, 0, 4, 4, 4, 0) == -1
    assert L.thvm_hip_linear_grad(1, 0, 0, 2, 0, 3, 4, 0, 4, 4, 4, 0) == -1
    assert L.thvm_hip_muon_step(one, one, one, 1, 4, 4, 0.1, 1.0, 0.0, 0.9, 1, 5, 0) == -1
