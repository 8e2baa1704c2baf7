"""What the residual block's operators make of single values: activations on
their own, NaN and infinities through them, and rows of nothing."""
import math

import numpy as np
import pytest

from tests import blockops as bo
from tests import blockplan as bp
from tests.blockops import ACTS, F16, F32, NP, U32
from tests.test_gpu_block import within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


# ---- rows of nothing ----

@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 700])
def test_statistics_of_empty_rows(hip, rows, dt):
    """The mean of no values is 0 / 0, and so is what stands on it."""
    y, mean, rstd = bo.run_layer_norm(hip, np.zeros((rows, 0), NP[dt]), None, None, 1e-5, dt)
    with bo.Bufs(hip) as b:
        m, r = b.put(np.ones(rows, np.float32)), b.put(np.ones(rows, np.float32))
        x = b.put(np.zeros((rows, 0), NP[dt]))
        assert hip.thvm_hip_layer_norm(b.out((rows, 0), NP[dt]), m, r, x, 0, 0, rows, 0, 1e-5, dt) == 0
        assert np.isnan(b.get(m)).all() and np.isnan(b.get(r)).all()


# ---- NaN and infinities through an activation ----

# a layer's kernels: few rows, 32-bit tiles as they lie, packed, 16-bit as they lie
KERNELS = [((1, 40, 60), F32, "thvm_few1n_f32"), ((20, 40, 60), F32, "thvm_few16n_f32"), ((500, 60, 2000), F32, "thvm_direct_f32"),
           ((2100, 70, 1900), F32, "thvm_gemm_64x64_f32"), ((1, 40, 60), F16, "thvm_few1n_f16"), ((200, 1192, 264), F16, "thvm_gemm_rc_64x64_f16"),
           ((2100, 70, 1900), F16, "thvm_gemm_64x64_f16")]


def _layer(shape, dt):
    m, k, n = shape
    rng = np.random.default_rng(m + n)
    return rng, rng.standard_normal((m, k)).astype(NP[dt]), (rng.standard_normal((k, n)) / math.sqrt(k)).astype(NP[dt])


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("shape,dt,kernel", KERNELS, ids=str)
def test_nan_stays(hip, shape, dt, kernel, name):
    """A row that diverged does not come out healthy, and spoils no other."""
    got = bp.linear(*shape, dt)[-1]
    assert got == kernel
    _, x, w = _layer(shape, dt)
    m = shape[0]
    clean, _ = bo.run_linear(hip, x, w, None, None, name, dt)
    x[m // 2, 7] = np.nan
    y, z = bo.run_linear(hip, x, w, None, None, name, dt)
    assert np.isnan(z[m // 2]).all() and np.isnan(y[m // 2]).all()
    keep = np.arange(m) != m // 2
    assert np.array_equal(y[keep], clean[keep])


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_nan_stays_in_gradients(hip, dt, name):
    """From dy and from the kept values: in its row of dx, its column of dw
    and of db."""
    m, k, n = 70, 50, 90
    rng, x, w = _layer((m, k, n), dt)
    dy, z = rng.standard_normal((2, m, n)).astype(NP[dt])
    clean = bo.run_linear_grad(hip, dy, z, x, w, name, dt)
    for where in ("dy", "z") if name != "none" else ("dy",):
        a = {"dy": dy.copy(), "z": z.copy()}
        a[where][9, 11] = np.nan
        dx, dw, db = bo.run_linear_grad(hip, a["dy"], a["z"], x, w, name, dt)
        assert np.isnan(dx[9]).all() and np.isnan(dw[:, 11]).all() and np.isnan(db[11])
        assert np.array_equal(np.delete(dx, 9, 0), np.delete(clean[0], 9, 0))
        assert np.array_equal(np.delete(dw, 11, 1), np.delete(clean[1], 11, 1)) and np.array_equal(np.delete(db, 11), np.delete(clean[2], 11))


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_infinities_through_an_activation(hip, dt, name):
    """Up, every activation is its argument; down, relu's is 0 and the others'
    formulas are a product of 0 and infinity."""
    bias = np.array([np.inf, -np.inf, 1.0, -1.0], NP[dt])
    y, z = bo.run_linear(hip, np.zeros((3, 0), NP[dt]), np.zeros((0, 4), NP[dt]), bias, None, name, dt)
    assert np.array_equal(z, np.broadcast_to(bias, z.shape))
    assert np.all(y[:, 0] == np.inf) and np.isfinite(y[:, 2:]).all()
    low = {"none": -np.inf, "relu": 0.0}.get(name, np.nan)
    assert np.array_equal(y[:, 1], np.full(3, low, NP[dt]), equal_nan=True)


# ---- activations on their own: no sum, z is the bias ----

def _grid():
    z = np.r_[np.linspace(-13, 13, 4001), np.linspace(-0.5, 0.5, 2001), np.ldexp(1.0, np.arange(-120, 3)), -np.ldexp(1.0, np.arange(-120, 3))]
    return z.astype(np.float32)


def _exact(name, z):
    """The activation in 64 bits, its small tail computed as a small number."""
    z = z.astype(np.float64)
    if name == "relu":
        return np.maximum(z, 0.0)
    if name == "gelu":
        return 0.5 * z * np.vectorize(math.erfc)(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def _units(name, z):
    """How many 2^-24 of itself an activation may be off (thvm_hip.h): 8, and
    what the rounding of an exponential's argument makes of it."""
    z = np.abs(z.astype(np.float64))
    return 8 + {"gelu": 2 * z * z, "gelu_tanh": 10 * (z + 0.045 * z ** 3), "silu": 2 * z}.get(name, 0.0)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_activation(hip, name, dt):
    z = _grid().astype(NP[dt])
    y, _ = bo.run_linear(hip, np.zeros((1, 0), NP[dt]), np.zeros((0, len(z)), NP[dt]), z, None, name, dt)
    want = _exact(name, z)
    within(y[0], want, _units(name, z) * U32 * np.abs(want) + bo.rounding(dt, want) + 2.0 ** -120)


@pytest.mark.parametrize("name", ACTS[1:])
def test_slope(hip, name):
    """act' alone: the products of dy = 1 and its one partner 1 pass it on. Of
    values around 0 and of far ones, within 16 (1 + |z|) units of 2^-24 of 1."""
    z = _grid()
    z = z[z != 0]
    m = len(z)
    dx, _, _ = bo.run_linear_grad(hip, np.ones((m, 1), np.float32), z[:, None], None, np.ones((1, 1), np.float32), name, F32, (True, False, False))
    want = bo.slope(name, z)
    within(dx[:, 0], want, 16 * U32 * (1 + np.abs(z.astype(np.float64))) * np.maximum(np.abs(want), 2.0 ** -3) + 2.0 ** -120)
