"""32-bit products over the whole range of 32 bits, on every kernel that
computes them: infinities that meet values far below their row's largest.

A sum of K products is within (2 K + 8) 2^-24 of the sum of the products'
magnitudes; an output is rounded once more."""
import numpy as np
import pytest

from tests import blockops as bo
from tests import blockplan as bp
from tests.blockops import F32, U32
from tests.test_gpu_block import within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


def _sum_bound(k, mag, want):
    return (2 * k + 8) * U32 * mag + bo.rounding(F32, want)


def _some(n, count=40):
    """The first, the last and some between."""
    return np.unique(np.r_[0:min(n, 12), np.linspace(0, n - 1, count).astype(int), max(0, n - 6):n])


def _spread(rng, a, b, kind):
    """a [M][K] and b [N][K] (float32, in place) whose product sum_k a b is
    asked for. broken: an infinity, which meets tiny values and zeros, and a NaN in a,
    another infinity in b."""
    (m, k), n = a.shape, b.shape[0]
    if "broken" in kind:
        a[m - 1, k - 1], a[m // 2, k // 2] = np.inf, np.nan
        b[n // 2, k - 1], b[n - 1, k - 1] = 1e-13, 0.0
        b[1, k // 3] = -np.inf
        a[0, k // 3] = -1e-20


def _reference(a, b, rows, cols):
    a64, b64 = a[rows].astype(np.float64), b[cols].astype(np.float64)
    with np.errstate(invalid="ignore"):
        return a64 @ b64.T, np.abs(a64) @ np.abs(b64).T


KINDS = ["broken"]
LAYERS = [((3, 300, 200), "thvm_few16n_f32"), ((17, 2100, 301), "thvm_few16_f32"), ((500, 60, 2000), "thvm_direct_f32"),
          ((130, 4096, 4095), "thvm_direct_f32"), ((700, 5000, 300), "thvm_direct_f32"), ((2100, 70, 1900), "thvm_gemm_64x64_f32"), ((1100, 2000, 1100), "thvm_gemm_64x64_f32"),
          ((1500, 1601, 1499), "thvm_gemm_128x128_f32"), ((8000, 150, 7999), "thvm_gemm_256x256_f32")]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,kernel", LAYERS, ids=str)
def test_layer(hip, shape, kernel, kind):
    assert bp.linear(*shape, F32)[-1] == kernel
    m, k, n = shape
    rng = np.random.default_rng(m + k + n)
    a, b = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    _spread(rng, a, b, kind)
    bias, res = rng.standard_normal((2, n)).astype(np.float32)
    res = np.broadcast_to(res, (m, n))
    y, z = bo.run_linear(hip, a, b.T, None, res, "none", F32)
    rows, cols = np.union1d(_some(m), [m // 2]), np.union1d(_some(n), [n // 2])
    want, mag = _reference(a, b, rows, cols)
    z, y = z[rows][:, cols], y[rows][:, cols]
    within(z, want, _sum_bound(k, mag, want))
    full = want + res[rows][:, cols].astype(np.float64)
    within(y, full, _sum_bound(k, mag, want) + U32 * np.abs(full) + bo.rounding(F32, full))


GRADS = [((50, 60, 70), "thvm_gemm_64x64_f32", "thvm_gemm_64x64_f32"), ((300, 130, 2049), "thvm_gemm_64x64_f32", "thvm_gemm_64x64_f32"),
         ((4100, 70, 90), "thvm_gemm_64x64_f32", "thvm_gemm_64x64_f32"), ((1500, 1601, 1499), "thvm_gemm_128x128_f32", "thvm_gemm_128x128_f32"),
         ((8000, 7999, 150), "thvm_gemm_256x256_f32", None),
         ((150, 8001, 7900), None, "thvm_gemm_256x256_f32")]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,dx_kernel,dw_kernel", GRADS, ids=str)
def test_gradient_of_x(hip, shape, dx_kernel, dw_kernel, kind):
    if dx_kernel is None:
        pytest.skip("its other gradient is the case")
    assert bp.linear_grad(*shape, F32)[2] == dx_kernel
    m, k, n = shape
    rng = np.random.default_rng(m + k + n)
    dy, w = rng.standard_normal((m, n)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    _spread(rng, dy, w, kind)
    dx, _, _ = bo.run_linear_grad(hip, dy, None, None, w, "none", F32, (True, False, False))
    rows, cols = np.union1d(_some(m), [m // 2]), np.union1d(_some(k), [k // 2])
    want, mag = _reference(dy, w, rows, cols)
    within(dx[rows][:, cols], want, _sum_bound(n, mag, want))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,dx_kernel,dw_kernel", GRADS, ids=str)
def test_gradient_of_weights(hip, shape, dx_kernel, dw_kernel, kind):
    if dw_kernel is None:
        pytest.skip("its other gradient is the case")
    assert bp.linear_grad(*shape, F32)[3] == dw_kernel
    m, k, n = shape
    rng = np.random.default_rng(m + k + n)
    x, dy = rng.standard_normal((k, m)).astype(np.float32), rng.standard_normal((n, m)).astype(np.float32)
    _spread(rng, x, dy, kind)
    _, dw, db = bo.run_linear_grad(hip, dy.T, None, x.T, np.broadcast_to(np.float32(0), (k, n)), "none", F32, (False, True, True))
    rows, cols = np.union1d(_some(k), [k // 2]), np.union1d(_some(n), [n // 2])
    want, mag = _reference(x, dy, rows, cols)
    within(dw[rows][:, cols], want, _sum_bound(m, mag, want))
    within(db, dy.astype(np.float64).sum(1), (m + 4) * U32 * np.abs(dy.astype(np.float64)).sum(1) + bo.rounding(F32, dy.astype(np.float64).sum(1)))
