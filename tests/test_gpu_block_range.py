"""32-bit products over the whole range of 32 bits, on every kernel that
computes them: values far below their row's or column's largest where that one
is multiplied by 0, and infinities that meet values as small.

A sum of K products is within (2 K + 8) 2^-24 of the sum of the products'
magnitudes (thvm_hip.h); an output is rounded once more."""
import numpy as np
import pytest

from tests import blockops as bo
from tests import blockplan as bp
from tests.blockops import F16, F32, U32
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
    asked for. wide: row 2 of a and rows 3, 5, 7 of b hold one large value
    beside tiny ones, and meet rows in which the large one's partner is 0.
    broken: an infinity, which meets tiny values and zeros, and a NaN in a,
    another infinity in b."""
    (m, k), n = a.shape, b.shape[0]
    if "wide" in kind:
        a[2] = np.ldexp(a[2], -45)
        a[2, 0] = 2.0 ** 20
        b[::2, 0] = 0
        for r in (3, 5, 7):
            if r < n and k > 1:
                b[r] = np.ldexp(b[r], -30)
                b[r, 1] = 2.0 ** 60
        a[m // 2:, 1] = 0
        a[4 % m] = 0                       # a row of zeros stays one
    if "broken" in kind:
        a[m - 1, k - 1], a[m // 2, k // 2] = np.inf, np.nan
        b[n // 2, k - 1], b[n - 1, k - 1] = 1e-13, 0.0
        b[1, k // 3] = -np.inf
        a[0, k // 3] = -1e-20


def _reference(a, b, rows, cols):
    a64, b64 = a[rows].astype(np.float64), b[cols].astype(np.float64)
    with np.errstate(invalid="ignore"):
        return a64 @ b64.T, np.abs(a64) @ np.abs(b64).T


KINDS = ["wide", "broken", "wide, broken"]
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


@pytest.mark.parametrize("name", ["gelu", "silu"])
@pytest.mark.parametrize("shape", [(50, 60, 70), (300, 130, 260)], ids=str)
def test_gradient_through_an_activation(hip, shape, name):
    """What is computed again is dy act'(z), not dy."""
    m, k, n = shape
    rng = np.random.default_rng(m + k + n)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    dy, z = rng.standard_normal((2, m, n)).astype(np.float32)
    dy[2] = np.ldexp(dy[2], -45)
    dy[2, 0] = 2.0 ** 20
    w[::2, 0] = 0
    dy[:, 5] = np.ldexp(dy[:, 5], -45)
    dy[3, 5] = 2.0 ** 20
    x[3, ::2] = 0
    x[m - 1, 1] = np.inf
    s = bo.slope(name, z)
    dz = dy.astype(np.float64) * s
    edz = np.abs(dy.astype(np.float64)) * (16 * U32 * (1 + np.abs(z.astype(np.float64))))     # act' in 32 bits
    dx, dw, _ = bo.run_linear_grad(hip, dy, z, x, w, name, F32)
    w64, x64 = w.astype(np.float64), x.astype(np.float64)
    want = dz @ w64.T
    within(dx, want, _sum_bound(n, np.abs(dz) @ np.abs(w64.T), want) + 2 * edz @ np.abs(w64.T))
    with np.errstate(invalid="ignore"):
        want = x64.T @ dz
        within(dw, want, _sum_bound(m, np.abs(x64.T) @ np.abs(dz), want) + 2 * np.abs(x64.T) @ edz)


@pytest.mark.parametrize("k", [1, 70, 1000])
def test_equal_operands(hip, k):
    """1 + 2^-11 everywhere: what two 16-bit planes leave out has one sign."""
    m, n = 2100, 1900
    v = np.float32(1 + 2.0 ** -11)
    x, w = np.full((m, k), v), np.full((k, n), v)
    want = np.float64(v) ** 2 * k
    y, _ = bo.run_linear(hip, x, w, None, None, "none", F32)
    within(y, np.full((m, n), want), _sum_bound(k, want, want))
    dx, _, _ = bo.run_linear_grad(hip, np.full((m, n), v), None, None, w, "none", F32, (True, False, False))
    want = np.float64(v) ** 2 * n
    within(dx, np.full((m, k), want), _sum_bound(n, want, want))


@pytest.mark.parametrize("shape,kernel", [((2100, 300, 1900), "thvm_gemm_64x64_f32"), ((8000, 150, 7999), "thvm_gemm_256x256_f32")], ids=str)
def test_operands_that_never_meet(hip, shape, kernel):
    """Faint values whose partners are all 0 leave a sum exactly 0."""
    m, k, n = shape
    assert bp.linear(m, k, n, F32)[-1] == kernel
    rng = np.random.default_rng(k)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    x[:, 3] = np.ldexp(x[:, 3], -50)
    w[4] = np.ldexp(w[4], -20)
    x[1::2, :k // 2] = 0
    x[::2, k // 2:] = 0
    w[:k // 2, 1::2] = 0
    w[k // 2:, ::2] = 0
    y, _ = bo.run_linear(hip, x, w, None, None, "none", F32)
    assert not y[::2, 1::2].any() and not y[1::2, ::2].any()
    rows, cols = _some(m), _some(n)
    want, mag = _reference(x, w.T, rows, cols)
    within(y[rows][:, cols], want, _sum_bound(k, mag, want))


@pytest.mark.parametrize("shape,kernel", [((2100, 300, 1900), "thvm_gemm_64x64_f32"), ((2000, 1801, 1900), "thvm_gemm_128x128_f32")], ids=str)
@pytest.mark.parametrize("far", [10, 25, 60])
def test_one_large_feature(hip, shape, kernel, far):
    """One input and one output far above the others, which then are faint
    in every row and column; every second output does not see the large one."""
    m, k, n = shape
    assert bp.linear(m, k, n, F32)[-1] == kernel
    rng = np.random.default_rng(far)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    x[:, 5] = np.ldexp(x[:, 5], far)
    w[:, 6] = np.ldexp(w[:, 6], far)
    w[5, ::2] = 0
    y, _ = bo.run_linear(hip, x, w, None, None, "none", F32)
    rows, cols = _some(m), _some(n, 80)
    want, mag = _reference(x, w.T, rows, cols)
    within(y[rows][:, cols], want, _sum_bound(k, mag, want))


# ---- 16-bit gradients whose dy act'(z) is out of 16 bits ----

@pytest.mark.parametrize("shape", [(70, 90, 110), (1500, 1601, 1499)], ids=str)
def test_16_bit_gradient_past_the_range(hip, shape):
    """dy under 65504 and a slope of 1.13: the gradients are those of the
    product, which 32 bits hold, and not infinities."""
    m, k, n = shape
    rng = np.random.default_rng(m)
    x, w = (rng.standard_normal((m, k)) / 256).astype(np.float16), (rng.standard_normal((k, n)) / 256).astype(np.float16)
    dy, z = rng.standard_normal((2, m, n)).astype(np.float16)
    dy[3, 5], z[3, 5] = 60000, 1.4
    dy[m - 1, n - 1], z[m - 1, n - 1] = -65504, 1.5
    w[::2, 5] = 0
    x[3, 1::2] = 0
    s = bo.slope("gelu", z)
    dz = dy.astype(np.float64) * s
    assert np.abs(dz).max() > 65520
    dx, dw, db = bo.run_linear_grad(hip, dy, z, x, w, "gelu", F16)
    # act' in 32 bits; dz is rounded to 16 bits
    edz = np.abs(dy.astype(np.float64)) * (16 * U32 * (1 + np.abs(z.astype(np.float64)))) + np.abs(dz) * 2.0 ** -11 + 2.0 ** -25
    rows, cols = np.union1d(_some(m), [3]), _some(k)
    w64, x64 = w.astype(np.float64), x.astype(np.float64)
    want = dz[rows] @ w64[cols].T
    mag = np.abs(dz[rows]) @ np.abs(w64[cols]).T
    within(dx[rows][:, cols], want, (n + 4) * U32 * mag + edz[rows] @ np.abs(w64[cols]).T + bo.rounding(F16, want))
    rows, cols = _some(k), np.union1d(_some(n), [5])
    want = x64[:, rows].T @ dz[:, cols]
    mag = np.abs(x64[:, rows]).T @ np.abs(dz[:, cols])
    within(dw[rows][:, cols], want, (m + 4) * U32 * mag + np.abs(x64[:, rows]).T @ edz[:, cols] + bo.rounding(F16, want))
    # the column that holds the value is within 16 bits again once rounded, or an infinity
    want = dz.sum(0)
    fits = np.abs(want) < 65500
    bound = (edz - np.abs(dz) * 2.0 ** -11).sum(0) + (m + 4) * U32 * np.abs(dz).sum(0) + bo.rounding(F16, want)
    within(db[fits], want[fits], bound[fits])
    assert np.isinf(db[~fits]).sum() == (np.abs(want[~fits]) > 65520).sum()
