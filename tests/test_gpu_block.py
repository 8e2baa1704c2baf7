"""The residual block's operators on the GPU against their definitions in 64
bits, with bounds from the arithmetic:

Sums of K values or products in 32 bits, in any order, are within K * 2^-24
of the sum of the magnitudes. 32-bit products are three of the four products
of two f16 planes: each operand is within 2^-24 of itself or, far below its
row's largest value, 2^-39 of that, and the product left out is within 2^-24.
An output is rounded once to its type."""
import numpy as np
import pytest

from tests import blockops as bo
from tests.blockops import ACTS, F16, F32, NP, U32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


def within(got, want, bound):
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    err = np.abs(got[ok] - want[ok]) / np.broadcast_to(bound, want.shape)[ok]
    assert err.size == 0 or np.max(err) <= 1.0, np.max(err)


# ---- layer norm ----

# a row a wave, a workgroup of 256, of 1024 or longer than registers hold; odd lengths; one of each
LN = [(1, 1), (3, 5), (5, 63), (7, 64), (1030, 257), (4, 1000), (2, 1001), (9, 2048), (300, 4096), (3, 4099), (2, 8192),
      (2, 12289), (5, 16384), (2, 40001), (1, 66000)]


def _ln_inputs(rows, cols, dt, seed, offset=3.0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal(cols)) + offset * rng.standard_normal((rows, 1))).astype(NP[dt])
    gamma, beta = (1 + 0.2 * rng.standard_normal(cols)).astype(NP[dt]), rng.standard_normal(cols).astype(NP[dt])
    return rng, x, gamma, beta


def _ln_check(L, x, gamma, beta, eps, dt):
    y, mean, rstd = bo.run_layer_norm(L, x, gamma, beta, eps, dt)
    wy, wm, wr = bo.layer_norm(x, gamma, beta, eps)
    c = x.shape[1]
    d = min(c, 64 + c // 4096) + 8     # additions that follow each other in a sum
    size = np.abs(x.astype(np.float64)).mean(1)
    within(mean, wm, d * U32 * size + 1e-45)
    # the mean's error moves each centred value; the variance sums squares of those
    shift = d * U32 * size + U32 * np.abs(x.astype(np.float64)).max(1)
    rel = 2 * d * U32 + 2 * shift * wr
    within(rstd, wr, (rel + 4 * U32) * wr)
    g = 1.0 if gamma is None else np.abs(gamma.astype(np.float64))
    b = 0.0 if beta is None else np.abs(beta.astype(np.float64))
    plain = np.abs(wy - (0.0 if beta is None else beta.astype(np.float64)))
    within(y, wy, (shift * wr)[:, None] * g + (rel + 8 * U32)[:, None] * plain + 2 * U32 * b + bo.rounding(dt, wy))


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows,cols", LN, ids=str)
def test_layer_norm(hip, rows, cols, dt):
    _, x, gamma, beta = _ln_inputs(rows, cols, dt, rows * 31 + cols)
    _ln_check(hip, x, gamma, beta, 1e-5, dt)


@pytest.mark.parametrize("which", ["gamma", "beta", "none"])
def test_layer_norm_without_weights(hip, which):
    _, x, gamma, beta = _ln_inputs(6, 300, F32, 4)
    _ln_check(hip, x, gamma if which == "gamma" else None, beta if which == "beta" else None, 1e-5, F32)


def test_layer_norm_of_a_large_mean(hip):
    _, x, gamma, beta = _ln_inputs(40, 1024, F32, 5, offset=1000.0)
    _ln_check(hip, x, gamma, beta, 1e-5, F32)


def test_layer_norm_rows_stay_apart(hip):
    """A constant row, an infinity and a NaN: their own rows alone."""
    _, x, gamma, beta = _ln_inputs(8, 500, F32, 6)
    x[1] = 2.5
    clean = bo.run_layer_norm(hip, x, gamma, beta, 1e-5, F32)[0]
    assert np.allclose(clean[1], beta, atol=1e-6)
    x[3, 7], x[5, 499] = np.inf, np.nan
    y, _, _ = bo.run_layer_norm(hip, x, gamma, beta, 1e-5, F32)
    assert np.isnan(y[3]).all() and np.isnan(y[5]).all()
    keep = [0, 1, 2, 4, 6, 7]
    assert np.array_equal(y[keep], clean[keep])


def test_layer_norm_in_place(hip):
    _, x, gamma, beta = _ln_inputs(5, 777, F16, 7)
    want = bo.run_layer_norm(hip, x, gamma, beta, 1e-5, F16)[0]
    with bo.Bufs(hip) as b:
        i = b.put(x)
        assert hip.thvm_hip_layer_norm(i, 0, 0, i, b.put(gamma), b.put(beta), 5, 777, 1e-5, F16) == 0
        assert np.array_equal(b.get(i), want)


def _lng_check(L, dy, x, mean, rstd, gamma, add, dt, want=(True, True, True)):
    got = bo.run_layer_norm_grad(L, dy, x, mean, rstd, gamma, add, dt, want)
    dx, dg, db = bo.layer_norm_grad(dy, x, mean, rstd, gamma, add)
    rows, c = x.shape
    y64, r64 = np.abs(dy.astype(np.float64)), rstd.astype(np.float64)
    xh = np.abs((x.astype(np.float64) - mean.astype(np.float64)[:, None]) * r64[:, None])
    # the centred value is rounded once at the size of x or the mean
    dxh = U32 * (2 * xh + r64[:, None] * np.abs(x.astype(np.float64) - mean.astype(np.float64)[:, None]))
    g = y64 if gamma is None else y64 * np.abs(gamma.astype(np.float64))
    d = min(c, 64 + c // 4096) + 10
    s0, s1 = g.mean(1)[:, None], (g * xh).mean(1)[:, None]
    e1 = d * U32 * s1 + (g * dxh).mean(1)[:, None]
    b = r64[:, None] * (8 * U32 * (g + s0 + xh * s1) + d * U32 * s0 + xh * e1 + dxh * s1)
    if want[0]:
        within(got[0], dx, b + (0.0 if add is None else 2 * U32 * np.abs(add.astype(np.float64))) + bo.rounding(dt, dx) + 1e-40)
    if want[1]:
        within(got[1], dg, (rows + 4) * U32 * (y64 * xh).sum(0) + (y64 * dxh).sum(0) + bo.rounding(dt, dg) + 1e-40)
    if want[2]:
        within(got[2], db, (rows + 4) * U32 * y64.sum(0) + bo.rounding(dt, db) + 1e-40)
    return got


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows,cols", LN + [(2500, 96), (1999, 1000)], ids=str)
def test_layer_norm_grad(hip, rows, cols, dt):
    rng, x, gamma, _ = _ln_inputs(rows, cols, dt, rows * 17 + cols, offset=1.0)
    _, mean, rstd = (v.astype(np.float32) for v in bo.layer_norm(x, None, None, 1e-5))
    dy, add = (0.1 * rng.standard_normal((2, rows, cols))).astype(NP[dt])
    _lng_check(hip, dy, x, mean, rstd, gamma, add, dt)


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)], ids=str)
@pytest.mark.parametrize("cols", [100, 20000])
def test_layer_norm_grad_some(hip, want, cols):
    rng, x, gamma, _ = _ln_inputs(11, cols, F32, 8)
    _, mean, rstd = (v.astype(np.float32) for v in bo.layer_norm(x, None, None, 1e-5))
    _lng_check(hip, rng.standard_normal((11, cols)).astype(np.float32), x, mean, rstd, None, None, F32, want)


def test_layer_norm_grad_against_differences(hip):
    """Along a direction d of x (gamma, beta), the loss sum(y * c) changes by
    the gradient's product with d: central differences of the forward pass,
    whose third-order rest and rounding over the step bound what is left."""
    rng, x, gamma, beta = _ln_inputs(6, 130, F32, 9, offset=0.5)
    c = rng.standard_normal((6, 130)).astype(np.float32)
    _, mean, rstd = bo.run_layer_norm(hip, x, gamma, beta, 1e-5, F32)
    grads = bo.run_layer_norm_grad(hip, c, x, mean, rstd, gamma, None, F32)
    h = 2.0 ** -7

    def loss(*a):
        return float((bo.run_layer_norm(hip, *(v.astype(np.float32) for v in a), 1e-5, F32)[0].astype(np.float64) * c).sum())

    for which, g in enumerate(grads):
        args = [x, gamma, beta]
        d = rng.choice([-1.0, 1.0], args[which].shape).astype(np.float32)
        hi, lo = list(args), list(args)
        hi[which], lo[which] = args[which] + np.float32(h) * d, args[which] - np.float32(h) * d
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        exact = float((g.astype(np.float64) * d).sum())
        scale = float(np.abs(c).sum()) * float(np.abs(gamma).max()) * float(rstd.max() if which == 0 else 4)
        assert abs(diff - exact) <= (h * h * max(1.0, float(rstd.max()) ** 2) + 64 * U32 / h) * scale


@pytest.mark.parametrize("which", ["dy", "x", "add"])
@pytest.mark.parametrize("cols", [300, 20000])
def test_layer_norm_grad_in_place(hip, which, cols):
    rng, x, gamma, _ = _ln_inputs(9, cols, F32, 10)
    _, mean, rstd = (v.astype(np.float32) for v in bo.layer_norm(x, None, None, 1e-5))
    dy, add = rng.standard_normal((2, 9, cols)).astype(np.float32)
    want = bo.run_layer_norm_grad(hip, dy, x, mean, rstd, gamma, add, F32)
    with bo.Bufs(hip) as b:
        i = {"dy": b.put(dy), "x": b.put(x), "add": b.put(add)}
        dg, db = b.out((cols,), np.float32), b.out((cols,), np.float32)
        assert hip.thvm_hip_layer_norm_grad(i[which], dg, db, i["dy"], i["x"], b.put(mean), b.put(rstd), b.put(gamma), i["add"],
                                            9, cols, F32) == 0
        for j, w in zip((i[which], dg, db), want):
            assert np.array_equal(b.get(j), w)


# ---- linear ----

# one row to four to sixteen, tiles of 64, 128 and 256 and their edges, K splits, odd sizes
LINEAR = [(1, 64, 64), (1, 1, 1), (1, 771, 1501), (3, 33, 65), (4, 4096, 96), (5, 130, 17), (16, 1000, 257), (17, 16, 16), (64, 784, 128),
          (65, 63, 64), (200, 100, 72), (129, 771, 130), (1031, 40, 515), (100, 3000, 90), (2100, 70, 1900), (3600, 36, 3400)]


def _mag(x, w):
    """The sums of magnitudes, and of what the planes' absolute part may add."""
    ax, aw = np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64))
    far = 2.0 ** -38 * (ax.max(1, initial=0.0)[:, None] * aw.sum(0)[None, :] + ax.sum(1)[:, None] * aw.max(0, initial=0.0)[None, :])
    return ax @ aw, far


def _linear_check(L, x, w, bias, res, name, dt, keep=True):
    y, z = bo.run_linear(L, x, w, bias, res, name, dt, keep)
    wz = x.astype(np.float64) @ w.astype(np.float64)
    mag, far = _mag(x, w)
    if bias is not None:
        wz = wz + bias.astype(np.float64)
        mag = mag + np.abs(bias.astype(np.float64))
    bz = (x.shape[1] + 4) * U32 * mag + far
    if keep:
        within(z, wz, bz + bo.rounding(dt, wz))
    a = bo.act(name, wz)
    want = a if res is None else a + res.astype(np.float64)
    # an activation's slope is at most 1.13; its own roundings are a few units of 1 + |z|
    act = 0.0 if name == "none" else 16 * U32 * np.abs(wz) + 2.0 ** -40
    within(y, want, 1.13 * bz + act + (0.0 if res is None else U32 * np.abs(want)) + bo.rounding(dt, want))
    return y, z


def _linear_inputs(m, k, n, dt, seed):
    rng = np.random.default_rng(seed)
    return (rng, rng.standard_normal((m, k)).astype(NP[dt]), (rng.standard_normal((k, n)) / np.sqrt(max(1, k))).astype(NP[dt]),
            rng.standard_normal(n).astype(NP[dt]), rng.standard_normal((m, n)).astype(NP[dt]))


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("m,k,n", LINEAR, ids=str)
def test_linear(hip, m, k, n, dt):
    _, x, w, bias, res = _linear_inputs(m, k, n, dt, m * 7 + k * 3 + n)
    _linear_check(hip, x, w, bias, res, ACTS[(m + n) % len(ACTS)], dt)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("m", [2, 40])
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_linear_activations(hip, name, m, dt):
    _, x, w, bias, res = _linear_inputs(m, 50, 60, dt, 3)
    _linear_check(hip, (x * 4).astype(NP[dt]), w, bias, None, name, dt)
    _linear_check(hip, x, w, None, res, name, dt, keep=False)


@pytest.mark.parametrize("m", [2, 40])
def test_linear_in_place(hip, m):
    _, x, w, bias, res = _linear_inputs(m, 70, 90, F32, 4)
    want, _ = bo.run_linear(hip, x, w, bias, res, "gelu", F32)
    with bo.Bufs(hip) as b:
        r = b.put(res)
        assert hip.thvm_hip_linear(r, 0, b.put(x), b.put(w), b.put(bias), r, 2, m, 70, 90, F32) == 0
        assert np.array_equal(b.get(r), want)


@pytest.mark.parametrize("shape", [(0, 5, 7), (5, 0, 7), (5, 6, 0), (40, 0, 9)], ids=str)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_linear_of_nothing(hip, shape, dt):
    _, x, w, bias, res = _linear_inputs(*shape, dt, 5)
    y, z = bo.run_linear(hip, x, w, bias, res, "silu", dt)
    if 0 not in (shape[0], shape[2]):
        assert np.array_equal(z, np.broadcast_to(bias, z.shape))
        within(y, bo.act("silu", z) + res, 1e-6 + bo.rounding(dt, bo.act("silu", z) + res))
    dy = res
    dx, dw, db = bo.run_linear_grad(hip, dy, z, x, w, "none", dt)
    assert not dx.any() and not dw.any() or 0 not in shape
    within(db, dy.astype(np.float64).sum(0), 1e-5 + bo.rounding(dt, dy.astype(np.float64).sum(0)))


@pytest.mark.parametrize("m", [3, 50])
def test_linear_of_many_sizes_of_value(hip, m):
    """Rows and columns from 2^-120 to 2^110, and rows that hold both."""
    rng, x, w, bias, res = _linear_inputs(m, 200, 130, F32, 6)
    x = np.ldexp(x, rng.integers(-120, 10, (m, 1))).astype(np.float32)
    x[1] = np.ldexp(x[1], rng.integers(-30, 30, 200))
    w = np.ldexp(w, rng.integers(-20, 100, (1, 130))).astype(np.float32)
    w[:, 5] = np.ldexp(w[:, 5], rng.integers(-25, 0, 200))
    x[2] = 0
    w[:, 9] = 0
    _linear_check(hip, x, w, None, None, "none", F32)


@pytest.mark.parametrize("m", [3, 70])
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_linear_infinities_and_nan(hip, m, dt):
    """What a sum of products makes of them, and nothing in other rows and columns."""
    _, x, w, _, _ = _linear_inputs(m, 90, 80, dt, 7)
    x[0, 3], x[1, 5], x[1, 60], x[2, 7] = np.inf, np.inf, -np.inf, np.nan
    w[11, 2], w[12, 4], w[13, 4], w[3, 6] = -np.inf, np.nan, 1.0, 0.0
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
    got, _ = bo.run_linear(hip, x, w, None, None, "none", dt)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    fin = np.isfinite(want)
    assert np.allclose(got[fin], want[fin], rtol=0, atol=94 * U32 * 90 * 4 if dt == F32 else 2e-2)


def _grad_check(L, dy, z, x, w, name, dt, want=(True, True, True)):
    got = bo.run_linear_grad(L, dy, z, x, w, name, dt, want)
    s = bo.slope(name, z)
    dz = dy.astype(np.float64) * s
    # act' in 32 bits; of f16, dz is rounded once more before the products
    edz = np.abs(dy.astype(np.float64)) * (16 * U32 * (1 + np.abs(z.astype(np.float64))))
    db_bound = edz.sum(0) + (dy.shape[0] + 4) * U32 * np.abs(dz).sum(0)
    if dt == F16:
        edz = edz + np.abs(dz) * 2.0 ** -11 + 2.0 ** -25
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    if want[0]:
        mag, far = _mag(dz, w64.T)
        wx = dz @ w64.T
        within(got[0], wx, (dy.shape[1] + 4) * U32 * mag + far + edz @ np.abs(w64.T) + bo.rounding(dt, wx) + 1e-40)
    if want[1]:
        mag, far = _mag(x64.T, dz)
        ww = x64.T @ dz
        within(got[1], ww, (dy.shape[0] + 4) * U32 * mag + far + np.abs(x64.T) @ edz + bo.rounding(dt, ww) + 1e-40)
    if want[2]:
        within(got[2], dz.sum(0), db_bound + bo.rounding(dt, dz.sum(0)) + 1e-40)


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("m,k,n", LINEAR, ids=str)
def test_linear_grad(hip, m, k, n, dt):
    rng, x, w, _, res = _linear_inputs(m, k, n, dt, m * 5 + k * 3 + n)
    _grad_check(hip, (0.1 * rng.standard_normal((m, n))).astype(NP[dt]), res, x, w, ACTS[(m + k) % len(ACTS)], dt)


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True), (True, True, False)], ids=str)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_linear_grad_some(hip, want, dt):
    rng, x, w, _, res = _linear_inputs(70, 90, 110, dt, 8)
    _grad_check(hip, (0.1 * rng.standard_normal((70, 110))).astype(NP[dt]), res, x, w, "gelu", dt, want)


@pytest.mark.parametrize("name", ACTS)
def test_linear_grad_against_differences(hip, name):
    """As for layer norm: the second derivatives of the activations are under
    1.2 and their third ones under 3, but for relu's, whose z stay off 0."""
    rng, x, w, bias, _ = _linear_inputs(20, 30, 40, F32, 9)
    if name == "relu":
        x, w, bias = (np.round(x * 8) / 8).astype(np.float32), (np.round(w * 64) / 64).astype(np.float32), bias * 0 + np.float32(2.0 ** -10)
    c = rng.standard_normal((20, 40)).astype(np.float32)
    _, z = bo.run_linear(hip, x, w, bias, None, name, F32)
    grads = bo.run_linear_grad(hip, c, z, x, w, name, F32)
    h = 2.0 ** -17 if name == "relu" else 2.0 ** -7

    def loss(*a):
        y, _ = bo.run_linear(hip, *(v.astype(np.float32) for v in a), None, name, F32)
        return float((y.astype(np.float64) * c).sum())

    for which, g in enumerate(grads):
        args = [x, w, bias]
        d = rng.choice([-1.0, 1.0], args[which].shape).astype(np.float32)
        hi, lo = list(args), list(args)
        hi[which], lo[which] = args[which] + np.float32(h) * d, args[which] - np.float32(h) * d
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        exact = float((g.astype(np.float64) * d).sum())
        # how far z moves, the third-order rest, and the outputs' roundings over the step
        move = np.abs(w).sum(0).max() if which == 0 else np.abs(x).sum(1).max() if which == 1 else 1.0
        rest = 0.0 if name in ("none", "relu") else 3 * h * h * move ** 3 / 6
        noise = 40 * U32 * float((np.abs(x) @ np.abs(w)).max()) / h / np.sqrt(c.size) * 4
        assert abs(diff - exact) <= (rest + noise) * float(np.abs(c).sum())


def test_linear_twice_the_same_bits(hip):
    """No order of sums depends on the run."""
    rng, x, w, bias, res = _linear_inputs(300, 2000, 200, F32, 10)
    a, b = (bo.run_linear(hip, x, w, bias, res, "gelu", F32)[0] for _ in range(2))
    assert np.array_equal(a, b)
    dy = rng.standard_normal((300, 200)).astype(np.float32)
    for p, q in zip(*(bo.run_linear_grad(hip, dy, res, x, w, "gelu", F32) for _ in range(2))):
        assert np.array_equal(p, q)


# ---- the orthogonalised step ----

MUON = [(1, 1, 1), (1, 1, 9), (2, 7, 5), (1, 64, 64), (3, 64, 200), (1, 784, 128), (2, 130, 61), (1, 33, 1000), (1, 500, 500), (1, 1100, 900)]


def _muon_inputs(count, rows, cols, dt, seed):
    rng = np.random.default_rng(seed)
    return ([(rng.standard_normal((rows, cols)) / 8).astype(NP[dt]) for _ in range(count)],
            [(rng.standard_normal((rows, cols)) * 1e-2).astype(NP[dt]) for _ in range(count)],
            [(rng.standard_normal((rows, cols)) * 1e-1).astype(np.float32) for _ in range(count)])


def _muon_check(L, p, g, m, hyper, dt):
    """The update's distance from the one in 64 bits is at most four times that
    of the same steps in plain 32-bit sums (16 bits: with X, A and B rounded as
    documented), or 16 roundings; the momentum is two roundings from its own."""
    gp, gm = bo.run_muon(L, p, g, m, *hyper, dt)
    for i in range(len(p)):
        wp, wm = bo.muon(p[i], g[i], m[i], *hyper)
        pp, _ = bo.muon(p[i], g[i], m[i], *hyper, rounded=None if dt == F32 else np.float16,
                        wide=np.float32 if dt == F32 else np.float64)
        within(gm[i], wm, 2 * U32 * (np.abs(wm) + np.abs(m[i]).astype(np.float64)))
        off, plain = np.linalg.norm(gp[i].astype(np.float64) - wp), np.linalg.norm(pp.astype(np.float64) - wp)
        size = np.linalg.norm(wp - p[i].astype(np.float64))
        assert off <= 4 * plain + 16 * U32 * size + np.linalg.norm(bo.rounding(dt, wp)), (off, plain, size)


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("count,rows,cols", MUON, ids=str)
def test_muon(hip, count, rows, cols, dt):
    p, g, m = _muon_inputs(count, rows, cols, dt, rows + cols)
    _muon_check(hip, p, g, m, (0.05, 1.5, 0.1, 0.9, rows % 2, 5), dt)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_muon_steps(hip, steps):
    p, g, m = _muon_inputs(1, 70, 40, F32, 3)
    _muon_check(hip, p, g, m, (0.05, 1.0, 0.0, 0.0, 1, steps), F32)


def test_muon_of_many_matrices(hip):
    """More than one launch names."""
    p, g, m = _muon_inputs(19, 20, 30, F32, 4)
    _muon_check(hip, p, g, m, (0.02, 1.0, 0.1, 0.95, 1, 5), F32)


@pytest.mark.parametrize("size", [0.0, 1e-30, 1e30, 3e38])
def test_muon_sizes_of_gradients(hip, size):
    """No gradient's size overflows the norm, and a zero one moves nothing."""
    p, g, m = _muon_inputs(1, 40, 70, F32, 5)
    g = [np.sign(v) * np.float32(size) if size else v * 0 for v in g]
    m = [v * 0 for v in m]
    hyper = (0.05, 1.0, 0.0, 0.0, 0, 5)
    if size < 1e-20:      # under the constant that keeps the norm off 0
        gp, _ = bo.run_muon(hip, p, g, m, *hyper, F32)
        assert np.isfinite(gp[0]).all() and np.abs(gp[0] - p[0]).max() <= 1e-6
    else:
        _muon_check(hip, p, g, m, hyper, F32)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_muon_of_a_broken_gradient(hip, bad):
    """It shows in the matrix it belongs to and in no other."""
    p, g, m = _muon_inputs(2, 40, 70, F32, 6)
    clean, _ = bo.run_muon(hip, p, g, m, 0.05, 1.0, 0.0, 0.9, 1, 5, F32)
    g[0][3, 4] = bad
    gp, _ = bo.run_muon(hip, p, g, m, 0.05, 1.0, 0.0, 0.9, 1, 5, F32)
    assert np.isnan(gp[0]).any() and np.array_equal(gp[1], clean[1])


# ---- the backend's manner ----

def test_refusals(hip, capfd):
    L = hip
    with bo.Bufs(L) as b:
        x, w, y, v = b.out((8, 8), np.float32), b.out((8, 8), np.float32), b.out((8, 8), np.float32), b.out((8,), np.float32)
        u = b.out((8,), np.float32)
        E = -1
        assert L.thvm_hip_layer_norm(y, 0, 0, x, 0, 0, 8, 9, 1e-5, F32) == E           # shorter than its tensor
        assert L.thvm_hip_layer_norm(y, 0, 0, x, 0, 0, 8, 8, 1e-5, 2) == E             # an integer type
        assert L.thvm_hip_layer_norm(y, 0, 0, 0, 0, 0, 8, 8, 1e-5, F32) == E           # no input
        assert L.thvm_hip_layer_norm(y, 0, 0, 9999, 0, 0, 8, 8, 1e-5, F32) == E        # unknown
        assert L.thvm_hip_layer_norm(y, v, v, x, 0, 0, 8, 8, 1e-5, F32) == E           # one buffer, two outputs
        assert L.thvm_hip_layer_norm(y, 0, 0, x, y, 0, 8, 8, 1e-5, F32) == E
        assert L.thvm_hip_layer_norm_grad(0, 0, 0, x, w, v, u, 0, 0, 8, 8, F32) == E   # no output
        assert L.thvm_hip_layer_norm_grad(y, 0, 0, x, w, 0, u, 0, 0, 8, 8, F32) == E   # no statistics
        assert L.thvm_hip_layer_norm_grad(y, v, 0, x, w, v, u, 0, 0, 8, 8, F32) == E
        assert L.thvm_hip_linear(y, 0, x, w, 0, 0, 5, 8, 8, 8, F32) == E               # unknown activation
        assert L.thvm_hip_linear(x, 0, x, w, 0, 0, 0, 8, 8, 8, F32) == E               # y is x
        assert L.thvm_hip_linear(y, y, x, w, 0, 0, 0, 8, 8, 8, F32) == E               # y is z
        assert L.thvm_hip_linear(y, 0, x, w, 0, 0, 0, 8, 16, 8, F32) == E
        assert L.thvm_hip_linear(y, 0, x, w, 0, 0, 0, 65536, 65536, 65536, F32) == E   # sizes that pass 32 bits
        assert L.thvm_hip_linear_grad(y, 0, 0, x, 0, w, w, 1, 8, 8, 8, F32) == E       # no z
        assert L.thvm_hip_linear_grad(y, 0, 0, x, 0, w, 0, 0, 8, 8, 8, F32) == E       # no w
        assert L.thvm_hip_linear_grad(0, 0, 0, x, 0, w, w, 0, 8, 8, 8, F32) == E
        one = bo.ids([x])
        assert L.thvm_hip_muon_step(one, bo.ids([w]), bo.ids([y]), 1, 8, 8, 0.1, 1, 0, 0.9, 1, 0, F32) == E   # no steps
        assert L.thvm_hip_muon_step(one, bo.ids([w]), one, 1, 8, 8, 0.1, 1, 0, 0.9, 1, 5, F32) == E
        assert L.thvm_hip_muon_step(bo.ids([x, x]), bo.ids([w, w]), bo.ids([y, y]), 2, 8, 8, 0.1, 1, 0, 0.9, 1, 5, F32) == E
        assert L.thvm_hip_muon_step(one, bo.ids([w]), bo.ids([v]), 1, 8, 8, 0.1, 1, 0, 0.9, 1, 5, F32) == E
        assert np.isnan(b.get(y)).all() and np.isnan(b.get(x)).all()                   # nothing ran
    assert "tinyhvm-hip: linear: " in capfd.readouterr().err


def test_step_in_a_graph(hip):
    """A block's step captured once and launched again and again, with eager
    work between, leaves what the same eager steps leave, bit for bit."""
    L, rng = hip, np.random.default_rng(11)
    m, k, n = 70, 48, 96
    arrays = {"x": rng.standard_normal((m, k)), "w1": rng.standard_normal((k, n)) / 7, "w2": rng.standard_normal((n, k)) / 10,
              "b1": rng.standard_normal(n), "b2": rng.standard_normal(k), "gamma": 1 + 0.1 * rng.standard_normal(k),
              "beta": rng.standard_normal(k), "dy": rng.standard_normal((m, k)), "m1": np.zeros((k, n)), "m2": np.zeros((n, k))}
    out = {"h": (m, k), "mean": (m,), "rstd": (m,), "z": (m, n), "a": (m, n), "y": (m, k), "da": (m, n), "dw2": (n, k), "db2": (k,),
           "dh": (m, k), "dw1": (k, n), "db1": (n,), "dx": (m, k), "dgamma": (k,), "dbeta": (k,)}

    def step(i):
        calls = [
            L.thvm_hip_layer_norm(i["h"], i["mean"], i["rstd"], i["x"], i["gamma"], i["beta"], m, k, 1e-5, F32),
            L.thvm_hip_linear(i["a"], i["z"], i["h"], i["w1"], i["b1"], 0, 3, m, k, n, F32),
            L.thvm_hip_linear(i["y"], 0, i["a"], i["w2"], i["b2"], i["x"], 0, m, n, k, F32),
            L.thvm_hip_linear_grad(i["da"], i["dw2"], i["db2"], i["dy"], 0, i["a"], i["w2"], 0, m, n, k, F32),
            L.thvm_hip_linear_grad(i["dh"], i["dw1"], i["db1"], i["da"], i["z"], i["h"], i["w1"], 3, m, k, n, F32),
            L.thvm_hip_layer_norm_grad(i["dx"], i["dgamma"], i["dbeta"], i["dh"], i["x"], i["mean"], i["rstd"], i["gamma"], i["dy"], m, k, F32),
            L.thvm_hip_muon_step(bo.ids([i["w1"]]), bo.ids([i["dw1"]]), bo.ids([i["m1"]]), 1, k, n, 0.02, 1.0, 0.01, 0.95, 1, 5, F32),
            L.thvm_hip_muon_step(bo.ids([i["w2"]]), bo.ids([i["dw2"]]), bo.ids([i["m2"]]), 1, n, k, 0.02, 1.4, 0.01, 0.95, 1, 5, F32)]
        assert not any(calls)

    with bo.Bufs(L) as b:
        eager, graph = ({**{s: b.put(v.astype(np.float32)) for s, v in arrays.items()}, **{s: b.out(v, np.float32) for s, v in out.items()}}
                        for _ in range(2))
        step(eager)
        for i in graph.values():
            assert L.thvm_hip_buf_device_ptr(i)
        assert L.thvm_hip_synchronize() == 0
        assert L.thvm_hip_graph_begin() == 0
        step(graph)
        g = L.thvm_hip_graph_end()
        assert g
        try:
            for rep in range(3):
                assert L.thvm_hip_graph_launch(g) == 0
                if rep:
                    step(eager)
                for s in eager:
                    assert np.array_equal(b.get(eager[s]), b.get(graph[s])), s
        finally:
            L.thvm_hip_graph_destroy(g)


def test_between_dispatches(hip):
    """Host writes, queued copies and reads around the calls keep their order."""
    L, rng = hip, np.random.default_rng(12)
    x, w = rng.standard_normal((20, 30)).astype(np.float32), rng.standard_normal((30, 40)).astype(np.float32)
    with bo.Bufs(L) as b:
        src, xi, wi, y = b.put(x), b.out((20, 30), np.float32), b.put(w), b.out((20, 40), np.float32)
        L.thvm_hip_buf_copy(xi, src, x.nbytes)
        assert L.thvm_hip_linear(y, 0, xi, wi, 0, 0, 0, 20, 30, 40, F32) == 0
        first = b.get(y)
        x2 = np.ascontiguousarray(x[::-1])
        L.thvm_hip_buf_write(xi, x2.ctypes.data, x2.nbytes)
        assert L.thvm_hip_linear(y, 0, xi, wi, 0, 0, 0, 20, 30, 40, F32) == 0
        assert np.array_equal(b.get(y), first[::-1])
