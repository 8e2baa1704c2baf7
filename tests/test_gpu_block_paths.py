"""Ways that the residual block's operators take by size, type and alignment
(test_gpu_block.py has the bounds): 16-bit matrices multiplied as they lie,
32-bit ones in tiles as they lie, few rows in narrow and wide strips with K
whole or split, large tiles of the orthogonalised step, tensors past 32-bit
offsets, and the limits."""
import numpy as np
import pytest

from tests import blockops as bo
from tests.blockops import F16, F32, NP, U32
from tests.test_gpu_block import _grad_check, _linear_check, _linear_inputs, _ln_check, _ln_inputs, _muon_inputs, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


# rows of 8, ends within a step of k and within a tile, tiles of 64, 128 and 256, K splits
LIES = [(65, 8, 8), (70, 72, 136), (64, 4000, 8), (300, 40, 264), (2, 1032, 520), (17, 2008, 72), (100, 4096, 200), (1000, 1032, 520),
        (2056, 200, 1928), (4000, 40, 4008), (3500, 2040, 3472)]
# rows that are not whole 16 bytes beside them: packed
PACKED = [(70, 72, 137), (70, 73, 136), (2000, 1801, 1900)]


@pytest.mark.parametrize("m,k,n", LIES + PACKED, ids=str)
def test_16_bit_layer(hip, m, k, n):
    _, x, w, bias, res = _linear_inputs(m, k, n, F16, m + k + n)
    name = "relu" if m * n > 1 << 20 else "gelu"
    _linear_check(hip, x, w, bias, res, name, F16)


def test_16_bit_layer_infinities_and_nan(hip):
    """As they lie, too, they reach their own rows and columns only."""
    _, x, w, _, _ = _linear_inputs(150, 88, 80, F16, 7)
    x[0, 3], x[1, 5], x[1, 60], x[2, 7], x[149, 87] = np.inf, np.inf, -np.inf, np.nan, np.inf
    w[11, 2], w[12, 4], w[87, 79] = -np.inf, np.nan, np.inf
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
    got, _ = bo.run_linear(hip, x, w, None, None, "none", F16)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf])
    fin = np.isfinite(want)
    # 88 products of values under 5 and 1 in 32 bits, and one rounding to 16
    assert np.all(np.abs(got[fin] - want[fin]) <= 92 * U32 * 88 * 5 + 2.0 ** -11 * np.abs(want[fin]) + 2.0 ** -25)


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows,cols", [(600, 4096), (515, 4099), (4100, 1000), (4099, 1999), (1500, 1000), (1025, 500), (511, 4096)], ids=str)
def test_layer_norm_rows(hip, rows, cols, dt):
    """Rows enough for a wave, or a small workgroup, to take longer ones."""
    _, x, gamma, beta = _ln_inputs(rows, cols, dt, rows + cols)
    _ln_check(hip, x, gamma, beta, 1e-5, dt)


# few rows in narrow strips and wide ones, K whole, split and with an end of its own; two rows to hundreds
FEW = [(1, 1, 5), (1, 127, 3), (1, 1025, 63), (1, 5000, 130), (1, 1024, 5001), (2, 128, 16), (2, 129, 17), (5, 1023, 2), (16, 300, 2100),
       (17, 2100, 301), (31, 1024, 1030), (40, 700, 2), (64, 513, 333), (250, 256, 250), (600, 100, 64), (3, 9000, 1), (20, 3000, 1)]
# tiles of 64 as they lie: ends of rows, columns and K, and splits
TILES = [(100, 4100, 515), (130, 2047, 2050), (250, 1000, 4099), (300, 130, 2049), (65, 4096, 4097), (500, 60, 2000)]


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("m,k,n", FEW + TILES, ids=str)
def test_rows(hip, m, k, n, dt):
    _, x, w, bias, res = _linear_inputs(m, k, n, dt, m * 3 + k + n)
    _linear_check(hip, x, w, bias, res, "gelu_tanh" if m * n < 1 << 18 else "relu", dt)


@pytest.mark.parametrize("m,k,n", [(2, 200, 40), (100, 4100, 515), (130, 2047, 2050)], ids=str)
def test_rows_infinities_and_nan(hip, m, k, n):
    """Past the ends nothing is multiplied that a value could spoil."""
    _, x, w, _, _ = _linear_inputs(m, k, n, F32, 5)
    x[0, k - 1], x[1, 0] = np.inf, np.nan
    w[k - 1, n - 1], w[0, 1] = -np.inf, np.nan
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
    got, _ = bo.run_linear(hip, x, w, None, None, "none", F32)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf])


@pytest.mark.parametrize("want", [(False, False, True), (True, False, True), (False, True, True)], ids=str)
@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
def test_bias_gradient(hip, want, dt):
    rng, x, w, _, res = _linear_inputs(3000, 40, 130, dt, 8)
    _grad_check(hip, (0.1 * rng.standard_normal((3000, 130))).astype(NP[dt]), res, x, w, "silu", dt, want)


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("count,n,w", [(12, 1104, 1104), (16, 1232, 1232), (2, 1500, 700)], ids=str)
def test_muon_tiles(hip, count, n, w, dt):
    """Tiles of 128, 192 and 256; the first matrix and the last, as test_muon has it."""
    p, g, m = _muon_inputs(count, n, w, dt, n + w)
    hyper = (0.05, 1.5, 0.1, 0.9, 1, 5)
    gp, gm = bo.run_muon(hip, p, g, m, *hyper, dt)
    for i in (0, count - 1):
        wp, wm = bo.muon(p[i], g[i], m[i], *hyper)
        pp, _ = bo.muon(p[i], g[i], m[i], *hyper, rounded=None if dt == F32 else np.float16, wide=np.float32 if dt == F32 else np.float64)
        within(gm[i], wm, 2 * U32 * (np.abs(wm) + np.abs(m[i]).astype(np.float64)))
        off, plain = np.linalg.norm(gp[i].astype(np.float64) - wp), np.linalg.norm(pp.astype(np.float64) - wp)
        size = np.linalg.norm(wp - p[i].astype(np.float64))
        assert off <= 4 * plain + 16 * U32 * size + np.linalg.norm(bo.rounding(dt, wp)), (off, plain, size)


# ---- tensors past 32-bit offsets ----

def test_linear_past_32_bits(hip):
    """W and y longer than 4 GiB: one row, and rows enough for a product's tiles."""
    L, k, period = hip, 64, 4093
    n = (1 << 25) + 8
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((k, period)) / 8).astype(np.float16)
    x = rng.standard_normal((65, k)).astype(np.float16)
    want = x.astype(np.float64) @ w.astype(np.float64)
    mag = np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64))
    cols = np.r_[0:300, (1 << 24) - 70:(1 << 24) + 70, n - 300:n]
    with bo.Bufs(L) as b:
        wide = np.empty((k, n), np.float16)
        for c in range(0, n, period):
            wide[:, c:c + period] = w[:, :min(period, n - c)]
        wi = b.put(wide)
        del wide
        for m in (1, 65):
            y = b.out((m, n), np.float16)
            assert L.thvm_hip_linear(y, 0, b.put(x[:m]), wi, 0, 0, 0, m, k, n, F16) == 0
            got = b.get(y)[:, cols]
            ref = want[:m][:, cols % period]
            within(got, ref, (k + 4) * U32 * mag[:m][:, cols % period] + bo.rounding(F16, ref))
            del got


@pytest.mark.parametrize("k", [0, 1024])
def test_more_rows_than_a_launch_counts(hip, k):
    """Few columns, in blocks of 16 rows, of which a launch has 65535."""
    L, m, n, period = hip, 65535 * 16 + 37, 2, 101
    rng = np.random.default_rng(6)
    x, w = rng.standard_normal((period, k)).astype(np.float16), (rng.standard_normal((k, n)) / 32).astype(np.float16)
    res = rng.standard_normal((period, n)).astype(np.float16)
    bias = rng.standard_normal(n).astype(np.float16)
    at = np.arange(m) % period
    z64 = x.astype(np.float64) @ w.astype(np.float64) + bias.astype(np.float64)
    mag = np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64)) + np.abs(bias.astype(np.float64))
    with bo.Bufs(L) as b:
        y, z = b.out((m, n), np.float16), b.out((m, n), np.float16)
        assert L.thvm_hip_linear(y, z, b.put(x[at]), b.put(w), b.put(bias), b.put(res[at]), 1, m, k, n, F16) == 0
        bound = (k + 4) * U32 * mag
        within(b.get(z), z64[at], (bound + bo.rounding(F16, z64))[at])
        want = np.maximum(z64, 0) + res.astype(np.float64)
        within(b.get(y), want[at], (bound + U32 * np.abs(want) + bo.rounding(F16, want))[at])


def test_layer_norm_past_32_bits(hip):
    L, cols, period = hip, 65544, 97
    rows = 33000
    rng = np.random.default_rng(4)
    x = rng.standard_normal((period, cols)).astype(np.float16)
    some = np.r_[0:3, 16000:16003, rows - 3:rows]
    with bo.Bufs(L) as b:
        long = np.empty((rows, cols), np.float16)
        for r in range(0, rows, period):
            long[r:r + period] = x[:min(period, rows - r)]
        xi = b.put(long)
        del long
        mean, rstd = b.out((rows,), np.float32), b.out((rows,), np.float32)
        y = b.out((rows, cols), np.float16)
        assert L.thvm_hip_layer_norm(y, mean, rstd, xi, 0, 0, rows, cols, 1e-5, F16) == 0
        wy, wm, wr = bo.layer_norm(x[some % period], None, None, 1e-5)
        got = b.get(y)[some]
        # sums of 65544 values of size 1: 80 additions follow each other, of 2^-24 each
        within(got, wy, 200 * U32 * (1 + np.abs(wy)) + bo.rounding(F16, wy))
        del got
        # dy = x: in place of y
        assert L.thvm_hip_layer_norm_grad(y, 0, 0, xi, xi, mean, rstd, 0, 0, rows, cols, F16) == 0
        wdx, _, _ = bo.layer_norm_grad(x[some % period], x[some % period], wm, wr, None, None)
        # what is left of dy is near 0: the difference of values of size 5
        within(b.get(y)[some], wdx, 1000 * U32 * 5 + bo.rounding(F16, wdx))


def test_limits(hip, capfd):
    """Sizes that no launch could hold are refused before any buffer is asked about."""
    L = hip
    with bo.Bufs(L) as b:
        y, x, w, v = (b.out((8, 8), np.float32) for _ in range(4))
        big = 1 << 24
        assert L.thvm_hip_linear(y, 0, x, w, 0, 0, 0, 1, big + 1, 1, F32) == -1
        assert L.thvm_hip_linear(y, 0, x, w, 0, 0, 0, (1 << 28) + 1, 0, 0, F32) == -1
        assert L.thvm_hip_linear_grad(y, 0, 0, x, 0, 0, w, 0, 1, 1, big + 1, F32) == -1
        assert L.thvm_hip_linear_grad(0, y, 0, x, 0, w, 0, 0, big + 1, 1, 1, F32) == -1
        assert L.thvm_hip_layer_norm(y, 0, 0, x, 0, 0, 1, big + 1, 1e-5, F32) == -1
        assert L.thvm_hip_layer_norm_grad(y, 0, 0, x, w, v, v, 0, 0, 1, big + 1, F32) == -1
        assert L.thvm_hip_muon_step(bo.ids([y]), bo.ids([x]), bo.ids([w]), 1, 1, big + 1, 0.1, 1, 0, 0.9, 1, 5, F32) == -1
    assert "2^24" in capfd.readouterr().err
