"""Each kernel of the residual block's products at sizes that reach it, as
blockplan.py finds them on the host: a choice by size that changes fails here
and does not leave a kernel untested. Large results are compared on rows and
columns at the tiles' edges and between; bounds as in test_gpu_block.py."""
import math

import numpy as np
import pytest

from tests import blockops as bo
from tests import blockplan as bp
from tests.blockops import ACTS, F16, F32, NP, U32
from tests.test_gpu_block import _linear_check, _linear_inputs, _ln_check, _ln_inputs, _lng_check, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


def kernel(m, k, n, dt):
    """A layer's last kernel and its K splits."""
    last = bp.launches("thvm_hip_linear", 1, 2, 3, 4, 5, 6, 1, m, k, n, dt)[-1]
    return last.name.decode(), last.gy


def kernels(m, k, n, dt):
    """dx's and dw's, and whether K is split."""
    return [(v.name.decode(), v.gy > 1) for v in bp.launches("thvm_hip_linear_grad", 1, 2, 3, 4, 5, 6, 7, 1, m, k, n, dt)[-2:]]


# 32-bit tiles as they lie: whole units of 64 k and what is left of them, odd rows and columns, 1 to 4 splits
DIRECT = [((300, 700, 3001), 1), ((127, 4001, 4095), 2), ((64, 4001, 5003), 2), ((64, 4096, 4096), 4), ((700, 5001, 299), 4), ((128, 2049, 4094), 2)]


@pytest.mark.parametrize("shape,splits", DIRECT, ids=str)
def test_tiles_as_they_lie(hip, shape, splits):
    assert kernel(*shape, F32) == ("thvm_direct_f32", splits)
    _, x, w, bias, res = _linear_inputs(*shape, F32, sum(shape))
    _linear_check(hip, x, w, bias, res, "relu", F32)


def _edges(n):
    """Around the ends of tiles of 64, 128 and 256, the first and the last, and some between."""
    at = np.r_[0:3, 30:34, 62:66, 126:130, 190:194, 254:258, np.linspace(0, n - 1, 24).astype(int), n - 70:n - 66, n - 3:n]
    return np.unique(at[(at >= 0) & (at < n)])


# packed, and in 16 bits as they lie
LAYERS = [((2100, 70, 1900), F16, "thvm_gemm_64x64_f16"), ((1500, 1601, 1499), F16, "thvm_gemm_128x128_f16"),
          ((8000, 150, 8001), F16, "thvm_gemm_256x256_f16"), ((2100, 70, 1900), F32, "thvm_gemm_64x64_f32"),
          ((1500, 1601, 1499), F32, "thvm_gemm_128x128_f32"), ((8000, 150, 8001), F32, "thvm_gemm_256x256_f32"),
          ((70, 1192, 264), F16, "thvm_gemm_rc_64x64_f16"), ((4104, 1032, 4104), F16, "thvm_gemm_rc_128x128_f16"),
          ((8008, 152, 8008), F16, "thvm_gemm_rc_256x256_f16")]


@pytest.mark.parametrize("shape,dt,name", LAYERS, ids=str)
def test_layers(hip, shape, dt, name):
    assert kernel(*shape, dt)[0] == name
    m, k, n = shape
    rng = np.random.default_rng(m + n)
    x, w = rng.standard_normal((m, k), np.float32).astype(NP[dt]), (rng.standard_normal((k, n), np.float32) / np.float32(math.sqrt(k))).astype(NP[dt])
    bias, row = rng.standard_normal((2, n), np.float32).astype(NP[dt])
    res = np.broadcast_to(row, (m, n))
    y, z = bo.run_linear(hip, x, w, bias, res, "relu", dt)
    r, c = _edges(m), _edges(n)
    x64, w64 = x[r].astype(np.float64), w[:, c].astype(np.float64)
    want = x64 @ w64 + bias[c].astype(np.float64)
    bound = (2 * k + 9) * U32 * (np.abs(x64) @ np.abs(w64) + np.abs(bias[c].astype(np.float64)))
    within(z[r][:, c], want, bound + bo.rounding(dt, want))
    full = np.maximum(want, 0) + row[c].astype(np.float64)
    within(y[r][:, c], full, bound + U32 * np.abs(full) + bo.rounding(dt, full))


# tiles of 64, 128 and 256 with ragged edges, with and without K splits
GRADS = [((300, 130, 2049), ("thvm_gemm_64x64", True), ("thvm_gemm_64x64", False)), ((4100, 70, 90), ("thvm_gemm_64x64", False), ("thvm_gemm_64x64", True)),
         ((1700, 1500, 1601), ("thvm_gemm_128x128", False), ("thvm_gemm_128x128", False)), ((3500, 3401, 3301), ("thvm_gemm_128x128", False), ("thvm_gemm_128x128", False)),
         ((8000, 7999, 150), ("thvm_gemm_256x256", False), ("thvm_gemm_128x128", True)), ((150, 8001, 7900), ("thvm_gemm_128x128", True), ("thvm_gemm_256x256", False))]


@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape,dx_kernel,dw_kernel", GRADS, ids=str)
def test_gradients(hip, shape, dx_kernel, dw_kernel, dt):
    tail = "_f16" if dt == F16 else "_f32"
    assert kernels(*shape, dt) == [(v[0] + tail, v[1]) for v in (dx_kernel, dw_kernel)]
    m, k, n = shape
    rng = np.random.default_rng(m + n)
    x, w = rng.standard_normal((m, k), np.float32).astype(NP[dt]), (rng.standard_normal((k, n), np.float32) / np.float32(math.sqrt(k))).astype(NP[dt])
    dy, z = (np.float32(0.1) * rng.standard_normal((m, n), np.float32)).astype(NP[dt]), rng.standard_normal((m, n), np.float32).astype(NP[dt])
    name = ACTS[2 + m % 3]
    got = bo.run_linear_grad(hip, dy, z, x, w, name, dt)
    again = bo.run_linear_grad(hip, dy, z, x, w, name, dt)
    assert all(np.array_equal(p, q) for p, q in zip(got, again))       # no order of sums depends on the run
    rm, rk, rn = _edges(m), _edges(k), _edges(n)

    def dz(rows, cols):
        d, v = dy[rows][:, cols].astype(np.float64), z[rows][:, cols].astype(np.float64)
        out = d * bo.slope(name, v)
        # act' in 32 bits; of f16, dz is rounded once more before the products
        off = np.abs(d) * (16 * U32 * (1 + np.abs(v))) + (np.abs(out) * 2.0 ** -11 + 2.0 ** -25 if dt == F16 else 0.0)
        return out, off

    full = slice(None)
    d, off = dz(rm, full)
    w64 = w[rk].astype(np.float64)
    want = d @ w64.T
    within(got[0][rm][:, rk], want, (2 * n + 8) * U32 * (np.abs(d) @ np.abs(w64.T)) + 1.01 * off @ np.abs(w64.T) + bo.rounding(dt, want) + 1e-40)
    d, off = dz(full, rn)
    x64 = x[:, rk].astype(np.float64)
    want = x64.T @ d
    within(got[1][rk][:, rn], want, (2 * m + 8) * U32 * (np.abs(x64.T) @ np.abs(d)) + 1.01 * np.abs(x64.T) @ off + bo.rounding(dt, want) + 1e-40)
    want = d.sum(0)
    off = np.abs(dy[:, rn].astype(np.float64)) * (16 * U32 * (1 + np.abs(z[:, rn].astype(np.float64))))
    within(got[2][rn], want, off.sum(0) + (m + 4) * U32 * np.abs(d).sum(0) + bo.rounding(dt, want) + 1e-40)


@pytest.mark.parametrize("rows,cols", [(3, 30001), (2, 24576)], ids=str)
def test_layer_norm_of_long_rows(hip, rows, cols):
    """16-bit rows that fill a workgroup's registers."""
    assert bp.names("thvm_hip_layer_norm", 1, 2, 3, 4, 5, 6, rows, cols, 1e-5, F16) == ["thvm_ln_f16_1024_4"]
    rng, x, gamma, beta = _ln_inputs(rows, cols, F16, cols)
    _ln_check(hip, x, gamma, beta, 1e-5, F16)
    _, mean, rstd = (v.astype(np.float32) for v in bo.layer_norm(x, None, None, 1e-5))
    dy, add = (0.1 * rng.standard_normal((2, rows, cols))).astype(np.float16)
    _lng_check(hip, dy, x, mean, rstd, gamma, add, F16)
