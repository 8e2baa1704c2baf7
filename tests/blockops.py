"""Calls of the residual block's operators on numpy arrays, and the same from
their definitions in 64 bits: what the GPU tests compare, kept apart so that
the CPU tests can check the definitions themselves."""
import ctypes as C
import math

import numpy as np

from tinyhvm_amd import _lib, abi

F32, F16 = abi.DTYPE_F32, abi.DTYPE_F16
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
U32 = 2.0 ** -24            # half a unit in the last place of 32 bits, relative
NP = {F32: np.float32, F16: np.float16}

_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(name, z):
    z = np.asarray(z, np.float64)
    with np.errstate(over="ignore"):
        if name == "relu":
            return np.where(z > 0, z, 0.0)
        if name == "gelu":
            return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
        if name == "gelu_tanh":
            return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
        if name == "silu":
            return z / (1 + np.exp(-z))
    return z


def slope(name, z):
    z = np.asarray(z, np.float64)
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        u = math.sqrt(2 / math.pi)
        t = np.tanh(u * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * u * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s + z * s * (1 - s)
    return np.ones_like(z)


def layer_norm(x, gamma, beta, eps):
    x = x.astype(np.float64)
    mean = x.mean(1)
    rstd = 1 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    y = (x - mean[:, None]) * rstd[:, None]
    if gamma is not None:
        y = y * gamma.astype(np.float64)
    if beta is not None:
        y = y + beta.astype(np.float64)
    return y, mean, rstd


def layer_norm_grad(dy, x, mean, rstd, gamma, add):
    dy, x = dy.astype(np.float64), x.astype(np.float64)
    xh = (x - mean.astype(np.float64)[:, None]) * rstd.astype(np.float64)[:, None]
    g = dy if gamma is None else dy * gamma.astype(np.float64)
    dx = rstd.astype(np.float64)[:, None] * (g - g.mean(1)[:, None] - xh * (g * xh).mean(1)[:, None])
    if add is not None:
        dx = dx + add.astype(np.float64)
    return dx, (dy * xh).sum(0), dy.sum(0)


def muon(param, grad, m, lr, scale, decay, beta, nesterov, steps, rounded=None, wide=np.float64):
    """The step in 64 bits, or in `wide`; `rounded`: a type that X, A and B are
    rounded to between products."""
    param, grad, m = (v.astype(wide) for v in (param, grad, m))
    # what the entry point takes of its factors: 32 bits
    lr, scale, decay, beta = (float(np.float32(v)) for v in (lr, scale, decay, beta))
    r = (lambda v: v) if rounded is None else (lambda v: (v * 16384).astype(rounded).astype(wide) / 16384)
    rb = (lambda v: v) if rounded is None else (lambda v: (v * 8192).astype(rounded).astype(wide) / 8192)
    m = wide(beta) * m + grad
    u = grad + wide(beta) * m if nesterov else m
    x = r((u / (np.sqrt((u.astype(np.float64) ** 2).sum()) + 1e-7)).astype(wide))
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    for i in range(steps):
        a = r(x @ x.T)
        b = rb(wide(-4.7750) * a + wide(2.0315) * (a @ a))
        x = wide(3.4445) * x + b @ x
        if i + 1 < steps:
            x = r(x)
    if tall:
        x = x.T
    return wide(1 - lr * decay) * param - wide(lr * scale) * x, m


class Bufs:
    """Backend buffers of arrays; freed at the end."""

    def __init__(self, L):
        self.L, self.ids, self.meta = L, [], {}

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for i in self.ids:
            self.L.thvm_hip_buf_free(i)

    def put(self, a):
        if a is None:
            return 0
        a = np.ascontiguousarray(a)
        i = self.L.thvm_hip_buf_alloc(max(4, a.nbytes))
        assert i
        if a.nbytes:
            self.L.thvm_hip_buf_write(i, a.ctypes.data_as(C.c_void_p), a.nbytes)
        self.ids.append(i)
        self.meta[i] = (a.shape, a.dtype)
        return i

    def out(self, shape, dt):
        """A buffer of NaN, so that what is not written shows."""
        return self.put(np.full(shape, np.nan, dt))

    def get(self, i):
        shape, dt = self.meta[i]
        a = np.empty(shape, dt)
        if a.nbytes:
            self.L.thvm_hip_buf_read(i, a.ctypes.data_as(C.c_void_p), a.nbytes)
        assert self.L.thvm_hip_synchronize() == 0
        return a


def ids(values):
    return (C.c_uint32 * max(1, len(values)))(*values)


def run_linear(L, x, w, bias, res, name, dt, keep=True):
    (m, k), n = x.shape, w.shape[1]
    with Bufs(L) as b:
        y, z = b.out((m, n), NP[dt]), b.out((m, n), NP[dt]) if keep else 0
        rc = L.thvm_hip_linear(y, z, b.put(x), b.put(w), b.put(bias), b.put(res), ACTS.index(name), m, k, n, dt)
        assert rc == 0
        return b.get(y), b.get(z) if keep else None


def run_linear_grad(L, dy, z, x, w, name, dt, want=(True, True, True)):
    (m, n), k = dy.shape, w.shape[0]
    with Bufs(L) as b:
        dx, dw, db = (b.out(s, NP[dt]) if on else 0 for s, on in zip(((m, k), (k, n), (n,)), want))
        rc = L.thvm_hip_linear_grad(dx, dw, db, b.put(dy), b.put(z), b.put(x) if want[1] else 0, b.put(w) if want[0] else 0,
                                    ACTS.index(name), m, k, n, dt)
        assert rc == 0
        return [b.get(i) if i else None for i in (dx, dw, db)]


def run_layer_norm(L, x, gamma, beta, eps, dt, stats=True):
    with Bufs(L) as b:
        y = b.out(x.shape, NP[dt])
        mean, rstd = (b.out((x.shape[0],), np.float32) if stats else 0 for _ in range(2))
        rc = L.thvm_hip_layer_norm(y, mean, rstd, b.put(x), b.put(gamma), b.put(beta), *x.shape, eps, dt)
        assert rc == 0
        return [b.get(i) if i else None for i in (y, mean, rstd)]


def run_layer_norm_grad(L, dy, x, mean, rstd, gamma, add, dt, want=(True, True, True)):
    with Bufs(L) as b:
        r, c = x.shape
        dx, dg, db = (b.out(s, NP[dt]) if on else 0 for s, on in zip(((r, c), (c,), (c,)), want))
        rc = L.thvm_hip_layer_norm_grad(dx, dg, db, b.put(dy), b.put(x), b.put(mean), b.put(rstd), b.put(gamma), b.put(add), r, c, dt)
        assert rc == 0
        return [b.get(i) if i else None for i in (dx, dg, db)]


def run_muon(L, params, grads, ms, lr, scale, decay, beta, nesterov, steps, dt):
    with Bufs(L) as b:
        p, g, m = [b.put(v) for v in params], [b.put(v) for v in grads], [b.put(v) for v in ms]
        rc = L.thvm_hip_muon_step(ids(p), ids(g), ids(m), len(p), *params[0].shape, lr, scale, decay, beta, nesterov, steps, dt)
        assert rc == 0
        return [b.get(i) for i in p], [b.get(i) for i in m]


def rounding(dt, want):
    """What one rounding of an output to its type may add."""
    return (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if dt == F16 else np.abs(want) * U32 + 2.0 ** -149)


def lib():
    return _lib.lib()
