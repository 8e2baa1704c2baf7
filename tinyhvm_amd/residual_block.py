"""A residual feed-forward block and its training on the backend's operators:

    h = layer_norm(x);  a = gelu(h W1 + b1);  y = x + a W2 + b2

The matrices are stepped by the orthogonalised optimiser (thvm_hip_muon_step),
the vectors by adam_step, all on the backend's buffers and stream:

    python -m tinyhvm_amd.residual_block --rows 1024 --width 512 --hidden 2048

fits the block to a fixed random one of the same shape and prints the loss.
With --graph a step is captured once and launched again for each pass.
"""
import argparse
import ctypes as C
import math

import numpy as np

from . import _lib, abi

F32 = abi.DTYPE_F32
GELU = 2


def _one(i):
    return (C.c_uint32 * 1)(i)


def _view(rows, cols, stride=None):
    """[rows][cols] row-major, or one element everywhere (stride 0)."""
    v = abi.View()
    v.shape.rank, v.numel = 2, rows * cols
    v.shape.dims[0], v.shape.dims[1] = rows, cols
    v.strides[0], v.strides[1] = (cols, 1) if stride is None else (stride, stride)
    return v


def shape_factor(inputs, outputs):
    """The published factor of an orthogonalised update (K. Jordan et al.,
    "Muon", 2024): sqrt(max(1, outputs / inputs)). Matrices lie here as
    [inputs][outputs]."""
    return math.sqrt(max(1.0, outputs / inputs))


class ResidualBlock:
    """The block's buffers and its calls, for `rows` inputs at a time."""

    VECTORS = ("gamma", "beta", "b1", "b2")
    MATRICES = ("w1", "w2")

    def __init__(self, rows, width, hidden, seed=0):
        self.L = _lib.lib()
        self.rows, self.width, self.hidden = rows, width, hidden
        self.shapes = {"gamma": (width,), "beta": (width,), "w1": (width, hidden), "b1": (hidden,), "w2": (hidden, width), "b2": (width,)}
        self.buf, self.shape_of, self.steps = {}, {}, 0
        rng = np.random.default_rng(seed)
        for name, shape in self.shapes.items():
            scale = 1 / math.sqrt(shape[0]) if len(shape) == 2 else 0.0
            self.put(name, scale * rng.standard_normal(shape) + (name == "gamma"))
            self.put("d" + name, np.zeros(shape))
            self.put("m" + name, np.zeros(shape))
            if len(shape) == 1:
                self.put("v" + name, np.zeros(shape))
        r, w, n = rows, width, hidden
        for name, shape in {"x": (r, w), "target": (r, w), "h": (r, w), "mean": (r,), "rstd": (r,), "z": (r, n), "a": (r, n), "y": (r, w),
                            "diff": (r, w), "dy": (r, w), "da": (r, n), "dh": (r, w), "dx": (r, w)}.items():
            self.put(name, np.zeros(shape))
        self.put("scale", np.array([2.0 / (r * w)]))

    def put(self, name, values):
        a = np.ascontiguousarray(values, np.float32)
        if name not in self.buf:
            self.buf[name] = self.L.thvm_hip_buf_alloc(a.nbytes)
            if not self.buf[name]:
                raise MemoryError("no backend buffer of %d bytes" % a.nbytes)
            self.shape_of[name] = a.shape
        self.L.thvm_hip_buf_write(self.buf[name], a.ctypes.data_as(C.c_void_p), a.nbytes)

    def get(self, name):
        a = np.empty(self.shape_of[name], np.float32)
        self.L.thvm_hip_buf_read(self.buf[name], a.ctypes.data_as(C.c_void_p), a.nbytes)
        return a

    def close(self):
        for i in self.buf.values():
            self.L.thvm_hip_buf_free(i)
        self.buf = {}

    @staticmethod
    def _done(rc):
        if rc:
            raise RuntimeError("the backend refused the call (%d)" % rc)

    def forward(self):
        L, b, r, w, n = self.L, self.buf, self.rows, self.width, self.hidden
        self._done(L.thvm_hip_layer_norm(b["h"], b["mean"], b["rstd"], b["x"], b["gamma"], b["beta"], r, w, 1e-5, F32))
        self._done(L.thvm_hip_linear(b["a"], b["z"], b["h"], b["w1"], b["b1"], 0, GELU, r, w, n, F32))
        self._done(L.thvm_hip_linear(b["y"], 0, b["a"], b["w2"], b["b2"], b["x"], 0, r, n, w, F32))

    def backward(self):
        """From the mean squared distance to the target."""
        L, b, r, w, n = self.L, self.buf, self.rows, self.width, self.hidden
        full, one = _view(r, w), _view(r, w, 0)
        L.thvm_hip_op_binary(abi.UOP_SUB, b["diff"], full, F32, b["y"], full, F32, b["target"], full, F32)
        L.thvm_hip_op_binary(abi.UOP_MUL, b["dy"], full, F32, b["diff"], full, F32, b["scale"], one, F32)
        self._done(L.thvm_hip_linear_grad(b["da"], b["dw2"], b["db2"], b["dy"], 0, b["a"], b["w2"], 0, r, n, w, F32))
        self._done(L.thvm_hip_linear_grad(b["dh"], b["dw1"], b["db1"], b["da"], b["z"], b["h"], b["w1"], GELU, r, w, n, F32))
        # dy reaches x past the block as well
        self._done(L.thvm_hip_layer_norm_grad(b["dx"], b["dgamma"], b["dbeta"], b["dh"], b["x"], b["mean"], b["rstd"], b["gamma"], b["dy"],
                                              r, w, F32))

    def update(self, lr, lr_vectors, step):
        L, b = self.L, self.buf
        for name in self.MATRICES:
            rows, cols = self.shapes[name]
            self._done(L.thvm_hip_muon_step(_one(b[name]), _one(b["d" + name]), _one(b["m" + name]), 1, rows, cols, lr,
                                            shape_factor(rows, cols), 0.0, 0.95, 1, 5, F32))
        for name in self.VECTORS:
            L.thvm_hip_adam_step(b[name], b["d" + name], b["m" + name], b["v" + name], lr_vectors, 0.9, 0.99, 1e-8,
                                 1 - 0.9 ** step, 1 - 0.99 ** step, self.shapes[name][0])

    def step(self, lr=0.005, lr_vectors=0.003):
        self.steps += 1
        self.forward()
        self.backward()
        self.update(lr, lr_vectors, self.steps)

    def loss(self):
        return float(np.mean((self.get("y") - self.get("target")) ** 2))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=1024)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--graph", action="store_true", help="capture a step once and launch it (the vectors' bias correction stays the first launch's)")
    a = ap.parse_args(argv)
    L = _lib.lib()
    if L.thvm_hip_init() != 0:
        raise SystemExit("the HIP backend does not initialise on this device")
    rng = np.random.default_rng(1)
    x = rng.standard_normal((a.rows, a.width))
    teacher = ResidualBlock(a.rows, a.width, a.hidden, seed=7)
    teacher.put("x", x)
    teacher.forward()
    block = ResidualBlock(a.rows, a.width, a.hidden, seed=8)
    block.put("x", x)
    block.put("target", teacher.get("y"))
    teacher.close()
    graph, losses = None, []
    for s in range(a.steps):
        if graph:
            if L.thvm_hip_graph_launch(graph) != 0:
                raise RuntimeError("the graph did not launch")
        else:
            block.step()
            if a.graph and s == 0:
                losses.append(block.loss())
                if L.thvm_hip_graph_begin() != 0:
                    raise RuntimeError("no capture")
                block.step()
                graph = L.thvm_hip_graph_end()
        if s % 10 == 0 or s + 1 == a.steps:
            losses.append(block.loss())
            print("step %3d  loss %.6f" % (s, losses[-1]), flush=True)
    if graph:
        L.thvm_hip_graph_destroy(graph)
    block.close()
    return losses


if __name__ == "__main__":
    main()
