"""The operators of a residual feed-forward block and of its training, as
measurable cases.

  layer_norm        y = (x - mean) * rstd * gamma + beta over each row
  layer_norm_grad   the gradients of x, gamma and beta, with the gradient that
                    reaches the block's input past the normalisation added in
  linear            y = act(x W + b) + r: a layer with its bias, activation and
                    residual
  linear_grad       the gradients of x, W and b from that of y and the values
                    before the activation
  muon              one optimiser step on weight matrices: the momentum,
                    orthogonalised by Newton-Schulz products, off the weights

Each case is one call. `own` chooses between the plain form (elementary torch
operations in 32 bits) and the backend's calls on its own buffers.
"""
import ctypes as C
import math

import torch

own = False
DEV = "cuda:0"
EPS = 1e-5
# the coefficients of the quintic step and what keeps the norm of a zero matrix off zero
NS_A, NS_B, NS_C, NS_EPS = 3.4445, -4.7750, 2.0315, 1e-7
BETA, LR, DECAY, STEPS = 0.95, 0.02, 0.01, 5
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


# ---- the cases ---------------------------------------------------------

def listed():
    return [
        # a handful of tokens being answered: no statistics are kept
        {"name": "ln_8x4096_f16", "op": "layer_norm", "rows": 8, "cols": 4096, "dtype": "f16", "stats": False},
        # a training batch in 32 bits, statistics kept for the gradient
        {"name": "ln_8192x4096", "op": "layer_norm", "rows": 8192, "cols": 4096, "dtype": "f32", "stats": True},
        # an odd number of rows of a width that ends inside a vector block, in 32 bits
        {"name": "ln_grad_4097x1000", "op": "layer_norm_grad", "rows": 4097, "cols": 1000, "dtype": "f32", "add": True},
        # a training batch in 16 bits
        {"name": "ln_grad_8192x4096_f16", "op": "layer_norm_grad", "rows": 8192, "cols": 4096, "dtype": "f16", "add": True},
        # a single token through a large layer: bound by the weights' bytes
        {"name": "linear_1x4096x4096_f16", "op": "linear", "m": 1, "k": 4096, "n": 4096, "dtype": "f16", "act": "gelu_tanh",
         "bias": True, "residual": True, "keep": False},
        # the benchmark network's first layer: a small training batch
        {"name": "linear_64x784x128", "op": "linear", "m": 64, "k": 784, "n": 128, "dtype": "f32", "act": "relu",
         "bias": True, "residual": False, "keep": True},
        # sizes that fit no tile, with the residual added
        {"name": "linear_1031x771x1501", "op": "linear", "m": 1031, "k": 771, "n": 1501, "dtype": "f32", "act": "silu",
         "bias": True, "residual": True, "keep": True},
        # the benchmark's largest layer, held in 16 bits
        {"name": "linear_4096_f16", "op": "linear", "m": 4096, "k": 4096, "n": 4096, "dtype": "f16", "act": "gelu",
         "bias": True, "residual": True, "keep": True},
        # its gradient in 32 bits
        {"name": "linear_grad_4096", "op": "linear_grad", "m": 4096, "k": 4096, "n": 4096, "dtype": "f32", "act": "gelu"},
        # a middling layer's gradient in 16 bits
        {"name": "linear_grad_2048_f16", "op": "linear_grad", "m": 2048, "k": 2048, "n": 2048, "dtype": "f16", "act": "gelu_tanh"},
        # the benchmark network's first weights: launches count
        {"name": "muon_784x128", "op": "muon", "count": 1, "rows": 784, "cols": 128, "dtype": "f32", "nesterov": True},
        # the weights of the benchmark's largest layer
        {"name": "muon_4096x4096", "op": "muon", "count": 1, "rows": 4096, "cols": 4096, "dtype": "f32", "nesterov": True},
    ]


def _log(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: odd ones as likely as their neighbours."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm_grad", "linear", "linear", "linear", "linear_grad", "linear_grad", "muon", "muon"])
    dtype = rng.choice(["f32", "f16"])
    if op.startswith("layer_norm"):
        rows, cols = _log(rng, 1, 16384), _log(rng, 64, 8192)
        if rng.random() < 0.5:   # widths are often round, batches less so
            cols = cols // 64 * 64
        while rows * cols > 8192 * 4096:
            rows = max(1, rows // 2)
        c = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
        c["stats" if op == "layer_norm" else "add"] = rng.random() < 0.5
        return c
    if op == "muon":
        c = {"op": op, "count": rng.choice([1, 1, 2, 4]), "rows": _log(rng, 64, 4096), "cols": _log(rng, 64, 4096), "dtype": dtype,
             "nesterov": rng.random() < 0.7}
        if rng.random() < 0.6:
            c["rows"], c["cols"] = c["rows"] // 32 * 32, c["cols"] // 32 * 32
        while c["count"] * c["rows"] * c["cols"] * min(c["rows"], c["cols"]) > 4096 ** 3:
            c["count"] = max(1, c["count"] // 2)
        return c
    m = _log(rng, 1, 16) if op == "linear" and rng.random() < 0.3 else _log(rng, 8, 4096)
    k, n = _log(rng, 64, 4096), _log(rng, 64, 4096)
    if rng.random() < 0.6:
        k, n = k // 16 * 16, n // 16 * 16
    c = {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": rng.choice(ACTS)}
    if op == "linear":
        c["bias"], c["residual"], c["keep"] = rng.random() < 0.8, rng.random() < 0.5, m > 16 and rng.random() < 0.5
    return c


# ---- inputs ------------------------------------------------------------

def _dt(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _inputs(case, seed):
    """The tensors a program has in hand, by name, made on the GPU from the seed."""
    g = torch.Generator(DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0, dt=_dt(case)):
        return torch.randn(shape, generator=g, device=DEV).mul_(std).add_(mean).to(dt)

    op, t = case["op"], {}
    if op.startswith("layer_norm"):
        r, c = case["rows"], case["cols"]
        # activations: a few features stand out, each row has a mean of its own
        feature = normal(c, std=0.5, dt=torch.float32).exp_()
        x = normal(r, c, dt=torch.float32).mul_(feature).add_(normal(r, 1, std=0.5, dt=torch.float32))
        t["x"] = x.to(_dt(case))
        t["gamma"] = normal(c, std=0.1, mean=1.0)
        if op == "layer_norm":
            t["beta"] = normal(c, std=0.1)
            return t
        t["dy"] = normal(r, c, std=0.02)
        if case["add"]:
            t["add"] = normal(r, c, std=0.02)
        x = t["x"].float()
        t["mean"] = x.mean(1)
        t["rstd"] = torch.rsqrt((x - t["mean"][:, None]).square().mean(1) + EPS)
        return t
    if op == "muon":
        cnt, r, c = case["count"], case["rows"], case["cols"]
        k = max(1, min(r, c) // 4)    # a batch's gradient: a product of fewer rows than the matrix has, and noise

        def gradient(std):
            low = torch.matmul(normal(cnt, r, k, dt=torch.float32), normal(cnt, k, c, dt=torch.float32)).mul_(std / math.sqrt(k))
            return low.add_(normal(cnt, r, c, std=0.3 * std, dt=torch.float32))

        t["param"] = normal(cnt, r, c, std=1 / math.sqrt(r))
        t["grad"] = gradient(1e-2).to(_dt(case))
        t["m"] = gradient(1e-1)
        return t
    m, k, n = case["m"], case["k"], case["n"]
    t["x"] = normal(m, k)
    t["w"] = normal(k, n, std=1 / math.sqrt(k))
    if op == "linear":
        if case["bias"]:
            t["b"] = normal(n, std=0.1)
        if case["residual"]:
            t["r"] = normal(m, n)
        return t
    t["dy"] = normal(m, n, std=0.02)
    if case["act"] != "none":
        t["z"] = normal(m, n)
    return t


# ---- the plain forms ---------------------------------------------------

def _act(name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-u * (z + 0.044715 * z * z * z)))
        return s + z * s * (1 - s) * u * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def _plain_layer_norm(case, t):
    x = t["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    out = {"y": (d * rstd * t["gamma"].float() + t["beta"].float()).to(_dt(case))}
    if case["stats"]:
        out["mean"], out["rstd"] = mean[:, 0], rstd[:, 0]
    return out


def _plain_layer_norm_grad(case, t):
    dy, rstd = t["dy"].float(), t["rstd"][:, None]
    xh = (t["x"].float() - t["mean"][:, None]) * rstd
    g = dy * t["gamma"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if case["add"]:
        dx = dx + t["add"].float()
    return {"dx": dx.to(_dt(case)), "dgamma": (dy * xh).sum(0).to(_dt(case)), "dbeta": dy.sum(0).to(_dt(case))}


def _plain_linear(case, t):
    z = torch.matmul(t["x"].float(), t["w"].float())
    if case["bias"]:
        z = z + t["b"].float()
    y = _act(case["act"], z)
    if case["residual"]:
        y = y + t["r"].float()
    out = {"y": y.to(_dt(case))}
    if case["keep"]:
        out["z"] = z.to(_dt(case))
    return out


def _plain_linear_grad(case, t):
    dz = t["dy"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(case["act"], t["z"].float())
    dx = torch.matmul(dz, t["w"].float().t())
    dw = torch.matmul(t["x"].float().t(), dz)
    return {"dx": dx.to(_dt(case)), "dw": dw.to(_dt(case)), "db": dz.sum(0).to(_dt(case))}


def _plain_muon(case, t):
    g, p, m = t["grad"].float(), t["param"], t["m"]
    m.mul_(BETA).add_(g)
    u = g + BETA * m if case["nesterov"] else m
    x = u / ((u * u).sum((1, 2), keepdim=True).sqrt() + NS_EPS)
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        a = torch.matmul(x, x.transpose(1, 2))
        b = NS_B * a + NS_C * torch.matmul(a, a)
        x = NS_A * x + torch.matmul(b, x)
    if tall:
        x = x.transpose(1, 2)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    p.copy_((1 - LR * DECAY) * p.float() - LR * scale * x)
    return {"param": p, "m": m}


_PLAIN = {"layer_norm": _plain_layer_norm, "layer_norm_grad": _plain_layer_norm_grad, "linear": _plain_linear,
          "linear_grad": _plain_linear_grad, "muon": _plain_muon}


# ---- the backend's calls -----------------------------------------------

_live = 0


class _Buffers:
    """The backend buffers of one state; given back when their last user (the
    state, or a tensor over one of them) is gone."""

    def __init__(self):
        global _live
        from tinyhvm_amd import _lib
        self.L, self.ids = _lib.lib(), []
        _live += 1
        if _live == 1:
            if self.L.thvm_hip_stream() is None:
                if self.L.thvm_hip_init() != 0:
                    raise RuntimeError("the HIP backend does not initialise on this device")
            else:
                self.L.thvm_hip_pool_reset(0)   # no buffer is in use: numbering starts again
        self.L.thvm_hip_synchronize()           # torch fills buffers that earlier work may have used

    def tensor(self, shape, dt):
        """(id, torch's view) of a new buffer."""
        n = math.prod(shape) * (2 if dt == torch.float16 else 4)
        i = self.L.thvm_hip_buf_alloc(max(4, n))
        if not i:
            raise RuntimeError("out of memory: no backend buffer of %d bytes" % n)
        self.ids.append(i)
        return i, torch.as_tensor(_Memory(self, i, shape, dt), device=DEV)

    def put(self, t):
        i, v = self.tensor(tuple(t.shape), t.dtype)
        v.copy_(t)
        return i, v

    def __del__(self):
        global _live
        for i in self.ids:
            self.L.thvm_hip_buf_free(i)
        _live -= 1


class _Memory:
    """A buffer's device memory as torch sees it."""

    def __init__(self, bufs, i, shape, dt):
        self.bufs = bufs
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f2" if dt == torch.float16 else "<f4", "version": 3,
                                         "strides": None, "data": (bufs.L.thvm_hip_buf_device_ptr(i), False)}


def _backend_state(case, t):
    """The call of one pass and the tensors it leaves its outputs in."""
    from tinyhvm_amd import abi
    bufs = _Buffers()
    L, dt = bufs.L, _dt(case)
    code = abi.DTYPE_F16 if dt == torch.float16 else abi.DTYPE_F32
    op, outs = case["op"], {}
    if op == "muon":
        cnt, r, c = case["count"], case["rows"], case["cols"]
        ids, views = {}, {}
        for name in ("param", "grad", "m"):
            got = [bufs.put(v) for v in t[name]]
            ids[name], views[name] = (C.c_uint32 * cnt)(*[i for i, _ in got]), [v for _, v in got]
        scale = math.sqrt(max(1.0, r / c))
        args = (ids["param"], ids["grad"], ids["m"], cnt, r, c, LR, scale, DECAY, BETA, int(case["nesterov"]), STEPS, code)
        return {"call": L.thvm_hip_muon_step, "args": args, "outs": {"param": views["param"], "m": views["m"]}, "bufs": bufs}
    b = {name: bufs.put(v)[0] for name, v in t.items()}

    def out(name, shape, d=dt):
        i, outs[name] = bufs.tensor(shape, d)
        return i

    if op == "layer_norm":
        r, c = case["rows"], case["cols"]
        mean, rstd = (out(s, (r,), torch.float32) if case["stats"] else 0 for s in ("mean", "rstd"))
        call, args = L.thvm_hip_layer_norm, (out("y", (r, c)), mean, rstd, b["x"], b["gamma"], b["beta"], r, c, EPS, code)
    elif op == "layer_norm_grad":
        r, c = case["rows"], case["cols"]
        call = L.thvm_hip_layer_norm_grad
        args = (out("dx", (r, c)), out("dgamma", (c,)), out("dbeta", (c,)), b["dy"], b["x"], b["mean"], b["rstd"], b["gamma"],
                b.get("add", 0), r, c, code)
    else:
        m, k, n, act = case["m"], case["k"], case["n"], ACTS.index(case["act"])
        if op == "linear":
            call = L.thvm_hip_linear
            args = (out("y", (m, n)), out("z", (m, n)) if case["keep"] else 0, b["x"], b["w"], b.get("b", 0), b.get("r", 0), act,
                    m, k, n, code)
        else:
            call = L.thvm_hip_linear_grad
            args = (out("dx", (m, k)), out("dw", (k, n)), out("db", (n,)), b["dy"], b.get("z", 0), b["x"], b["w"], act, m, k, n, code)
    return {"call": call, "args": args, "outs": outs, "bufs": bufs}


# ---- the interface -----------------------------------------------------

def prepare(case, seed):
    t = _inputs(case, seed)
    return _backend_state(case, t) if own else {"case": case, "t": t}


def run(state):
    if own:
        if state["call"](*state["args"]) != 0:
            raise RuntimeError("the call was refused")
        return state["outs"]
    out = _PLAIN[state["case"]["op"]](state["case"], state["t"])
    if state["case"]["op"] == "muon":   # a program keeps its matrices apart
        return {name: list(v) for name, v in out.items()}
    return out


def work(case):
    op, s = case["op"], 2 if case["dtype"] == "f16" else 4
    if op.startswith("layer_norm"):
        r, c = case["rows"], case["cols"]
        if op == "layer_norm":
            return {"bytes": s * (2 * r * c + 2 * c) + (8 * r if case["stats"] else 0), "flops": 8 * r * c}
        return {"bytes": s * ((4 if case["add"] else 3) * r * c + 3 * c) + 8 * r, "flops": 14 * r * c}
    if op == "muon":
        r, c = case["rows"], case["cols"]
        n, w = min(r, c), max(r, c)
        # X X^T and its square are symmetric: half of each suffices
        return {"bytes": case["count"] * r * c * (3 * s + 8), "flops": case["count"] * STEPS * (n * n * w + n ** 3 + 2 * n * n * w)}
    m, k, n = case["m"], case["k"], case["n"]
    if op == "linear":
        mn = 1 + int(case["residual"]) + int(case["keep"])
        return {"bytes": s * (m * k + k * n + mn * m * n + (n if case["bias"] else 0)), "flops": 2 * m * k * n}
    mn = 1 if case["act"] == "none" else 2
    return {"bytes": s * (2 * m * k + 2 * k * n + mn * m * n + n), "flops": 4 * m * k * n}


# ---- in 64 bits --------------------------------------------------------

def _activation64(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z * 1.0


def _exact_muon(case, t):
    g, m = t["grad"], BETA * t["m"] + t["grad"]
    u = g + BETA * m if case["nesterov"] else m
    x = u / (torch.linalg.matrix_norm(u)[:, None, None] + NS_EPS)
    eye = torch.eye(min(case["rows"], case["cols"]), dtype=torch.float64, device=DEV)
    for _ in range(STEPS):   # x (a + b G + c G G) with the Gram matrix G of the shorter side, on that side
        if case["rows"] > case["cols"]:
            gram = torch.matmul(x.mT.contiguous(), x)
            x = torch.matmul(x, NS_A * eye + torch.matmul(gram, NS_B * eye + NS_C * gram))
        else:
            gram = torch.matmul(x, x.mT.contiguous())
            x = torch.matmul(NS_A * eye + torch.matmul(gram, NS_B * eye + NS_C * gram), x)
    scale = max(1.0, case["rows"] / case["cols"]) ** 0.5
    return {"param": list(t["param"] - LR * (DECAY * t["param"] + scale * x)), "m": list(m)}


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    op = case["op"]
    if op == "muon":
        return _exact_muon(case, t)
    if op == "layer_norm":
        var, mean = torch.var_mean(t["x"], 1, correction=0, keepdim=True)
        out = {"y": (t["x"] - mean) / (var + EPS).sqrt() * t["gamma"] + t["beta"]}
        if case["stats"]:
            out["mean"], out["rstd"] = mean[:, 0], (var + EPS).rsqrt()[:, 0]
        return out
    if op == "layer_norm_grad":
        # of the normalisation whose statistics are the ones in hand: x's own, to 32 bits
        x, gamma = t["x"].requires_grad_(), t["gamma"].requires_grad_()
        beta = torch.zeros_like(t["gamma"]).requires_grad_()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / (var + EPS).sqrt() * gamma + beta
        dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), t["dy"])
        return {"dx": dx + t["add"] if case["add"] else dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "linear":
        z = torch.mm(t["x"], t["w"]) + (t["b"] if case["bias"] else 0.0)
        out = {"y": _activation64(case["act"], z) + (t["r"] if case["residual"] else 0.0)}
        if case["keep"]:
            out["z"] = z
        return out
    dz = t["dy"]
    if case["act"] != "none":
        z = t["z"].requires_grad_()
        dz, = torch.autograd.grad(_activation64(case["act"], z), z, t["dy"])
    return {"dx": torch.mm(dz, t["w"].t().contiguous()), "dw": torch.mm(t["x"].t().contiguous(), dz), "db": torch.sum(dz, 0)}
