"""Timed cases of the dense-layer and layer-norm operators (mace_inference.operators).

The four calls are the building blocks of the radial networks (Linear, LayerNorm, SiLU) and of any
head that is trained or served beside the model:

  dense                y = act(x W^T + b) + r            (z = x W^T + b kept for training)
  dense_backward       dx, dW, db                        from dy, x, W and z
  layer_norm           y = act(xhat gamma + beta)        xhat = (x - mean) rstd, row by row
  layer_norm_backward  dx, dgamma, dbeta                 from dy, x, mean, rstd, gamma, beta

``run`` computes a case in plain torch operations, or (``own``) with the framework's kernels.
"""
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def dense_case(name, dtype, rows, inputs, outputs, act="none", bias=True, residual=False, keep=False):
    return {"name": name, "op": "dense", "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs,
            "act": act, "bias": bias, "residual": residual, "keep": keep}


def dense_backward_case(name, dtype, rows, inputs, outputs, act="none"):
    return {"name": name, "op": "dense_backward", "dtype": dtype, "rows": rows, "inputs": inputs,
            "outputs": outputs, "act": act}


def norm_case(name, op, dtype, rows, width, act="none"):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width, "act": act}


def listed():
    return [
        # The radial network's first layer (10 Bessel functions -> 64) over the edges of a small
        # cell: rows of 40 bytes, a call that is all latency.
        dense_case("dense f32 5417x10-64", "f32", 5417, 10, 64),
        # Its projection onto the 10 tensor-product paths (64 -> 1280), edges of a 1,000-atom cell.
        dense_case("dense f32 84613x64-1280", "f32", 84613, 64, 1280),
        # A residual block on the node features of a 10,000-atom cell.
        dense_case("dense f32 10000x512-512 silu", "f32", 10000, 512, 512, "silu", residual=True),
        # One token through a wide layer: the weights are read once.
        dense_case("dense bf16 1x4096-16384 gelu", "bf16", 1, 4096, 16384, "gelu"),
        # A training step's first feed-forward product, z kept for the backward pass.
        dense_case("dense bf16 8192x4096-16384", "bf16", 8192, 4096, 16384, "gelu", keep=True),
        # A ragged batch through odd widths: no row of the output starts on a vector boundary.
        dense_case("dense f16 1237x1000-2055 relu", "f16", 1237, 1000, 2055, "relu", residual=True),
        # Gradients of the projection.
        dense_backward_case("dense_bwd f32 84613x64-1280", "f32", 84613, 64, 1280),
        # Gradients of a feed-forward product with its activation.
        dense_backward_case("dense_bwd bf16 4096x2048-8192", "bf16", 4096, 2048, 8192, "silu"),
        # The radial network's LayerNorm + SiLU over the same edges, forward and backward.
        norm_case("norm f32 84613x64 silu", "layer_norm", "f32", 84613, 64, "silu"),
        norm_case("norm_bwd f32 84613x64 silu", "layer_norm_backward", "f32", 84613, 64, "silu"),
        # Wide rows of a training batch, and odd ones.
        norm_case("norm bf16 16384x4096", "layer_norm", "bf16", 16384, 4096),
        norm_case("norm_bwd f16 8191x2053", "layer_norm_backward", "f16", 8191, 2053),
    ]


def between(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["dense", "dense", "dense_backward", "layer_norm", "layer_norm_backward"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["none", "silu", "gelu", "relu"])
    while True:
        if op.startswith("dense"):
            wide = 2048 if dtype == "f32" else 16384
            case = {"op": op, "dtype": dtype, "rows": between(rng, 1, 84613), "inputs": between(rng, 1, wide),
                    "outputs": between(rng, 1, wide), "act": act}
            if op == "dense":
                case.update(bias=rng.random() < 0.7, residual=rng.random() < 0.4, keep=rng.random() < 0.4)
        else:
            # From 8 values a row on: fewer leave a gradient that is mostly cancellation.  No relu
            # in the backward pass: its step lands on another side of a value that rounds to zero.
            case = {"op": op, "dtype": dtype, "rows": between(rng, 1, 84613), "width": between(rng, 8, 16384),
                    "act": "silu" if act == "relu" and op == "layer_norm_backward" else act}
        w = work(case)
        if w["flops"] <= 2.0 * 8192 * 4096 * 16384 and w["bytes"] <= 5e8:
            return case


def work(case):
    b, rows = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "dense":
        k, n = case["inputs"], case["outputs"]
        moved = rows * k + n * k + rows * n * (1 + case["residual"] + case["keep"]) + n * case["bias"]
        return {"bytes": b * moved, "flops": 2 * rows * n * k}
    if case["op"] == "dense_backward":
        k, n = case["inputs"], case["outputs"]
        moved = rows * n * (1 + (case["act"] != "none")) + 2 * rows * k + 2 * n * k + n
        return {"bytes": b * moved, "flops": 4 * rows * n * k}
    n = case["width"]
    if case["op"] == "layer_norm":
        return {"bytes": b * (2 * rows * n + 2 * n) + 8 * rows, "flops": 8 * rows * n}
    return {"bytes": b * (3 * rows * n + 4 * n) + 8 * rows, "flops": 16 * rows * n}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows = DTYPES[case["dtype"]], case["rows"]

    def normal(*shape, scale=1.0, shift=0.0):
        v = torch.randn(*shape, device="cuda", generator=g)
        return v.mul_(scale).add_(shift).to(dtype)

    s = {"op": case["op"], "act": None if case["act"] == "none" else case["act"]}
    if case["op"].startswith("dense"):
        k, n = case["inputs"], case["outputs"]
        s["x"] = normal(rows, k)
        s["weight"] = normal(n, k, scale=k ** -0.5)
        if case["op"] == "dense":
            s["bias"] = normal(n, scale=0.3) if case["bias"] else None
            s["residual"] = normal(rows, n) if case["residual"] else None
            s["keep"] = case["keep"]
        else:
            s["dy"] = normal(rows, n, scale=0.1)
            s["z"] = None if s["act"] is None else normal(rows, n)
        return s
    n = case["width"]
    s["x"] = normal(rows, n, scale=1.7, shift=0.4)
    s["gamma"] = normal(n, scale=0.2, shift=1.0)
    s["beta"] = normal(n, scale=0.2)
    if case["op"] == "layer_norm_backward":
        s["dy"] = normal(rows, n, scale=0.1)
        x = s["x"].float()
        s["mean"] = x.mean(1)
        s["rstd"] = ((x - s["mean"][:, None]).square().mean(1) + EPS).rsqrt()
    return s


def activate(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return torch.where(z < 0, torch.zeros_like(z), z) if act == "relu" else z


def slope(z, act):
    """d act / dz."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    return (z > 0).to(z.dtype)


def run(s):
    if own:
        return run_own(s)
    dtype, act = s["x"].dtype, s["act"]
    x = s["x"].float()
    if s["op"] == "dense":
        z = x @ s["weight"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = activate(z, act)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return {"y": y.to(dtype), "z": z.to(dtype)} if s["keep"] else {"y": y.to(dtype)}
    if s["op"] == "dense_backward":
        dz = s["dy"].float()
        if act is not None:
            dz = dz * slope(s["z"].float(), act)
        return {"dx": (dz @ s["weight"].float()).to(dtype), "dweight": (dz.t() @ x).to(dtype),
                "dbias": dz.sum(0).to(dtype)}
    gamma, beta = s["gamma"].float(), s["beta"].float()
    if s["op"] == "layer_norm":
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = (centred.square().mean(1) + EPS).rsqrt()
        y = activate(centred * rstd[:, None] * gamma + beta, act)
        return {"y": y.to(dtype), "mean": mean, "rstd": rstd}
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    dz = s["dy"].float()
    if act is not None:
        dz = dz * slope(xhat * gamma + beta, act)
    dxhat = dz * gamma
    along = (dxhat * xhat).mean(1, keepdim=True)
    dx = s["rstd"][:, None] * (dxhat - dxhat.mean(1, keepdim=True) - xhat * along)
    return {"dx": dx.to(dtype), "dgamma": (dz * xhat).sum(0).to(dtype), "dbeta": dz.sum(0).to(dtype)}


def run_own(s):
    if "lasp-pis_b200/python" not in sys.path:
        sys.path.insert(0, "lasp-pis_b200/python")
    from mace_inference import operators as op
    if s["op"] == "dense":
        if s["keep"]:
            y, z = op.dense(s["x"], s["weight"], s["bias"], s["act"], s["residual"], keep=True)
            return {"y": y, "z": z}
        return {"y": op.dense(s["x"], s["weight"], s["bias"], s["act"], s["residual"])}
    if s["op"] == "dense_backward":
        dx, dweight, dbias = op.dense_backward(s["dy"], s["x"], s["weight"], s["act"], s["z"])
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if s["op"] == "layer_norm":
        y, mean, rstd = op.layer_norm(s["x"], s["gamma"], s["beta"], EPS, s["act"], keep=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    dx, dgamma, dbeta = op.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"], s["beta"],
                                               s["act"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def exact(case, seed):
    """The definitions in 64 bits: products by einsum, means and variances from raw moments about
    a row's first value, gradients by automatic differentiation."""
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    act = {None: lambda v: v, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "relu": torch.nn.functional.relu}[s["act"]]
    x = s["x"]
    if s["op"] == "dense":
        z = torch.einsum("mk,nk->mn", x, s["weight"])
        z = z if s["bias"] is None else z + s["bias"]
        y = act(z) if s["residual"] is None else act(z) + s["residual"]
        return {"y": y, "z": z} if s["keep"] else {"y": y}
    if s["op"] == "dense_backward":
        dz = s["dy"]
        if s["z"] is not None:
            z = s["z"].requires_grad_()
            dz, = torch.autograd.grad(act(z), z, dz)
        return {"dx": torch.einsum("mn,nk->mk", dz, s["weight"]), "dweight": torch.einsum("mn,mk->nk", dz, x),
                "dbias": torch.einsum("mn->n", dz)}
    if s["op"] == "layer_norm":
        first = x[:, :1]
        m1, m2 = (x - first).mean(1), (x - first).square().mean(1)
        rstd = (m2 - m1 * m1 + EPS) ** -0.5
        mean = first[:, 0] + m1
        return {"y": act((x - mean[:, None]) * rstd[:, None] * s["gamma"] + s["beta"]), "mean": mean, "rstd": rstd}
    # With xhat fixed by the given statistics, the parameters' gradients are those of
    # act(xhat gamma + beta); dx adds the statistics' own dependence on x.
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    leaves = [v.requires_grad_() for v in (xhat, s["gamma"], s["beta"])]
    dxhat, dgamma, dbeta = torch.autograd.grad(act(leaves[0] * leaves[1] + leaves[2]), leaves, s["dy"])
    xhat, n = xhat.detach(), x.shape[1]
    inner = torch.einsum("rn,rn->r", dxhat, xhat) / n
    dx = s["rstd"][:, None] * (dxhat - dxhat.sum(1, keepdim=True) / n - xhat * inner[:, None])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
