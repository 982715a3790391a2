"""Dense layer and layer norm, forward and backward, on torch CUDA tensors (ctypes over
include/mace/operators.h).

These are the blocks of the MH1 radial networks (Linear, LayerNorm, SiLU) as calls of their own,
for networks that are trained or served beside the model:

    h = dense(x, weight, bias)                                # x weight^T + bias
    y, mean, rstd = layer_norm(h, gamma, beta, activation="silu", keep=True)
    dh, dgamma, dbeta = layer_norm_backward(dy, h, mean, rstd, gamma, beta, "silu")
    dx, dweight, dbias = dense_backward(dh, x, weight)

All tensors of a call have one type (float32, bfloat16 or float16) and one device; statistics
are float32.  A leading tensor is (..., features); tensors whose last index is not contiguous, or
whose leading indices do not collapse into rows, are copied first.  Work is queued on torch's
current stream of the tensors' device, and outputs are new contiguous tensors.  The calls record
no autograd graph: the backward calls give the gradients.  Wrong arguments raise ValueError (or
TypeError), a failed call RuntimeError.
"""
from __future__ import annotations

import ctypes as ct

from .native import _error, load

ACTIVATIONS = {None: 0, "none": 0, "silu": 1, "gelu": 2, "relu": 3}

_bound = None
_types = {}


def _library():
    global _bound
    if _bound is None:
        import torch
        lib = load()
        p, n, i = ct.c_void_p, ct.c_longlong, ct.c_int
        lib.mace_dense.argtypes = [i, n, n, n, p, n, p, n, p, i, p, n, p, n, p, n, p, n, p]
        lib.mace_dense_workspace.argtypes = [i, n, n, n, p, n, p, n]
        lib.mace_dense_workspace.restype = n
        lib.mace_dense_backward.argtypes = [i, n, n, n, p, n, p, n, p, n, i, p, n, p, n, p, n, p, p, n, p]
        lib.mace_dense_backward_workspace.argtypes = [i, n, n, n, p, n, p, n, p, n, i]
        lib.mace_dense_backward_workspace.restype = n
        lib.mace_layer_norm.argtypes = [i, n, n, p, n, p, p, ct.c_float, i, p, n, p, p, p]
        lib.mace_layer_norm_backward.argtypes = [i, n, n, p, n, p, n, p, p, p, p, i, p, n, p, p, p, n, p]
        lib.mace_layer_norm_backward_workspace.argtypes = [i, n, n]
        lib.mace_layer_norm_backward_workspace.restype = n
        _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _bound = lib, torch
    return _bound


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation is one of {', '.join(map(str, ACTIVATIONS))}, not {name!r}") from None


def _type(t, name, torch):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a torch tensor, not {type(t).__name__}")
    code = _types.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} is float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: a CUDA tensor is needed")
    if t.dim() < 1:
        raise ValueError(f"{name} has no dimension")
    return code


def _like(t, x, name, torch, shape, dtype=None):
    """Checks a tensor that goes with `x`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a torch tensor, not {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != (dtype or x.dtype):
        raise TypeError(f"{name} is {t.dtype}, expected {dtype or x.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {x.device}")


def _rows(t):
    """`t` as rows with a contiguous last index: (tensor that keeps the memory alive, address, row distance)."""
    if t.dim() == 2:
        width = t.shape[1]
        s0, s1 = t.stride()
        if (s1 == 1 or width == 1) and (s0 >= width or t.shape[0] <= 1):
            return t, t.data_ptr(), max(s0, width)
    elif t.is_contiguous():
        return t, t.data_ptr(), t.shape[-1]
    else:
        two = t.reshape(-1, t.shape[-1])  # a view where the leading indices collapse
        return _rows(two) if two.dim() == 2 else _rows(two.contiguous())
    t = t.contiguous()
    return t, t.data_ptr(), t.shape[1]


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _address(t):
    return None if t is None else t.data_ptr()


class _On:
    """Makes a device current for a call (and back)."""

    def __init__(self, torch, device):
        self.guard = None
        if torch.cuda.current_device() != device.index:
            self.guard = torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *args):
        if self.guard is not None:
            self.guard.__exit__(*args)


def _stream(torch, device):
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(torch, lib, size, device):
    if size < 0:
        raise RuntimeError(_error(lib))
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _count(shape):
    n = 1
    for v in shape:
        n *= v
    return n


def dense(x, weight, bias=None, activation=None, residual=None, keep=False):
    """``activation(x weight^T + bias) + residual`` for x (..., inputs), weight (outputs, inputs),
    bias (outputs,) and residual (..., outputs).  ``keep=True`` returns (y, z) with
    z = x weight^T + bias, which ``dense_backward`` takes where there is an activation."""
    lib, torch = _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight is a matrix (outputs, inputs)")
    inputs, outputs = x.shape[-1], weight.shape[0]
    _like(weight, x, "weight", torch, (outputs, inputs))
    shape = x.shape[:-1] + (outputs,)
    if bias is not None:
        _like(bias, x, "bias", torch, (outputs,))
        bias = _flat(bias)
    if residual is not None:
        _like(residual, x, "residual", torch, shape)
    device = x.device
    with _On(torch, device):
        y = torch.empty(shape, dtype=x.dtype, device=device)
        z = torch.empty(shape, dtype=x.dtype, device=device) if keep else None
        rows = _count(shape[:-1])
        x, px, ldx = _rows(x)
        weight, pw, ldw = _rows(weight)
        pr, ldr = None, 0
        if residual is not None:
            residual, pr, ldr = _rows(residual)
        size = lib.mace_dense_workspace(code, rows, inputs, outputs, px, ldx, pw, ldw)
        ws = _workspace(torch, lib, size, device)
        if lib.mace_dense(code, rows, inputs, outputs, px, ldx, pw, ldw, _address(bias), act, pr, ldr, y.data_ptr(),
                          outputs, _address(z), outputs, _address(ws), size, _stream(torch, device)):
            raise RuntimeError(_error(lib))
    return (y, z) if keep else y


def dense_backward(dy, x, weight, activation=None, z=None, need=(True, True, True)):
    """(dx, dweight, dbias) of ``dense`` for the output gradient dy (..., outputs); z is what
    ``dense(..., keep=True)`` gave (not needed without an activation).  The residual's gradient
    is dy itself.  ``need`` leaves gradients out: None comes back in their place."""
    lib, torch = _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight is a matrix (outputs, inputs)")
    inputs, outputs = x.shape[-1], weight.shape[0]
    _like(weight, x, "weight", torch, (outputs, inputs))
    shape = x.shape[:-1] + (outputs,)
    _like(dy, x, "dy", torch, shape)
    if act:
        if z is None:
            raise ValueError(f"the gradient of {activation} needs z")
        _like(z, x, "z", torch, shape)
    device = x.device
    with _On(torch, device):
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need[0] else None
        dweight = torch.empty((outputs, inputs), dtype=x.dtype, device=device) if need[1] else None
        dbias = torch.empty(outputs, dtype=x.dtype, device=device) if need[2] else None
        rows = _count(shape[:-1])
        x, px, ldx = _rows(x)
        weight, pw, ldw = _rows(weight)
        dy, pd, ldd = _rows(dy)
        pz, ldz = None, 0
        if act:
            z, pz, ldz = _rows(z)
        size = lib.mace_dense_backward_workspace(code, rows, inputs, outputs, pd, ldd, px, ldx, pw, ldw, act)
        ws = _workspace(torch, lib, size, device)
        if lib.mace_dense_backward(code, rows, inputs, outputs, pd, ldd, px, ldx, pw, ldw, act, pz, ldz, _address(dx),
                                   inputs, _address(dweight), inputs, _address(dbias), _address(ws), size,
                                   _stream(torch, device)):
            raise RuntimeError(_error(lib))
    return dx, dweight, dbias


def _parameters(x, gamma, beta, torch):
    width = x.shape[-1]
    if gamma is not None:
        _like(gamma, x, "gamma", torch, (width,))
    if beta is not None:
        _like(beta, x, "beta", torch, (width,))
    return width, _flat(gamma), _flat(beta)


def layer_norm(x, gamma=None, beta=None, eps=1e-5, activation=None, keep=False):
    """``activation((x - mean) rstd gamma + beta)`` over the last index, with the biased variance.
    ``keep=True`` returns (y, mean, rstd), the statistics float32 of shape x.shape[:-1]."""
    lib, torch = _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    width, gamma, beta = _parameters(x, gamma, beta, torch)
    device, shape = x.device, x.shape
    with _On(torch, device):
        y = torch.empty(shape, dtype=x.dtype, device=device)
        mean = torch.empty(shape[:-1], dtype=torch.float32, device=device) if keep else None
        rstd = torch.empty(shape[:-1], dtype=torch.float32, device=device) if keep else None
        x, px, ldx = _rows(x) if x.dim() > 1 else _rows(x[None])
        if lib.mace_layer_norm(code, _count(shape[:-1]), width, px, ldx, _address(gamma), _address(beta), eps, act,
                               y.data_ptr(), width, _address(mean), _address(rstd), _stream(torch, device)):
            raise RuntimeError(_error(lib))
    return (y, mean, rstd) if keep else y


def layer_norm_backward(dy, x, mean, rstd, gamma=None, beta=None, activation=None, need=(True, True, True)):
    """(dx, dgamma, dbeta) of ``layer_norm`` for the output gradient dy, with the statistics that
    ``layer_norm(..., keep=True)`` gave and the gamma, beta and activation of that call (beta is
    read only with an activation).  ``need`` leaves gradients out: None comes back in their
    place."""
    lib, torch = _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    width, gamma, beta = _parameters(x, gamma, beta, torch)
    device, shape = x.device, x.shape
    _like(dy, x, "dy", torch, shape)
    _like(mean, x, "mean", torch, shape[:-1], torch.float32)
    _like(rstd, x, "rstd", torch, shape[:-1], torch.float32)
    with _On(torch, device):
        dx = torch.empty(shape, dtype=x.dtype, device=device) if need[0] else None
        dgamma = torch.empty(width, dtype=x.dtype, device=device) if need[1] else None
        dbeta = torch.empty(width, dtype=x.dtype, device=device) if need[2] else None
        rows = _count(shape[:-1])
        x, px, ldx = _rows(x) if x.dim() > 1 else _rows(x[None])
        dy, pd, ldd = _rows(dy) if dy.dim() > 1 else _rows(dy[None])
        mean, rstd = _flat(mean), _flat(rstd)
        size = lib.mace_layer_norm_backward_workspace(code, rows, width) if need[1] or need[2] else 0
        ws = _workspace(torch, lib, size, device)
        if lib.mace_layer_norm_backward(code, rows, width, pd, ldd, px, ldx, mean.data_ptr(), rstd.data_ptr(),
                                        _address(gamma), _address(beta), act, _address(dx), width, _address(dgamma),
                                        _address(dbeta), _address(ws), size, _stream(torch, device)):
            raise RuntimeError(_error(lib))
    return dx, dgamma, dbeta
