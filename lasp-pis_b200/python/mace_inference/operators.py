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
no autograd graph: the backward calls give the gradients.  Where autograd is on and an argument of
a forward call requires a gradient, a UserWarning says so (torch.no_grad() or detach() around such
calls keeps it away).  Wrong arguments raise ValueError (or TypeError); what the library itself
refuses (an empty last index, a negative eps) and a failed call raise RuntimeError.
"""
from __future__ import annotations

import ctypes as ct
import math
import warnings

from .native import _error, load

ACTIVATIONS = {None: 0, "none": 0, "silu": 1, "gelu": 2, "relu": 3}

_bound = None   # (library, torch, the current stream's handle of a device index)
_types = {}     # torch type -> element type of the C interface
_sizes = {}     # workspace bytes by what they depend on: shapes, row distances, 16-byte alignment


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
        # The stream's handle without a stream object (2 us a call), where torch has it.
        stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: torch.cuda.current_stream(index).cuda_stream)
        _bound = lib, torch, stream
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


def _like(t, name, torch, shape, dtype, device):
    """Checks a tensor that goes with others; returns it."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a torch tensor, not {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    return t


def _warn_of_autograd(name):
    warnings.warn(f"{name} records no autograd graph, and an argument requires a gradient: its result has none "
                  f"(the gradients come from {name}_backward)", UserWarning, stacklevel=3)


def _rows(t):
    """`t` as rows with a contiguous last index: (tensor that keeps the memory alive, address, row distance)."""
    if t.dim() != 2:
        if t.is_contiguous():
            return t, t.data_ptr(), t.shape[-1]
        t = t.reshape(-1, t.shape[-1])  # a view where the leading indices collapse
    rows, width = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or width == 1) and (s0 >= width or rows <= 1):
        return t, t.data_ptr(), s0 if s0 > width else width
    t = t.contiguous()
    return t, t.data_ptr(), width


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _address(t):
    return None if t is None else t.data_ptr()


def _on(torch, device, call, *args, **kwargs):
    """call(...) with `device` current."""
    with torch.cuda.device(device):
        return call(*args, **kwargs)


def _size(lib, key, call, *args):
    """Workspace bytes, asked once for each `key`."""
    size = _sizes.get(key)
    if size is None:
        size = call(*args)
        if size < 0:
            raise RuntimeError(_error(lib))
        if len(_sizes) >= 4096:
            _sizes.clear()
        _sizes[key] = size
    return size


def _workspace(x, code, size):
    """`size` bytes (a multiple of 16) beside x."""
    return x.new_empty(size >> (1 if code else 2)) if size else None


def _new_like(t, torch):
    """A new contiguous tensor like t (empty_like costs half of new_empty, but keeps other layouts)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def dense(x, weight, bias=None, activation=None, residual=None, keep=False):
    """``activation(x weight^T + bias) + residual`` for x (..., inputs), weight (outputs, inputs),
    bias (outputs,) and residual (..., outputs).  ``keep=True`` returns (y, z) with
    z = x weight^T + bias, which ``dense_backward`` takes where there is an activation."""
    lib, torch, stream = _bound or _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    dtype, device, shape = x.dtype, x.device, x.shape
    if torch.cuda.current_device() != device.index:
        return _on(torch, device, dense, x, weight, bias, activation, residual, keep)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight is a matrix (outputs, inputs)")
    outputs, inputs = weight.shape[0], shape[-1]
    _like(weight, "weight", torch, (outputs, inputs), dtype, device)
    shape = (*shape[:-1], outputs)
    rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if bias is not None:
        bias = _flat(_like(bias, "bias", torch, (outputs,), dtype, device))
    pr, ldr = None, 0
    if residual is not None:
        residual, pr, ldr = _rows(_like(residual, "residual", torch, shape, dtype, device))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        _warn_of_autograd("dense")
    x, px, ldx = _rows(x)
    weight, pw, ldw = _rows(weight)
    y = x.new_empty(shape)
    z = torch.empty_like(y) if keep else None
    size = _size(lib, (0, code, rows, inputs, outputs, px & 15, ldx, pw & 15, ldw, device.index),
                 lib.mace_dense_workspace, code, rows, inputs, outputs, px, ldx, pw, ldw)
    ws = _workspace(x, code, size)
    if lib.mace_dense(code, rows, inputs, outputs, px, ldx, pw, ldw, _address(bias), act, pr, ldr, y.data_ptr(), outputs,
                      _address(z), outputs, _address(ws), size, stream(device.index)):
        raise RuntimeError(_error(lib))
    return (y, z) if keep else y


def dense_backward(dy, x, weight, activation=None, z=None, need=(True, True, True)):
    """(dx, dweight, dbias) of ``dense`` for the output gradient dy (..., outputs); z is what
    ``dense(..., keep=True)`` gave (not needed without an activation).  The residual's gradient
    is dy itself.  ``need`` leaves gradients out: None comes back in their place."""
    lib, torch, stream = _bound or _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    dtype, device, shape = x.dtype, x.device, x.shape
    if torch.cuda.current_device() != device.index:
        return _on(torch, device, dense_backward, dy, x, weight, activation, z, need)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight is a matrix (outputs, inputs)")
    outputs, inputs = weight.shape[0], shape[-1]
    _like(weight, "weight", torch, (outputs, inputs), dtype, device)
    out = (*shape[:-1], outputs)
    rows = out[0] if len(out) == 2 else math.prod(out[:-1])
    dy, pd, ldd = _rows(_like(dy, "dy", torch, out, dtype, device))
    pz, ldz = None, 0
    if act:
        if z is None:
            raise ValueError(f"the gradient of {activation} needs z")
        z, pz, ldz = _rows(_like(z, "z", torch, out, dtype, device))
    x, px, ldx = _rows(x)
    weight, pw, ldw = _rows(weight)
    dx = x.new_empty(shape) if need[0] else None
    dweight = _new_like(weight, torch) if need[1] else None
    dbias = x.new_empty(outputs) if need[2] else None
    size = _size(lib, (1, code, rows, inputs, outputs, pd & 15, ldd, px & 15, ldx, pw & 15, ldw, act, device.index),
                 lib.mace_dense_backward_workspace, code, rows, inputs, outputs, pd, ldd, px, ldx, pw, ldw, act)
    ws = _workspace(x, code, size)
    if lib.mace_dense_backward(code, rows, inputs, outputs, pd, ldd, px, ldx, pw, ldw, act, pz, ldz, _address(dx), inputs,
                               _address(dweight), inputs, _address(dbias), _address(ws), size, stream(device.index)):
        raise RuntimeError(_error(lib))
    return dx, dweight, dbias


def layer_norm(x, gamma=None, beta=None, eps=1e-5, activation=None, keep=False):
    """``activation((x - mean) rstd gamma + beta)`` over the last index, with the biased variance.
    ``keep=True`` returns (y, mean, rstd), the statistics float32 of shape x.shape[:-1]."""
    lib, torch, stream = _bound or _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    dtype, device, shape = x.dtype, x.device, x.shape
    if torch.cuda.current_device() != device.index:
        return _on(torch, device, layer_norm, x, gamma, beta, eps, activation, keep)
    width = shape[-1]
    rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if gamma is not None:
        gamma = _flat(_like(gamma, "gamma", torch, (width,), dtype, device))
    if beta is not None:
        beta = _flat(_like(beta, "beta", torch, (width,), dtype, device))
    if torch.is_grad_enabled() and (x.requires_grad or (gamma is not None and gamma.requires_grad)
                                    or (beta is not None and beta.requires_grad)):
        _warn_of_autograd("layer_norm")
    x, px, ldx = _rows(x)
    y = _new_like(x, torch) if x.dim() == len(shape) else x.new_empty(shape)
    mean = rstd = None
    if keep:
        mean = x.new_empty(shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    if lib.mace_layer_norm(code, rows, width, px, ldx, _address(gamma), _address(beta), eps, act, y.data_ptr(), width,
                           _address(mean), _address(rstd), stream(device.index)):
        raise RuntimeError(_error(lib))
    return (y, mean, rstd) if keep else y


def layer_norm_backward(dy, x, mean, rstd, gamma=None, beta=None, activation=None, need=(True, True, True)):
    """(dx, dgamma, dbeta) of ``layer_norm`` for the output gradient dy, with the statistics that
    ``layer_norm(..., keep=True)`` gave and the gamma, beta and activation of that call (beta is
    read only with an activation).  ``need`` leaves gradients out: None comes back in their
    place."""
    lib, torch, stream = _bound or _library()
    act = _activation(activation)
    code = _type(x, "x", torch)
    dtype, device, shape = x.dtype, x.device, x.shape
    if torch.cuda.current_device() != device.index:
        return _on(torch, device, layer_norm_backward, dy, x, mean, rstd, gamma, beta, activation, need)
    width = shape[-1]
    rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if gamma is not None:
        gamma = _flat(_like(gamma, "gamma", torch, (width,), dtype, device))
    if beta is not None:
        beta = _flat(_like(beta, "beta", torch, (width,), dtype, device))
    dy, pd, ldd = _rows(_like(dy, "dy", torch, shape, dtype, device))
    mean = _flat(_like(mean, "mean", torch, shape[:-1], torch.float32, device))
    rstd = _flat(_like(rstd, "rstd", torch, shape[:-1], torch.float32, device))
    x, px, ldx = _rows(x)
    dx = None
    if need[0]:
        dx = _new_like(x, torch) if x.dim() == len(shape) else x.new_empty(shape)
    dgamma = dbeta = None
    if need[1]:
        dgamma = x.new_empty(width) if gamma is None else torch.empty_like(gamma)
    if need[2]:
        dbeta = x.new_empty(width) if dgamma is None else torch.empty_like(dgamma)
    size = 0
    if need[1] or need[2]:
        size = _size(lib, (2, code, rows, width, device.index), lib.mace_layer_norm_backward_workspace, code, rows, width)
    ws = _workspace(x, code, size)
    if lib.mace_layer_norm_backward(code, rows, width, pd, ldd, px, ldx, mean.data_ptr(), rstd.data_ptr(),
                                    _address(gamma), _address(beta), act, _address(dx), width, _address(dgamma),
                                    _address(dbeta), _address(ws), size, stream(device.index)):
        raise RuntimeError(_error(lib))
    return dx, dgamma, dbeta
