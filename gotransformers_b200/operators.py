"""Operators without a handle over libgtmoe.so, for training a block: layer
norm, dropout with the residual, and matrix products of rows grouped by
expert, each with its gradients (the last section of include/gtmoe.h).

Arguments are CUDA tensors of one device, contiguous, float64, float32 or
bfloat16; a call runs on that device's current torch stream, waits for
nothing and may be captured into a CUDA graph.  Results carry no autograd
graph: the gradients are the functions named so; a tensor that a call was given
to write into counts as changed for autograd.  Misuse raises
``ValueError``, what the library refuses ``GtmoeError``."""
from __future__ import annotations

import ctypes
import numbers

from . import _lib
from ._lib import DTYPE_BF16, DTYPE_F32, DTYPE_F64, check

# torch, the library and the type codes, once an operator is first called
# (importing this package needs neither)
torch = None
_L = None
_CODES: dict = {}
_WORD = (1 << 64) - 1


def _load():
    global torch, _L
    if torch is None:
        import torch as torch_module

        _CODES.update({torch_module.float64: DTYPE_F64, torch_module.float32: DTYPE_F32,
                       torch_module.bfloat16: DTYPE_BF16})
        torch = torch_module
    if _L is None:
        _L = _lib.lib()


def _code(dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"values must be float64, float32 or bfloat16, got {dtype}")
    return code


def _refuse(name: str, a, shape, dtype, device):
    if not hasattr(a, "data_ptr"):
        raise ValueError(f"{name} must be a CUDA tensor, got {type(a).__name__}")
    if not a.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, got {a.device}")
    if not a.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if a.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(a.shape)}")
    if a.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {a.dtype}")
    raise ValueError(f"{name} is on {a.device} but the rows are on cuda:{device}")


def _tensor(name: str, a, shape, dtype, device: int):
    """The checks an argument goes through; returns its address."""
    try:
        if (a.is_cuda and a.dtype is dtype and a.shape == shape and a.get_device() == device and a.is_contiguous()):
            return a.data_ptr()
    except AttributeError:
        pass
    return _refuse(name, a, shape, dtype, device)


def _rows(name: str, a):
    """The checks of the tensor that the others are held to; its address and device."""
    address = _values(name, a)
    if a.ndim != 2:
        raise ValueError(f"{name} must be rows x width, got {a.ndim} dimensions")
    return address


def _values(name: str, a):
    """_rows for a tensor of any shape."""
    if torch is None or _L is None:
        _load()
    if not isinstance(a, torch.Tensor) or not a.is_cuda or not a.is_contiguous():
        _refuse(name, a, getattr(a, "shape", None), getattr(a, "dtype", None), None)
    return a.data_ptr(), a.get_device()


def _stream(device: int) -> int:
    """The device's current torch stream."""
    return torch._C._cuda_getCurrentRawStream(device)


def _number(name: str, v):
    if type(v) is float:
        return v
    try:
        if not isinstance(v, (str, bytes, bytearray)):  # float() would read these
            return float(v)
    except (TypeError, ValueError):
        pass
    raise ValueError(f"{name} must be a number, got {type(v).__name__}")


def _generator(seed, stream, offset=0):
    """The generator's arguments as the library takes them: seed and stream
    modulo 2^64, an offset that it would see only a part of refused."""
    if not type(seed) is type(stream) is type(offset) is int:
        for name, v in (("seed", seed), ("stream", stream), ("offset", offset)):
            if not isinstance(v, numbers.Integral):
                raise ValueError(f"{name} must be a whole number, got {type(v).__name__}")
        seed, stream, offset = int(seed), int(stream), int(offset)
    if not -(1 << 63) <= offset < 1 << 63:
        raise ValueError(f"offset must be below 2^63, got {offset}")
    return [seed & _WORD, stream & _WORD, offset]


def _wrote(*given):
    """The library writes through addresses: tells autograd that the caller's
    tensors have changed, so that it refuses to use what it had saved of them."""
    for t in given:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _dtype(a):
    """a's dtype; None for what is no tensor, which the checks then refuse."""
    return getattr(a, "dtype", None)


def _stats_dtype(x):
    return torch.float64 if x.dtype is torch.float64 else torch.float32


def layer_norm(x, weight=None, bias=None, epsilon: float = 1e-6, out=None):
    """(x - mean) * rstd * weight + bias over each row of x (rows x width).
    weight and bias have x's dtype, or float32 beside bfloat16 rows.  Returns
    (y, mean, rstd); the statistics (float32, float64 for float64 rows) are
    what layer_norm_backward takes.  `out` may be x."""
    px, dev = _rows("x", x)
    shape, dtype = x.shape, x.dtype
    rows, width = shape
    wdt = _dtype(weight) if weight is not None else _dtype(bias) if bias is not None else dtype
    if weight is not None and bias is not None and wdt != _dtype(bias):
        raise ValueError(f"weight and bias must be tensors of one dtype, got {wdt} and {_dtype(bias)}")
    pw = None if weight is None else _tensor("weight", weight, (width,), wdt, dev)
    pb = None if bias is None else _tensor("bias", bias, (width,), wdt, dev)
    code, wcode = _code(dtype), _code(wdt)
    given = out
    if out is None:
        out = torch.empty_like(x)
        po = out.data_ptr()
    else:
        po = _tensor("out", out, shape, dtype, dev)
    mean = torch.empty(rows, dtype=_stats_dtype(x), device=x.device)
    rstd = torch.empty_like(mean)
    check(_L.gtmoe_layer_norm(px, code, rows, width, pw, pb, wcode, _number("epsilon", epsilon), po, mean.data_ptr(),
                              rstd.data_ptr(), _stream(dev)))
    if given is not None:
        _wrote(given)
    return out, mean, rstd


def layer_norm_backward(output_gradients, x, mean, rstd, weight=None, residual_gradients=None, input_gradients=None,
                        weight_grad=None, bias_grad=None, want_parameters: bool = True):
    """The gradients of layer_norm at x with the statistics it returned:
    (input gradients, weight gradients, bias gradients).  residual_gradients
    (rows x width) are added to the input gradients.  weight_grad and
    bias_grad, where given, have theirs added; else new tensors of the
    weight's dtype (without a weight: float32, float64 for float64 rows) are
    returned, or None with want_parameters=False.  `input_gradients` may be
    any of the rows x width inputs."""
    g = output_gradients
    pg, dev = _rows("output_gradients", g)
    shape, dtype = g.shape, g.dtype
    rows, width = shape
    code = _code(dtype)
    px = _tensor("x", x, shape, dtype, dev)
    sdt = _stats_dtype(g)
    pm, pr = _tensor("mean", mean, (rows,), sdt, dev), _tensor("rstd", rstd, (rows,), sdt, dev)
    wdt = _dtype(weight) if weight is not None else _dtype(weight_grad) if weight_grad is not None else sdt
    pw = None if weight is None else _tensor("weight", weight, (width,), wdt, dev)
    pres = None
    if residual_gradients is not None:
        pres = _tensor("residual_gradients", residual_gradients, shape, dtype, dev)
    given = input_gradients
    if input_gradients is None:
        input_gradients = torch.empty_like(g)
        pdx = input_gradients.data_ptr()
    else:
        pdx = _tensor("input_gradients", input_gradients, shape, dtype, dev)
    if (weight_grad is None) != (bias_grad is None):
        raise ValueError("weight_grad and bias_grad are given together")
    accumulate = weight_grad is not None
    wcode = _code(wdt)
    pdw = pdb = pwork = None
    nbytes = 0
    if accumulate or want_parameters:
        if not accumulate:
            weight_grad = torch.empty(width, dtype=wdt, device=g.device)
            bias_grad = torch.empty_like(weight_grad)
            pdw, pdb = weight_grad.data_ptr(), bias_grad.data_ptr()
        else:
            pdw = _tensor("weight_grad", weight_grad, (width,), wdt, dev)
            pdb = _tensor("bias_grad", bias_grad, (width,), wdt, dev)
        need = ctypes.c_int64(0)
        check(_L.gtmoe_layer_norm_workspace(code, rows, width, ctypes.byref(need)))
        nbytes = need.value
        work = torch.empty(nbytes, dtype=torch.uint8, device=g.device)
        pwork = work.data_ptr()
    check(_L.gtmoe_layer_norm_backward(pg, px, code, rows, width, pw, wcode, pm, pr, pres, pdx, pdw, pdb,
                                       int(accumulate), pwork, nbytes, _stream(dev)))
    if given is not None or accumulate:
        _wrote(given, *((weight_grad, bias_grad) if accumulate else ()))
    return input_gradients, weight_grad, bias_grad


def dropout(x, rate: float, seed: int, stream: int = 0, offset: int = 0, residual=None, out=None):
    """residual + x * keep / (1 - rate) for a tensor of any shape.  Whether
    element i (in memory order) is kept depends on (seed, stream, offset + i)
    alone, seed and stream modulo 2^64, so dropout_backward makes the same
    decisions again.  `out` may be x or residual."""
    px, dev = _values("x", x)
    shape, dtype = x.shape, x.dtype
    pr = None if residual is None else _tensor("residual", residual, shape, dtype, dev)
    code = _code(dtype)
    given = out
    if out is None:
        out = torch.empty_like(x)
        po = out.data_ptr()
    else:
        po = _tensor("out", out, shape, dtype, dev)
    check(_L.gtmoe_dropout(px, pr, code, x.numel(), _number("rate", rate), *_generator(seed, stream, offset), po,
                           _stream(dev)))
    if given is not None:
        _wrote(given)
    return out


def dropout_backward(output_gradients, rate: float, seed: int, stream: int = 0, offset: int = 0,
                     input_gradients=None):
    """output_gradients * keep / (1 - rate), with dropout's decisions; the
    residual's gradients are the output gradients.  `input_gradients` may be
    output_gradients."""
    g = output_gradients
    pg, dev = _values("output_gradients", g)
    code = _code(g.dtype)
    given = input_gradients
    if input_gradients is None:
        input_gradients = torch.empty_like(g)
        pdx = input_gradients.data_ptr()
    else:
        pdx = _tensor("input_gradients", input_gradients, g.shape, g.dtype, dev)
    check(_L.gtmoe_dropout_backward(pg, code, g.numel(), _number("rate", rate), *_generator(seed, stream, offset),
                                    pdx, _stream(dev)))
    if given is not None:
        _wrote(given)
    return input_gradients


def _weights(weights, like, like_name: str, axis: int, dev: int):
    """The weights' address, groups, outputs and inputs."""
    shape = getattr(weights, "shape", ())
    if len(shape) != 3 or shape[axis] != like.shape[1]:
        raise ValueError(f"weights must be groups x outputs x inputs and fit {like_name}'s {like.shape[1]} columns, "
                         f"got {tuple(shape)}")
    return _tensor("weights", weights, shape, like.dtype, dev), *shape


def grouped_product(x, weights, counts, out=None):
    """x[r] @ weights[g].T for the rows r of each group g: x (rows x inputs)
    holds counts[0] rows of group 0, then counts[1] of group 1, ... (counts an
    int64 CUDA tensor); weights are groups x outputs x inputs.  Rows after the
    last group's are not written."""
    px, dev = _rows("x", x)
    pw, groups, outputs, inputs = _weights(weights, x, "x", 2, dev)
    rows, dtype = x.shape[0], x.dtype
    pc = _tensor("counts", counts, (groups,), torch.int64, dev)
    code = _code(dtype)
    given = out
    if out is None:
        out = torch.empty((rows, outputs), dtype=dtype, device=x.device)
        po = out.data_ptr()
    else:
        po = _tensor("out", out, (rows, outputs), dtype, dev)
    check(_L.gtmoe_grouped_product(px, pw, code, rows, inputs, outputs, groups, pc, po, _stream(dev)))
    if given is not None:
        _wrote(given)
    return out


def grouped_product_input_gradients(output_gradients, weights, counts, input_gradients=None):
    """output_gradients[r] @ weights[g] for the rows r of each group g."""
    g = output_gradients
    pg, dev = _rows("output_gradients", g)
    pw, groups, outputs, inputs = _weights(weights, g, "output_gradients", 1, dev)
    rows, dtype = g.shape[0], g.dtype
    pc = _tensor("counts", counts, (groups,), torch.int64, dev)
    code = _code(dtype)
    given = input_gradients
    if input_gradients is None:
        input_gradients = torch.empty((rows, inputs), dtype=dtype, device=g.device)
        pdx = input_gradients.data_ptr()
    else:
        pdx = _tensor("input_gradients", input_gradients, (rows, inputs), dtype, dev)
    check(_L.gtmoe_grouped_product_input_grad(pg, pw, code, rows, inputs, outputs, groups, pc, pdx, _stream(dev)))
    if given is not None:
        _wrote(given)
    return input_gradients


def grouped_product_weight_gradients(output_gradients, x, counts, weight_grad=None, dtype=None):
    """The sum over group g's rows of output_gradients[r].T @ x[r], groups x
    outputs x inputs.  weight_grad, where given, has them added; else a new
    tensor of `dtype` (x's dtype, or float32 beside bfloat16) is returned."""
    g = output_gradients
    pg, dev = _rows("output_gradients", g)
    px, _ = _rows("x", x)
    rows, outputs = g.shape
    inputs = x.shape[1]
    _tensor("x", x, (rows, inputs), g.dtype, dev)
    if getattr(counts, "ndim", None) != 1:
        raise ValueError("counts must be one number per group")
    groups = counts.shape[0]
    pc = _tensor("counts", counts, (groups,), torch.int64, dev)
    code = _code(g.dtype)
    accumulate = weight_grad is not None
    if not accumulate:
        weight_grad = torch.empty((groups, outputs, inputs), dtype=dtype or g.dtype, device=g.device)
    wdt = _dtype(weight_grad)
    if dtype is not None and wdt != dtype:
        raise ValueError(f"weight_grad is {wdt} but dtype {dtype}")
    pdw = _tensor("weight_grad", weight_grad, (groups, outputs, inputs), wdt, dev)
    wcode = _code(wdt)
    need, pwork = ctypes.c_int64(0), None
    check(_L.gtmoe_grouped_product_workspace(code, rows, inputs, outputs, groups, ctypes.byref(need)))
    if need.value:
        work = torch.empty(need.value, dtype=torch.uint8, device=g.device)
        pwork = work.data_ptr()
    check(_L.gtmoe_grouped_product_weight_grad(pg, px, code, rows, inputs, outputs, groups, pc, pdw, wcode,
                                               int(accumulate), pwork, need.value, _stream(dev)))
    if accumulate:
        _wrote(weight_grad)
    return weight_grad


def check_operators(device: int = 0):
    """Waits for the device and raises GtmoeError if an operator since the
    last check was given impossible counts (EINVAL) or gave up waiting
    (ETIMEOUT)."""
    check(_lib.lib().gtmoe_operators_check(device))
