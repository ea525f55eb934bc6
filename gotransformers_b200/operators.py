"""Operators without a handle over libgtmoe.so, for training a block: layer
norm, dropout with the residual, and matrix products of rows grouped by
expert, each with its gradients (the last section of include/gtmoe.h).

Arguments are CUDA tensors of one device, contiguous, float64, float32 or
bfloat16; a call runs on that device's current torch stream, waits for
nothing and may be captured into a CUDA graph.  Misuse raises ``ValueError``,
what the library refuses ``GtmoeError``."""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import DTYPE_BF16, DTYPE_F32, DTYPE_F64, check

_CODES: dict = {}


def _code(dtype) -> int:
    if not _CODES:
        import torch

        _CODES.update({torch.float64: DTYPE_F64, torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16})
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"values must be float64, float32 or bfloat16, got {dtype}")
    return code


def _tensor(name: str, a, shape=None, dtype=None, like=None):
    """The checks every argument goes through; returns its address."""
    if not hasattr(a, "data_ptr"):
        raise ValueError(f"{name} must be a CUDA tensor, got {type(a).__name__}")
    if not a.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, got {a.device}")
    if not a.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and a.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(a.shape)}")
    if dtype is not None and a.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {a.dtype}")
    if like is not None and a.device != like.device:
        raise ValueError(f"{name} is on {a.device} but the rows are on {like.device}")
    return a.data_ptr()


def _optional(name: str, a, shape=None, dtype=None, like=None):
    return None if a is None else _tensor(name, a, shape, dtype, like)


def _stream(a):
    import torch

    return torch.cuda.current_stream(a.device).cuda_stream


def _rows(name: str, a):
    if getattr(a, "ndim", None) != 2:
        raise ValueError(f"{name} must be rows x width, got {getattr(a, 'ndim', None)} dimensions")
    return _tensor(name, a)


def _stats_dtype(x):
    import torch

    return torch.float64 if x.dtype == torch.float64 else torch.float32


def layer_norm(x, weight=None, bias=None, epsilon: float = 1e-6, out=None):
    """(x - mean) * rstd * weight + bias over each row of x (rows x width).
    weight and bias have x's dtype, or float32 beside bfloat16 rows.  Returns
    (y, mean, rstd); the statistics (float32, float64 for float64 rows) are
    what layer_norm_backward takes.  `out` may be x."""
    import torch

    px = _rows("x", x)
    rows, width = x.shape
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    pw, pb = _optional("weight", weight, (width,), None, x), _optional("bias", bias, (width,), None, x)
    wdt = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    if out is None:
        out = torch.empty_like(x)
    po = _tensor("out", out, x.shape, x.dtype, x)
    sdt = _stats_dtype(x)
    mean, rstd = torch.empty(rows, dtype=sdt, device=x.device), torch.empty(rows, dtype=sdt, device=x.device)
    check(_lib.lib().gtmoe_layer_norm(px, _code(x.dtype), rows, width, pw, pb, _code(wdt), epsilon, po,
                                      mean.data_ptr(), rstd.data_ptr(), _stream(x)))
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
    import torch

    g = output_gradients
    pg = _rows("output_gradients", g)
    rows, width = g.shape
    px = _tensor("x", x, g.shape, g.dtype, g)
    sdt = _stats_dtype(g)
    pm, pr = _tensor("mean", mean, (rows,), sdt, g), _tensor("rstd", rstd, (rows,), sdt, g)
    pw = _optional("weight", weight, (width,), None, g)
    pres = _optional("residual_gradients", residual_gradients, g.shape, g.dtype, g)
    wdt = weight.dtype if weight is not None else sdt
    if input_gradients is None:
        input_gradients = torch.empty_like(g)
    pdx = _tensor("input_gradients", input_gradients, g.shape, g.dtype, g)
    if (weight_grad is None) != (bias_grad is None):
        raise ValueError("weight_grad and bias_grad are given together")
    accumulate = weight_grad is not None
    pdw = pdb = work = None
    nbytes = ctypes.c_int64(0)
    if accumulate or want_parameters:
        if not accumulate:
            weight_grad = torch.empty(width, dtype=wdt, device=g.device)
            bias_grad = torch.empty(width, dtype=wdt, device=g.device)
        pdw = _tensor("weight_grad", weight_grad, (width,), wdt, g)
        pdb = _tensor("bias_grad", bias_grad, (width,), wdt, g)
        check(_lib.lib().gtmoe_layer_norm_workspace(_code(g.dtype), rows, width, ctypes.byref(nbytes)))
        work = torch.empty(nbytes.value, dtype=torch.uint8, device=g.device)
    check(_lib.lib().gtmoe_layer_norm_backward(pg, px, _code(g.dtype), rows, width, pw, _code(wdt), pm, pr, pres, pdx,
                                               pdw, pdb, int(accumulate), work.data_ptr() if work is not None else None,
                                               nbytes.value, _stream(g)))
    return input_gradients, weight_grad, bias_grad


def dropout(x, rate: float, seed: int, stream: int = 0, offset: int = 0, residual=None, out=None):
    """residual + x * keep / (1 - rate) for a tensor of any shape.  Whether
    element i (in memory order) is kept depends on (seed, stream, offset + i)
    alone, so dropout_backward makes the same decisions again.  `out` may be
    x or residual."""
    import torch

    px = _tensor("x", x)
    pr = _optional("residual", residual, x.shape, x.dtype, x)
    if out is None:
        out = torch.empty_like(x)
    po = _tensor("out", out, x.shape, x.dtype, x)
    check(_lib.lib().gtmoe_dropout(px, pr, _code(x.dtype), x.numel(), rate, seed, stream, offset, po, _stream(x)))
    return out


def dropout_backward(output_gradients, rate: float, seed: int, stream: int = 0, offset: int = 0,
                     input_gradients=None):
    """output_gradients * keep / (1 - rate), with dropout's decisions; the
    residual's gradients are the output gradients.  `input_gradients` may be
    output_gradients."""
    import torch

    g = output_gradients
    pg = _tensor("output_gradients", g)
    if input_gradients is None:
        input_gradients = torch.empty_like(g)
    pdx = _tensor("input_gradients", input_gradients, g.shape, g.dtype, g)
    check(_lib.lib().gtmoe_dropout_backward(pg, _code(g.dtype), g.numel(), rate, seed, stream, offset, pdx,
                                            _stream(g)))
    return input_gradients


def _weights(weights, like, like_name: str, axis: int):
    pw = _tensor("weights", weights, None, like.dtype, like)
    if weights.ndim != 3 or weights.shape[axis] != like.shape[1]:
        raise ValueError(f"weights must be groups x outputs x inputs and fit {like_name}'s {like.shape[1]} columns, "
                         f"got {tuple(weights.shape)}")
    return pw


def _counts(counts, groups, like):
    import torch

    return _tensor("counts", counts, (groups,), torch.int64, like)


def grouped_product(x, weights, counts, out=None):
    """x[r] @ weights[g].T for the rows r of each group g: x (rows x inputs)
    holds counts[0] rows of group 0, then counts[1] of group 1, ... (counts an
    int64 CUDA tensor); weights are groups x outputs x inputs.  Rows after the
    last group's are not written."""
    import torch

    px = _rows("x", x)
    pw = _weights(weights, x, "x", 2)
    groups, outputs, inputs = weights.shape
    rows = x.shape[0]
    pc = _counts(counts, groups, x)
    if out is None:
        out = torch.empty((rows, outputs), dtype=x.dtype, device=x.device)
    po = _tensor("out", out, (rows, outputs), x.dtype, x)
    check(_lib.lib().gtmoe_grouped_product(px, pw, _code(x.dtype), rows, inputs, outputs, groups, pc, po, _stream(x)))
    return out


def grouped_product_input_gradients(output_gradients, weights, counts, input_gradients=None):
    """output_gradients[r] @ weights[g] for the rows r of each group g."""
    import torch

    g = output_gradients
    pg = _rows("output_gradients", g)
    pw = _weights(weights, g, "output_gradients", 1)
    groups, outputs, inputs = weights.shape
    rows = g.shape[0]
    pc = _counts(counts, groups, g)
    if input_gradients is None:
        input_gradients = torch.empty((rows, inputs), dtype=g.dtype, device=g.device)
    pdx = _tensor("input_gradients", input_gradients, (rows, inputs), g.dtype, g)
    check(_lib.lib().gtmoe_grouped_product_input_grad(pg, pw, _code(g.dtype), rows, inputs, outputs, groups, pc, pdx,
                                                      _stream(g)))
    return input_gradients


def grouped_product_weight_gradients(output_gradients, x, counts, weight_grad=None, dtype=None):
    """The sum over group g's rows of output_gradients[r].T @ x[r], groups x
    outputs x inputs.  weight_grad, where given, has them added; else a new
    tensor of `dtype` (x's dtype, or float32 beside bfloat16) is returned."""
    import torch

    g = output_gradients
    pg = _rows("output_gradients", g)
    px = _rows("x", x)
    _tensor("x", x, None, g.dtype, g)
    if x.shape[0] != g.shape[0]:
        raise ValueError(f"x has {x.shape[0]} rows but output_gradients {g.shape[0]}")
    rows, outputs, inputs = g.shape[0], g.shape[1], x.shape[1]
    if getattr(counts, "ndim", None) != 1:
        raise ValueError("counts must be one number per group")
    groups = counts.shape[0]
    pc = _counts(counts, groups, g)
    accumulate = weight_grad is not None
    if not accumulate:
        weight_grad = torch.empty((groups, outputs, inputs), dtype=dtype or g.dtype, device=g.device)
    elif dtype is not None and weight_grad.dtype != dtype:
        raise ValueError(f"weight_grad is {weight_grad.dtype} but dtype {dtype}")
    pdw = _tensor("weight_grad", weight_grad, (groups, outputs, inputs), None, g)
    nbytes, work = ctypes.c_int64(0), None
    check(_lib.lib().gtmoe_grouped_product_workspace(_code(g.dtype), rows, inputs, outputs, groups,
                                                     ctypes.byref(nbytes)))
    if nbytes.value:
        work = torch.empty(nbytes.value, dtype=torch.uint8, device=g.device)
    check(_lib.lib().gtmoe_grouped_product_weight_grad(pg, px, _code(g.dtype), rows, inputs, outputs, groups, pc, pdw,
                                                       _code(weight_grad.dtype), int(accumulate),
                                                       work.data_ptr() if work is not None else None, nbytes.value,
                                                       _stream(g)))
    return weight_grad


def check_operators(device: int = 0):
    """Waits for the device and raises GtmoeError if a grouped product since
    the last check was given impossible counts (EINVAL) or gave up waiting
    (ETIMEOUT)."""
    check(_lib.lib().gtmoe_operators_check(device))
